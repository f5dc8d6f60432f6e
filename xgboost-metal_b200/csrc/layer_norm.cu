// Layer norm over rows of n values, forward and backward.
//
//   m = mean x,  q = 1 / sqrt(mean (x - m)^2 + eps),  h = (x - m) q,  y = h w + b
//   g = dy w,  dx = q (g - mean g - h mean(g h)),  dw = sum dy h,  db = sum dy
//
// All arithmetic is float32; the variance is the mean square of the centred
// values, never a difference of two large sums. Results are rounded once.
#include <cooperative_groups.h>

#include <algorithm>
#include <initializer_list>

#include "nn_device.cuh"

namespace xgbb::nn {
namespace {

constexpr int kThreads = 256;

// 1 / sqrt(v): the device's approximation and one step of Newton's method.
// 0, infinity and NaN pass through the approximation.
__device__ __forceinline__ float inverse_sqrt(float v) {
  const float r = rsqrtf(v);
  const float e = fmaf(-v * r, r, 1.0f);  // NaN for v = 0 and infinity
  return fabsf(e) < 1.0f ? fmaf(0.5f * r, e, r) : r;
}

// Sums N values a thread over the block, in every thread. `part` is not the
// one that the call before used, so one barrier does: whoever still reads that
// one has not passed this one.
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float (*part)[N]) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int m = 16; m; m >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], m);
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) part[warp][i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = lane < warps ? part[lane][i] : 0.0f;
#pragma unroll
    for (int m = 16; m; m >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], m);
  }
}

// How a row lies in threads that hold CH pieces each. kBlock: over the block,
// every warp its own stretch; kWarp: in a warp; kLanes: in 2^lg lanes. Pieces of a
// thread are 32 apart (kLanes: 2^lg), so that but for kLanes their addresses
// differ by constants: with distances that only the launch knew, 65536 rows of
// 1001 16-bit values took 146 us forward, and take 76.
enum Place { kBlock, kWarp, kLanes };
template <int PLACE, int VE, int CH>
struct Layout {
  uint32_t G, lane, group, first;  // lanes of a row, this one, the row's place in the block, the thread's first column
  uint32_t dim;
  bool whole;  // the warp's pieces all exist
  __device__ __forceinline__ Layout(uint32_t n, int lg) : dim(n) {
    G = PLACE == kBlock ? blockDim.x : PLACE == kWarp ? 32 : 1u << lg;
    lane = PLACE == kBlock ? threadIdx.x : threadIdx.x & (G - 1);
    group = PLACE == kBlock ? 0 : PLACE == kWarp ? threadIdx.x >> 5 : threadIdx.x >> lg;
    const uint32_t begin = PLACE == kBlock ? (threadIdx.x >> 5) * (CH * 32 * VE) : 0;
    first = begin + (PLACE == kLanes ? lane : threadIdx.x & 31) * VE;
    whole = PLACE != kLanes && begin + CH * 32 * VE <= dim;
  }
  __device__ __forceinline__ uint32_t apart(int i) const { return PLACE == kLanes ? i * G * VE : i * 32 * VE; }
  __device__ __forceinline__ bool has(int i) const { return first + apart(i) < dim; }
};
// Calls f(i) for the pieces that exist.
template <int CH, class L, class F>
__device__ __forceinline__ void each_piece(const L& at, F&& f) {
  if (at.whole) {
#pragma unroll
    for (int i = 0; i < CH; ++i) f(i);
  } else {
#pragma unroll
    for (int i = 0; i < CH; ++i)
      if (at.has(i)) f(i);
  }
}

// Sums N values a thread over the row's threads.
template <int PLACE, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], uint32_t G, float (*part)[N]) {
  if constexpr (PLACE == kBlock) {
    block_sum<N>(v, part);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (PLACE == kWarp) {
#pragma unroll
        for (int m = 16; m; m >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], m);
      } else {
        for (uint32_t m = G >> 1; m; m >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], m);
      }
    }
  }
}

// Forward. A row stays in registers between its load and its store, CH pieces of
// VE values a thread in their own type. Bound by device memory where pieces are of
// 16 bytes (100000 x 784 f32: 96 us, the copy rate's time) and by instructions where
// they are single values (65536 x 1001 bf16: 76 us, 53 % of it).
template <class T, class P, int VE, int CH, int PLACE>
__global__ void __launch_bounds__(PLACE == kBlock ? 1024 : kThreads)
    norm_kernel(const T* __restrict__ x, int64_t x_stride, uint64_t rows, uint32_t dim, const P* __restrict__ w,
                const P* __restrict__ b, float eps, T* __restrict__ y, int64_t y_stride, float* __restrict__ mean,
                float* __restrict__ rstd, int lg) {
  __shared__ float part[2][32][1];
  const Layout<PLACE, VE, CH> at(dim, lg);
  const uint32_t groups = PLACE == kBlock ? 1 : PLACE == kWarp ? kThreads / 32 : kThreads >> lg;
  const uint64_t row = uint64_t(blockIdx.x) * groups + at.group;
  const bool here = row < rows;
  const T* const xr = x + int64_t(here ? row : 0) * x_stride + at.first;  // the sums of a row that is not there go nowhere
  Pack<T, VE> v[CH];
  each_piece<CH>(at, [&](int i) { v[i] = load<T, VE>(xr + at.apart(i)); });
  float sum[1] = {0.0f};
  each_piece<CH>(at, [&](int i) {
#pragma unroll
    for (int e = 0; e < VE; ++e) sum[0] += v[i].f(e);
  });
  row_sum<PLACE, 1>(sum, at.G, part[0]);
  const float m = sum[0] / float(dim);
  float square[1] = {0.0f};
  each_piece<CH>(at, [&](int i) {
#pragma unroll
    for (int e = 0; e < VE; ++e) square[0] = fmaf(v[i].f(e) - m, v[i].f(e) - m, square[0]);
  });
  row_sum<PLACE, 1>(square, at.G, part[1]);
  const float q = inverse_sqrt(square[0] / float(dim) + eps);
  if (!here) return;
  if (at.lane == 0) {
    if (mean) mean[row] = m;
    if (rstd) rstd[row] = q;
  }
  T* const yr = y + int64_t(row) * y_stride + at.first;
  if (w && b) {
    each_piece<CH>(at, [&](int i) {
      const auto f = load<P, VE>(w + at.first + at.apart(i)), g = load<P, VE>(b + at.first + at.apart(i));
      float r[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) r[e] = fmaf((v[i].f(e) - m) * q, f.f(e), g.f(e));
      store<T, VE>(yr + at.apart(i), r);
    });
  } else {
    each_piece<CH>(at, [&](int i) {
      float r[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        r[e] = (v[i].f(e) - m) * q;
        if (w) r[e] *= to_f32(w[at.first + at.apart(i) + e]);
        if (b) r[e] += to_f32(b[at.first + at.apart(i) + e]);
      }
      store<T, VE>(yr + at.apart(i), r);
    });
  }
}

// Sums N values a lane over the warp, N a power of two: each shuffle halves how
// many a lane holds, and lane j ends with the sum of value j / (32 / N).
template <int N>
__device__ __forceinline__ float warp_sums(float (&v)[N], uint32_t lane) {
  uint32_t k = 16;
#pragma unroll
  for (int n = N / 2; n >= 1; n >>= 1, k >>= 1) {
    const bool upper = lane & k;
#pragma unroll
    for (int i = 0; i < n; ++i)
      v[i] = (upper ? v[i + n] : v[i]) + __shfl_xor_sync(0xffffffffu, upper ? v[i] : v[i + n], k);
  }
  float s = v[0];
#pragma unroll
  for (int j = 16 / N; j; j >>= 1) s += __shfl_xor_sync(0xffffffffu, s, j);
  return s;
}

// Forward for many rows of 16-byte pieces, a block R rows at a time, whose sums
// share their shuffles and their barrier. Blocks stay, CH pieces a thread, and
// the next R rows are under way into shared memory, where each thread reads
// back only what it copied itself; weight and bias come from the L1 cache once
// for all R rows. A warp takes its own values' mean and squares about it, and
// one barrier joins the warps: with n_w values, sum s_w and squares M_w of
// warp w,
//   mean = sum s_w / n,  variance n = sum M_w + n_w (s_w / n_w - mean)^2,
// all of whose terms are positive. FULL: every thread holds CH pieces.
// Bound by device memory: 32768 x 8192 bf16 in 167 us, 98 % of the copy rate. What
// bounded it before was the chain of shuffles and barriers of a row: 262 us with two
// barriers a row, 213 with one, 188 with two rows a barrier and two blocks an SM, 167
// with four rows and one block of 128 registers a thread.
template <class T, class P, int CH, int R, int MOST, bool FULL>
__global__ void __launch_bounds__(MOST)
    norm_ring_kernel(const T* __restrict__ x, int64_t x_stride, uint32_t rows, uint32_t dim,
                     const P* __restrict__ w, const P* __restrict__ b, float eps, T* __restrict__ y,
                     int64_t y_stride, float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr int VE = 16 / sizeof(T), H = VE / 2, L = 32 / R, W = MOST / 32 / L;
  extern __shared__ uint4 ring[];  // [2][R][CH][threads]
  __shared__ __align__(16) float2 part[2][R][MOST / 32];
  const uint32_t G = blockDim.x, at = threadIdx.x, lane = at & 31, warp = at >> 5;
  const float inverse = 1.0f / float(dim);
  const auto has = [&](int i) { return FULL || (at + i * G) * VE < dim; };
  const auto count = [&](uint32_t q) {  // values that warp q holds
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const uint32_t first = (q * 32 + i * G) * VE;
      n += first < dim ? min(dim - first, 32u * VE) : 0u;
    }
    return q * 32 < G ? float(n) : 0.0f;
  };
  for (uint32_t i = at; i < 2 * R * (MOST / 32); i += G) (&part[0][0][0])[i] = both(0.0f);
  __syncthreads();
  const float warp_n = count(warp), warp_inverse = warp_n > 0.0f ? 1.0f / warp_n : 0.0f;
  // After the barrier L lanes join the warps of a row, W warps each.
  const uint32_t mine = lane / L, first = (lane & (L - 1)) * W;
  const uint32_t row_bytes = CH * G * 16, stage_bytes = R * row_bytes;
  char* const own = reinterpret_cast<char*>(ring + at);
  const auto fetch = [&](uint32_t row, char* to) {
    const T* from = x + int64_t(row) * x_stride + at * VE;
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (row + r < rows)
#pragma unroll
        for (int i = 0; i < CH; ++i)
          if (has(i)) copy_async16(to + r * row_bytes + i * G * 16, from + r * x_stride + i * G * VE);
    copy_commit();
  };
  const uint32_t step = gridDim.x * R;
  fetch(blockIdx.x * R, own);
  fetch(blockIdx.x * R + step, own + stage_bytes);
  uint32_t turn = 0;
  for (uint32_t row = blockIdx.x * R; row < rows; row += step, turn ^= 1) {
    char* const stage = own + turn * stage_bytes;
    copy_wait<1>();
    float2 v[R][CH][H];
    float s[R], near[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float2 sum = both(0.0f);
#pragma unroll
      for (int i = 0; i < CH; ++i)
        if (has(i)) {
          unpack16<T>(*reinterpret_cast<const uint4*>(stage + r * row_bytes + i * G * 16), v[r][i]);
#pragma unroll
          for (int e = 0; e < H; ++e) sum = add2(sum, v[r][i][e]);
        }
      s[r] = sum.x + sum.y;
    }
    fetch(row + 2 * step, stage);  // the thread has read its values out
    const float sum = warp_sums<R>(s, lane);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      near[r] = __shfl_sync(0xffffffffu, sum, r * L) * warp_inverse;
      float2 square = both(0.0f);
#pragma unroll
      for (int i = 0; i < CH; ++i)
        if (has(i))
#pragma unroll
          for (int e = 0; e < H; ++e) {
            v[r][i][e] = add2(v[r][i][e], both(-near[r]));
            square = fma2(v[r][i][e], v[r][i][e], square);
          }
      s[r] = square.x + square.y;
    }
    const float square = warp_sums<R>(s, lane);
    if ((lane & (L - 1)) == 0) part[turn][mine][warp] = make_float2(sum, square);
    __syncthreads();
    float2 other[W];
    float m = 0.0f, q = 0.0f;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      other[j] = part[turn][mine][first + j];
      m += other[j].x;
    }
#pragma unroll
    for (int k = L / 2; k; k >>= 1) m += __shfl_xor_sync(0xffffffffu, m, k);
    m *= inverse;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const float n = FULL ? warp_n : count(first + j);
      const float off = n > 0.0f && (!FULL || (first + j) * 32 < G) ? __fdividef(other[j].x, n) - m : 0.0f;
      q += fmaf(n * off, off, other[j].y);
    }
#pragma unroll
    for (int k = L / 2; k; k >>= 1) q += __shfl_xor_sync(0xffffffffu, q, k);
    q = inverse_sqrt(q * inverse + eps);
    if (warp == 0 && (lane & (L - 1)) == 0 && row + mine < rows) {
      if (mean) mean[row + mine] = m;
      if (rstd) rstd[row + mine] = q;
    }
    // (x - mean) q, from the value about the warp's mean.
    float2 scale[R], rest[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float qr = __shfl_sync(0xffffffffu, q, r * L), mr = __shfl_sync(0xffffffffu, m, r * L);
      scale[r] = both(qr);
      rest[r] = both((near[r] - mr) * qr);
    }
    T* to = y + int64_t(row) * y_stride + at * VE;
#pragma unroll
    for (int i = 0; i < CH; ++i)
      if (has(i)) {
        float2 wv[H], bv[H];
        if (w) load_pairs<P, H>(w + (at + i * G) * VE, wv);
        if (b) load_pairs<P, H>(b + (at + i * G) * VE, bv);
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
          for (int e = 0; e < H; ++e) {
            v[r][i][e] = fma2(v[r][i][e], scale[r], rest[r]);
            if (w) v[r][i][e] = b ? fma2(v[r][i][e], wv[e], bv[e]) : mul2(v[r][i][e], wv[e]);
            else if (b) v[r][i][e] = add2(v[r][i][e], bv[e]);
          }
          if (row + r < rows) *reinterpret_cast<uint4*>(to + r * y_stride + i * G * VE) = pack16<T>(v[r][i]);
        }
      }
  }
}

// Forward for rows that registers do not hold: three passes, a block a row.
template <class T, class P, int VE>
__global__ void __launch_bounds__(1024)
    norm_long_kernel(const T* __restrict__ x, int64_t x_stride, uint64_t rows, uint32_t dim,
                     const P* __restrict__ w, const P* __restrict__ b, float eps, T* __restrict__ y,
                     int64_t y_stride, float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float part[2][32][1];
  const uint64_t row = blockIdx.x;
  const T* xr = x + int64_t(row) * x_stride;
  float sum[1] = {0.0f};
  for (uint32_t c = threadIdx.x * VE; c < dim; c += blockDim.x * VE) {
    const auto v = load<T, VE>(xr + c);
#pragma unroll
    for (int e = 0; e < VE; ++e) sum[0] += v.f(e);
  }
  block_sum<1>(sum, part[0]);
  const float m = sum[0] / float(dim);
  float square[1] = {0.0f};
  for (uint32_t c = threadIdx.x * VE; c < dim; c += blockDim.x * VE) {
    const auto v = load<T, VE>(xr + c);
#pragma unroll
    for (int e = 0; e < VE; ++e) square[0] = fmaf(v.f(e) - m, v.f(e) - m, square[0]);
  }
  block_sum<1>(square, part[1]);
  const float q = inverse_sqrt(square[0] / float(dim) + eps);
  if (threadIdx.x == 0) {
    if (mean) mean[row] = m;
    if (rstd) rstd[row] = q;
  }
  for (uint32_t c = threadIdx.x * VE; c < dim; c += blockDim.x * VE) {
    const auto v = load<T, VE>(xr + c);
    float r[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      r[e] = (v.f(e) - m) * q;
      if (w) r[e] *= to_f32(w[c + e]);
      if (b) r[e] += to_f32(b[c + e]);
    }
    store<T, VE>(y + int64_t(row) * y_stride + c, r);
  }
}

constexpr int kRingStages = 3;

// Backward. A thread owns CH pieces of VE columns, 8 values in all, of every
// row that its group takes: the rows' dx from registers, and the columns' sums
// of dy h and dy kept in registers from the first row to the last. The next
// row's values are under way while this one's are summed, where registers allow
// it. parts[block][2][dim] gets the block's sums; ONE: the grid is one cluster,
// whose blocks add theirs up through each other's shared memory, block 0's first.
template <class T, class P, int VE, int CH, int PLACE, int MOST, bool ONE = false>
__global__ void __launch_bounds__(MOST, PLACE != kBlock && VE * sizeof(T) == 16 ? 4 : 1)
    norm_grad_kernel(const T* __restrict__ grad, int64_t grad_stride, const T* __restrict__ x, int64_t x_stride,
                     const float* __restrict__ mean, const float* __restrict__ rstd, uint64_t rows, uint32_t dim,
                     const P* __restrict__ w, T* __restrict__ dx, int64_t dx_stride, float* __restrict__ parts,
                     int lg, P* __restrict__ dweight, P* __restrict__ dbias) {
  // Pieces of 16 bytes come through shared memory, the next two rows under way;
  // other 16-bit values through registers, a row ahead.
  constexpr bool kRing = PLACE != kBlock && VE * sizeof(T) == 16;
  constexpr bool kAhead = !kRing && sizeof(T) == 2 && (VE == 8 || MOST < 1024);
  constexpr int E = CH * VE, S = kRing ? kRingStages : 1;
  extern __shared__ uint4 ring[];  // [S][2][CH][threads]; at the end the groups' sums
  __shared__ float part[2][32][2];
  const Layout<PLACE, VE, CH> at(dim, lg);
  const uint32_t groups = PLACE == kBlock ? 1 : PLACE == kWarp ? kThreads / 32 : kThreads >> lg;
  const uint64_t step = uint64_t(gridDim.x) * groups;
  const float inverse = 1.0f / float(dim);
  float wv[E], dw[E] = {}, db[E] = {};
#pragma unroll
  for (int i = 0; i < CH; ++i)
#pragma unroll
    for (int e = 0; e < VE; ++e) wv[i * VE + e] = w && at.has(i) ? to_f32(w[at.first + at.apart(i) + e]) : 1.0f;
  Pack<T, VE> nv[CH], nd[CH];
  float nm = 0.0f, nq = 0.0f;
  const auto fetch_stats = [&](uint64_t row) {
    if (row >= rows) return;
    nm = mean[row];
    nq = rstd[row];
  };
  const auto fetch = [&](uint64_t row, uint32_t stage) {
    if (row < rows) {
      const T* const xr = x + int64_t(row) * x_stride + at.first;
      const T* const gr = grad + int64_t(row) * grad_stride + at.first;
      each_piece<CH>(at, [&](int i) {
        if constexpr (kRing) {
          copy_async16(&ring[((stage * 2) * CH + i) * kThreads + threadIdx.x], xr + at.apart(i));
          copy_async16(&ring[((stage * 2 + 1) * CH + i) * kThreads + threadIdx.x], gr + at.apart(i));
        } else {
          nv[i] = load<T, VE>(xr + at.apart(i));
          nd[i] = load<T, VE>(gr + at.apart(i));
        }
      });
    }
    if constexpr (kRing) copy_commit();
  };
  uint64_t row = uint64_t(blockIdx.x) * groups + at.group;
  const uint64_t turns = (rows - min(rows, uint64_t(blockIdx.x) * groups) + step - 1) / step;
#pragma unroll
  for (int i = 0; i < S - 1; ++i) fetch(row + i * step, i);
  if (kAhead) fetch(row, 0);
  fetch_stats(row);
  uint32_t stage = 0;
  for (uint64_t turn = 0; turn < turns; ++turn, row += step) {
    const float m = nm, q = nq;
    Pack<T, VE> v[CH], d[CH];
    if constexpr (kRing) {
      fetch(row + (S - 1) * step, stage == 0 ? S - 1 : stage - 1);
      copy_wait<S - 1>();
      each_piece<CH>(at, [&](int i) {
        v[i] = reinterpret_cast<const Pack<T, VE>&>(ring[((stage * 2) * CH + i) * kThreads + threadIdx.x]);
        d[i] = reinterpret_cast<const Pack<T, VE>&>(ring[((stage * 2 + 1) * CH + i) * kThreads + threadIdx.x]);
      });
      stage = stage == S - 1 ? 0 : stage + 1;
    } else {
      if (!kAhead) fetch(row, 0);
#pragma unroll
      for (int i = 0; i < CH; ++i) v[i] = nv[i], d[i] = nd[i];
      if (kAhead) fetch(row + step, 0);
    }
    fetch_stats(row + step);
    const bool here = row < rows;
    float sum[2] = {0.0f, 0.0f};
    if (here)
      each_piece<CH>(at, [&](int i) {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const int j = i * VE + e;
          const float h = (v[i].f(e) - m) * q, g = d[i].f(e) * wv[j];
          sum[0] += g;
          sum[1] = fmaf(g, h, sum[1]);
          dw[j] = fmaf(d[i].f(e), h, dw[j]);
          db[j] += d[i].f(e);
        }
      });
    row_sum<PLACE, 2>(sum, at.G, part[turn & 1]);
    if (!here) continue;
    const float a = -sum[0] * inverse * q, bb = -sum[1] * inverse * q;
    T* const dxr = dx + int64_t(row) * dx_stride + at.first;
    each_piece<CH>(at, [&](int i) {
      float r[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float h = (v[i].f(e) - m) * q, g = d[i].f(e) * wv[i * VE + e];
        r[e] = fmaf(h, bb, fmaf(g, q, a));
      }
      store<T, VE>(dxr + at.apart(i), r);
    });
  }
  if (!parts && !ONE) return;
  float* out = parts + uint64_t(blockIdx.x) * 2 * dim;
  if constexpr (PLACE != kBlock) {
    // The groups' sums: over the warp's lanes, then over the warps in order.
    float* const sums = reinterpret_cast<float*>(ring);  // [warps][2][G * E]
    if constexpr (kRing) {
      copy_wait<0>();
      __syncthreads();
    }
    for (uint32_t m = at.G; m < 32; m <<= 1)
#pragma unroll
      for (int j = 0; j < E; ++j) {
        dw[j] += __shfl_xor_sync(0xffffffffu, dw[j], m);
        db[j] += __shfl_xor_sync(0xffffffffu, db[j], m);
      }
    const uint32_t width = at.G * E, warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) < at.G)
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const uint32_t c = at.first + at.apart(j / VE) + j % VE;
        sums[(warp * 2) * width + c] = dw[j];
        sums[(warp * 2 + 1) * width + c] = db[j];
      }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < 2 * width; i += kThreads) {
      const uint32_t which = i / width, c = i % width;
      float s = 0.0f;
#pragma unroll
      for (int q = 0; q < kThreads / 32; ++q) s += sums[q * 2 * width + i];
      if (ONE) sums[i] = s;  // the thread's own, and read by no other yet
      else if (c < dim) out[which * dim + c] = s;
    }
    if (ONE) {
      const auto cluster = cooperative_groups::this_cluster();
      const uint32_t blocks = cluster.num_blocks();
      cluster.sync();
      for (uint32_t i = cluster.block_rank() * kThreads + threadIdx.x; i < 2 * width; i += blocks * kThreads) {
        const uint32_t which = i / width, c = i % width;
        float s = 0.0f;
        for (uint32_t q = 0; q < blocks; ++q) s += cluster.map_shared_rank(sums, q)[i];
        P* to = which ? dbias : dweight;
        if (to && c < dim) to[c] = from_f32<P>(s);
      }
      cluster.sync();  // the blocks' memory is read until here
    }
  } else {
    each_piece<CH>(at, [&](int i) {
      float a[VE], b[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        a[e] = dw[i * VE + e];
        b[e] = db[i * VE + e];
      }
      store_global<float, VE>(out + at.first + at.apart(i), a);
      store_global<float, VE>(out + dim + at.first + at.apart(i), b);
    });
  }
}

// The same for many rows of 16-byte pieces, a block of 512 threads at most, or a
// cluster of C of them, R rows at a time: the rows' 2 R sums are reduced together,
// each shuffle halving how many of them a lane holds, and share their barrier;
// in a cluster each block leaves its warps' sums with all blocks. The next R
// rows are under way into shared memory. Bound by device memory: 32768 x 4096 bf16
// in 127 us, 97 % of the copy rate (179 us a row at a time); in clusters by their
// barriers (16384 x 8192: 164 us, 75 %; 8000 x 16384: 221 us, 54 %).
template <class T, class P, int R, int C, bool FULL>
__global__ void __launch_bounds__(512, 1)
    norm_grad_rows_kernel(const T* __restrict__ grad, int64_t grad_stride, const T* __restrict__ x,
                          int64_t x_stride, const float* __restrict__ mean, const float* __restrict__ rstd,
                          uint32_t rows, uint32_t dim, const P* __restrict__ w, T* __restrict__ dx,
                          int64_t dx_stride, float* __restrict__ parts) {
  constexpr int VE = 16 / sizeof(T), CH = 8 / VE, H = VE / 2, V = 2 * R, L = 32 / V, W = 16 / L;
  extern __shared__ uint4 ring[];  // [2][R][2][CH][threads]
  __shared__ __align__(16) float part[2][C][V][16];
  const auto cluster = cooperative_groups::this_cluster();
  const uint32_t rank = C > 1 ? cluster.block_rank() : 0, id = blockIdx.x / C;
  const auto barrier = [&] {
    if constexpr (C > 1) cluster.sync();
    else __syncthreads();
  };
  // The block's columns begin at those of the blocks before it.
  const uint32_t G = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t at = rank * G * CH + threadIdx.x;
  const float inverse = 1.0f / float(dim);
  const auto has = [&](int i) { return FULL || (at + i * G) * VE < dim; };
  for (uint32_t i = threadIdx.x; i < 2 * C * V * 16; i += G) (&part[0][0][0][0])[i] = 0.0f;
  barrier();
  float2 wv[CH][H], dw[CH][H] = {}, db[CH][H] = {};
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const uint32_t c = (at + i * G) * VE;
#pragma unroll
    for (int e = 0; e < H; ++e)
      wv[i][e] = w && c < dim ? make_float2(to_f32(w[c + 2 * e]), to_f32(w[c + 2 * e + 1])) : both(1.0f);
  }
  const uint32_t half = CH * G * 16, row_bytes = 2 * half, stage_bytes = R * row_bytes;
  char* const own = reinterpret_cast<char*>(ring + threadIdx.x);
  const auto fetch = [&](uint32_t row, char* to) {
    const T* xs = x + int64_t(row) * x_stride + at * VE;
    const T* gs = grad + int64_t(row) * grad_stride + at * VE;
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (row + r < rows)
#pragma unroll
        for (int i = 0; i < CH; ++i)
          if (has(i)) {
            copy_async16(to + r * row_bytes + i * G * 16, xs + r * x_stride + i * G * VE);
            copy_async16(to + r * row_bytes + half + i * G * 16, gs + r * grad_stride + i * G * VE);
          }
    copy_commit();
  };
  const uint32_t step = gridDim.x / C * R;
  float nm[R], nq[R];
  const auto fetch_stats = [&](uint32_t row) {
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (row + r < rows) {
        nm[r] = mean[row + r];
        nq[r] = rstd[row + r];
      }
  };
  fetch(id * R, own);
  fetch(id * R + step, own + stage_bytes);
  fetch_stats(id * R);
  uint32_t turn = 0;
  for (uint32_t row = id * R; row < rows; row += step, turn ^= 1) {
    char* const stage = own + turn * stage_bytes;
    float q[R], val[V];
    float2 h[R][CH][H], d[R][CH][H];
    copy_wait<1>();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      val[2 * r] = val[2 * r + 1] = 0.0f;
      q[r] = nq[r];
      if (row + r >= rows) continue;
      const float m = nm[r];
      float2 sum_g = both(0.0f), sum_gh = both(0.0f);
#pragma unroll
      for (int i = 0; i < CH; ++i)
        if (has(i)) {
          unpack16<T>(*reinterpret_cast<const uint4*>(stage + r * row_bytes + i * G * 16), h[r][i]);
          unpack16<T>(*reinterpret_cast<const uint4*>(stage + r * row_bytes + half + i * G * 16), d[r][i]);
#pragma unroll
          for (int e = 0; e < H; ++e) {
            h[r][i][e] = mul2(add2(h[r][i][e], both(-m)), both(q[r]));
            const float2 g = mul2(d[r][i][e], wv[i][e]);
            sum_g = add2(sum_g, g);
            sum_gh = fma2(g, h[r][i][e], sum_gh);
          }
        }
      val[2 * r] = sum_g.x + sum_g.y;
      val[2 * r + 1] = sum_gh.x + sum_gh.y;
    }
    fetch(row + 2 * step, stage);  // the thread has read its values out
    fetch_stats(row + step);
    float s = warp_sums<V>(val, lane);  // of value lane / L
    if ((lane & (L - 1)) == 0) {
      if constexpr (C > 1) {
#pragma unroll
        for (int q = 0; q < C; ++q) *cluster.map_shared_rank(&part[turn][rank][lane / L][warp], q) = s;
      } else {
        part[turn][0][lane / L][warp] = s;
      }
    }
    if constexpr (C > 1) cluster.barrier_arrive();
    // The columns' sums, while the sums travel.
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (row + r < rows)
#pragma unroll
        for (int i = 0; i < CH; ++i)
          if (has(i))
#pragma unroll
            for (int e = 0; e < H; ++e) {
              dw[i][e] = fma2(d[r][i][e], h[r][i][e], dw[i][e]);
              db[i][e] = add2(db[i][e], d[r][i][e]);
            }
    if constexpr (C > 1) cluster.barrier_wait();
    else __syncthreads();
    s = 0.0f;
#pragma unroll
    for (int q = 0; q < C; ++q) {
      const auto others = load<float, W>(&part[turn][q][lane / L][(lane & (L - 1)) * W]);
#pragma unroll
      for (int j = 0; j < W; ++j) s += others.v[j];
    }
#pragma unroll
    for (int j = L / 2; j; j >>= 1) s += __shfl_xor_sync(0xffffffffu, s, j);
    s *= -inverse;
    T* to = dx + int64_t(row) * dx_stride + at * VE;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      // q (g - a - h b), with -q a and -q b.
      const float2 a = both(__shfl_sync(0xffffffffu, s, 2 * r * L) * q[r]);
      const float2 b = both(__shfl_sync(0xffffffffu, s, (2 * r + 1) * L) * q[r]);
      if (row + r >= rows) continue;
#pragma unroll
      for (int i = 0; i < CH; ++i)
        if (has(i)) {
#pragma unroll
          for (int e = 0; e < H; ++e) h[r][i][e] = fma2(h[r][i][e], b, fma2(mul2(d[r][i][e], wv[i][e]), both(q[r]), a));
          *reinterpret_cast<uint4*>(to + r * dx_stride + i * G * VE) = pack16<T>(h[r][i]);
        }
    }
  }
  if (!parts) return;
  float* out = parts + uint64_t(id) * 2 * dim;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const uint32_t c = (at + i * G) * VE;
    float a[VE], b[VE];
#pragma unroll
    for (int e = 0; e < H; ++e) {
      a[2 * e] = dw[i][e].x;
      a[2 * e + 1] = dw[i][e].y;
      b[2 * e] = db[i][e].x;
      b[2 * e + 1] = db[i][e].y;
    }
    if (c < dim) {
      store_global<float, VE>(out + c, a);
      store_global<float, VE>(out + dim + c, b);
    }
  }
}

// dx for rows that registers do not hold: two passes, a block a row.
template <class T, class P, int VE>
__global__ void __launch_bounds__(1024)
    norm_grad_long_kernel(const T* __restrict__ grad, int64_t grad_stride, const T* __restrict__ x,
                          int64_t x_stride, const float* __restrict__ mean, const float* __restrict__ rstd,
                          uint32_t dim, const P* __restrict__ w, T* __restrict__ dx, int64_t dx_stride) {
  __shared__ float part[32][2];
  const uint64_t row = blockIdx.x;
  const T* xr = x + int64_t(row) * x_stride;
  const T* gr = grad + int64_t(row) * grad_stride;
  const float m = mean[row], q = rstd[row];
  float sum[2] = {0.0f, 0.0f};
  for (uint32_t c = threadIdx.x * VE; c < dim; c += blockDim.x * VE) {
    const auto v = load<T, VE>(xr + c);
    const auto d = load<T, VE>(gr + c);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const float g = w ? d.f(e) * to_f32(w[c + e]) : d.f(e);
      sum[0] += g;
      sum[1] = fmaf(g, (v.f(e) - m) * q, sum[1]);
    }
  }
  block_sum<2>(sum, part);
  const float a = sum[0] / float(dim), bb = sum[1] / float(dim);
  for (uint32_t c = threadIdx.x * VE; c < dim; c += blockDim.x * VE) {
    const auto v = load<T, VE>(xr + c);
    const auto d = load<T, VE>(gr + c);
    float r[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const float g = w ? d.f(e) * to_f32(w[c + e]) : d.f(e);
      r[e] = q * (g - a - (v.f(e) - m) * q * bb);
    }
    store<T, VE>(dx + int64_t(row) * dx_stride + c, r);
  }
}

// The column sums that go with norm_grad_long_kernel: block (x, y) sums the
// column tile y over a span of rows.
template <class T, int VE>
__global__ void __launch_bounds__(kThreads)
    norm_columns_kernel(const T* __restrict__ grad, int64_t grad_stride, const T* __restrict__ x, int64_t x_stride,
                        const float* __restrict__ mean, const float* __restrict__ rstd, uint64_t rows, uint32_t dim,
                        float* __restrict__ parts) {
  constexpr int U = 4;
  const uint32_t c = (blockIdx.y * kThreads + threadIdx.x) * VE;
  if (c >= dim) return;
  float dw[VE] = {}, db[VE] = {};
  for (uint64_t row = blockIdx.x; row < rows; row += uint64_t(gridDim.x) * U) {
    Pack<T, VE> v[U], d[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t r = row + uint64_t(u) * gridDim.x;
      if (r < rows) {
        v[u] = load<T, VE>(x + int64_t(r) * x_stride + c);
        d[u] = load<T, VE>(grad + int64_t(r) * grad_stride + c);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t r = row + uint64_t(u) * gridDim.x;
      if (r >= rows) break;
      const float m = mean[r], q = rstd[r];
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        dw[e] = fmaf(d[u].f(e), (v[u].f(e) - m) * q, dw[e]);
        db[e] += d[u].f(e);
      }
    }
  }
  float* out = parts + uint64_t(blockIdx.x) * 2 * dim + c;
  store_global<float, VE>(out, dw);
  store_global<float, VE>(out + dim, db);
}

// The parts' sums: 32 columns a block (of dw's and db's 2 dim), each warp every
// 32nd part, then the warps in order.
template <class P>
__global__ void __launch_bounds__(1024)
    norm_parts_kernel(const float* __restrict__ parts, uint32_t count, uint32_t dim, P* __restrict__ dw,
                      P* __restrict__ db) {
  constexpr int kWarps = 32, U = 4;
  __shared__ float sums[kWarps][33];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (c < 2 * dim)
    for (uint32_t p = warp; p < count; p += kWarps * U) {
      float v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = p + u * kWarps < count ? parts[uint64_t(p + u * kWarps) * 2 * dim + c] : 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u) s += v[u];
    }
  sums[warp][lane] = s;
  __syncthreads();
  s = sums[lane][warp];  // warp w adds up column w
#pragma unroll
  for (int m = 16; m; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
  const uint32_t mine = blockIdx.x * 32 + warp;
  if (lane || mine >= 2 * dim) return;
  P* to = mine < dim ? dw : db;
  if (to) to[mine < dim ? mine : mine - dim] = from_f32<P>(s);
}

bool param_aligned(const void* p, size_t size, uint64_t n) {
  return reinterpret_cast<uintptr_t>(p) % std::min<size_t>(32, n * size) == 0;
}

// Calls f with the widest VE that every matrix and vector allows: 16 bytes of T,
// a pair of 16-bit values, or one value.
template <class T, class F>
void with_norm_width(std::initializer_list<Mat> mats, std::initializer_list<const void*> vectors, int param_type,
                     uint64_t rows, uint64_t dim, F&& f) {
  const auto fits = [&](uint64_t n) {
    bool ok = dim % n == 0;
    for (const Mat& m : mats) ok = ok && row_aligned(m.data, m.stride, rows, type_size(m.type), n);
    for (const void* p : vectors) ok = ok && param_aligned(p, type_size(param_type), n);
    return ok;
  };
  constexpr int kWide = 16 / sizeof(T);
  if (fits(kWide)) return f(std::integral_constant<int, kWide>());
  if constexpr (kWide > 4) {
    if (fits(2)) return f(std::integral_constant<int, 2>());
  }
  f(std::integral_constant<int, 1>());
}

// What a launch may ask for: the stream kernels' ring, at its largest.
constexpr size_t kMostShared = 128 * 1024;

// Launches a kernel with more shared memory than a launch has unasked.
template <class... Params, class... Args>
void launch_ring(void (*kernel)(Params...), unsigned blocks, unsigned threads, size_t shared, cudaStream_t stream,
                 Args... args) {
  allow_shared(kernel, shared, kMostShared);
  kernel<<<blocks, threads, shared, stream>>>(args...);
}

// The same in clusters of `cluster` blocks.
template <class... Params, class... Args>
void launch_cluster(void (*kernel)(Params...), unsigned blocks, unsigned threads, unsigned cluster, size_t shared,
                    cudaStream_t stream, Args... args) {
  allow_shared(kernel, shared, kMostShared);
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim = {cluster, 1, 1};
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(blocks);
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  config.attrs = &attribute;
  config.numAttrs = 1;
  XGBB_CUDA(cudaLaunchKernelEx(&config, kernel, Params(args)...));
}

// How the gradient takes rows of `dim` values: in the lanes of a warp (one: in
// one cluster of blocks), in a block's registers where they hold them, else in
// passes; and, where there are rows enough and they come in 16-byte pieces, in a
// stream through shared memory (clusters of `ring` blocks).
struct GradPlan {
  bool warp, one = false, fits;
  uint32_t ring = 0;
  int lg = 0;
  uint32_t threads = 0, blocks = 0;            // of the first forms
  uint32_t ring_threads = 0, ring_blocks = 0;  // of the stream
  GradPlan(uint64_t rows, uint64_t dim) : warp(dim <= 256), fits(dim <= 8192) {
    if (warp) {
      while ((8ull << lg) < dim) ++lg;
      threads = kThreads;
      // Up to eight turns of eight blocks: one cluster, one launch and no workspace.
      // 512 x 64 f32, two turns: 4.5 us for 4.8 in parts; 2048 x 64, eight: 9.0 for
      // 5.0, but a call from Python takes 11.5 us for 15.6.
      const uint64_t once = kThreads >> lg;
      if (rows <= once * 64) {
        one = true;
        blocks = 1;
        while (blocks < 8 && blocks * once < rows) blocks *= 2;
        return;
      }
      blocks = uint32_t(std::min<uint64_t>(148 * 4, (rows + once - 1) / once));
      return;
    }
    // A block an SM, then four rows a block at least: the blocks' parts are read again.
    threads = fits ? uint32_t((dim + 255) / 256 * 32) : 1024;
    blocks = fits ? uint32_t(std::min<uint64_t>(148 * (1024 / threads), std::max((rows + 3) / 4, std::min<uint64_t>(rows, 148))))
                  : uint32_t(std::min<uint64_t>(296, (rows + 15) / 16));
    // One block of 512 threads an SM. (Clusters of four blocks of 256 threads, two
    // an SM, took 284 us for 16384 x 8192 of 16 bits where clusters of two blocks of
    // 512 took 186.) Clusters of four and eight do not fill every SM, and fit on 128.
    ring = dim <= 4096 ? 1 : dim <= 8192 ? 2 : dim <= 16384 ? 4 : dim <= 32768 ? 8 : 0;
    if (!ring) return;
    ring_threads = uint32_t((dim + 256 * ring - 1) / (256 * ring) * 32);
    ring_blocks = ring == 1 ? 148 * (512 / ring_threads) : ring == 2 ? 148 : 128;
    // The stream from 16 rows a block or cluster on. A row a block at a time takes
    // 24.8 us for 14.7 at 2368 x 4096 bf16, where it begins, and 10.2 for 8.8 at 592;
    // 9.6 for 8.4 at 2368 x 1024, 6.7 for 7.4 at 592.
    if (rows < uint64_t(ring_blocks / ring) * 16) ring = 0;
  }
  uint32_t parts() const { return one ? 0 : ring ? std::max(blocks, ring_blocks / ring) : blocks; }
};

}  // namespace

void layer_norm(const Mat& x, uint64_t rows, uint64_t dim, const void* weight, const void* bias, int param_type,
                float eps, const Mat& y, float* mean, float* rstd, cudaStream_t stream) {
  if (!rows) return;
  with_param_types(x.type, param_type, [&](auto* pt, auto* pp) {
    using T = std::remove_pointer_t<decltype(pt)>;
    using P = std::remove_pointer_t<decltype(pp)>;
    const T* in = static_cast<const T*>(x.data);
    T* out = static_cast<T*>(const_cast<void*>(y.data));
    const P *w = static_cast<const P*>(weight), *b = static_cast<const P*>(bias);
    with_norm_width<T>({x, y}, {weight, bias}, param_type, rows, dim, [&](auto width) {
      constexpr int VE = decltype(width)::value, kWide = 16 / sizeof(T);
      constexpr int kMost = std::min(32 / VE, 16);      // pieces that a thread may hold
      constexpr int kSome = VE == 1 ? 8 : 16 / VE;      // pieces that it holds rather than leave them to more lanes
      const uint64_t pieces = (dim + VE - 1) / VE;
      const auto go = [&](auto count, auto place, unsigned blocks, unsigned threads, int lg) {
        norm_kernel<T, P, VE, decltype(count)::value, decltype(place)::value><<<blocks, threads, 0, stream>>>(
            in, x.stride, rows, uint32_t(dim), w, b, eps, out, y.stride, mean, rstd, lg);
      };
      const auto pick = [&](uint64_t need, auto place, unsigned blocks, unsigned threads, int lg) {
        if (need <= 1) go(std::integral_constant<int, 1>(), place, blocks, threads, lg);
        else if (need <= 2) go(std::integral_constant<int, 2>(), place, blocks, threads, lg);
        else if (need <= 4) go(std::integral_constant<int, 4>(), place, blocks, threads, lg);
        else if constexpr (kMost >= 8) {
          if (need <= 8) go(std::integral_constant<int, 8>(), place, blocks, threads, lg);
          else if constexpr (kMost >= 16) {
            go(std::integral_constant<int, 16>(), place, blocks, threads, lg);
          }
        }
      };
      // Rows of up to 512 pieces in lanes of a warp, where there is one for each SM.
      // Fewer go faster in a block each: 74 x 255 f32 take 2.3 us for 3.3, and 2368 x 255
      // 3.5 for 3.5, 37888 x 255 22.3 for 14.9.
      if (pieces <= 32 * kMost && pieces <= 512 && rows >= 148) {
        int lg = 0;
        while (lg < 5 && (uint64_t(kSome) << lg) < pieces) ++lg;
        const uint64_t need = (pieces + (1u << lg) - 1) >> lg;
        if (lg == 5) pick(need, std::integral_constant<int, kWarp>(), blocks_for(rows, kThreads >> lg), kThreads, lg);
        else pick(need, std::integral_constant<int, kLanes>(), blocks_for(rows, kThreads >> lg), kThreads, lg);
        return;
      }
      if (dim > 16384) {
        norm_long_kernel<T, P, VE><<<unsigned(rows), 1024, 0, stream>>>(in, x.stride, rows, uint32_t(dim), w, b,
                                                                      eps, out, y.stride, mean, rstd);
        return;
      }
      if constexpr (VE == kWide) {
        constexpr int CH = 2;
        const unsigned threads = blocks_for(pieces, CH * 32) * 32;
        const bool full = pieces == CH * threads;
        const auto ring = [&](auto most, auto at_once) {
          constexpr int MOST = decltype(most)::value, R = decltype(at_once)::value;
          launch_ring(full ? norm_ring_kernel<T, P, CH, R, MOST, true> : norm_ring_kernel<T, P, CH, R, MOST, false>,
                      148 * (MOST / threads), threads, size_t(2) * R * CH * threads * 16, stream, in, x.stride,
                      uint32_t(rows), uint32_t(dim), w, b, eps, out, y.stride, mean, rstd);
        };
        // The stream from 16 rows an SM on: 2368 x 4096 bf16 in 7.4 us for 12.2 with a
        // block a row, 592 rows 4.5 for 4.4. (float32: 32768 x 8192 in 362 for 358, 4096
        // columns 186 for 155.)
        if (rows >= 148 * 16 && param_aligned(weight, 32, 1) && param_aligned(bias, 32, 1)) {
          if (threads <= 512) return ring(std::integral_constant<int, 512>(), std::integral_constant<int, 4>());
          if (threads <= 1024) return ring(std::integral_constant<int, 1024>(), std::integral_constant<int, 2>());
        }
      }
      // Many rows: as few threads a row as hold it. Few: as many as it has pieces.
      const uint64_t each = rows >= 148 ? 16 / VE : 1;
      const uint64_t threads =
          std::max<uint64_t>(std::min<uint64_t>(1024, ((pieces + each - 1) / each + 31) / 32 * 32), 32);
      pick((pieces + threads - 1) / threads, std::integral_constant<int, kBlock>(), unsigned(rows), unsigned(threads), 0);
    });
  });
  XGBB_CUDA(cudaGetLastError());
}

size_t layer_norm_backward_workspace(uint64_t rows, uint64_t dim) {
  return size_t(GradPlan(rows, dim).parts()) * 2 * dim * 4;
}

void layer_norm_backward(const Mat& grad, const Mat& x, const float* mean, const float* rstd, uint64_t rows,
                         uint64_t dim, const void* weight, int param_type, const Mat& dx, void* dweight,
                         void* dbias, void* workspace, cudaStream_t stream) {
  const bool params = dweight || dbias;
  const GradPlan plan(rows, dim);
  float* parts = params ? static_cast<float*>(workspace) : nullptr;
  uint32_t used = plan.blocks;  // parts that are written
  with_param_types(x.type, param_type, [&](auto* pt, auto* pp) {
    using T = std::remove_pointer_t<decltype(pt)>;
    using P = std::remove_pointer_t<decltype(pp)>;
    const T* g = static_cast<const T*>(grad.data);
    const T* v = static_cast<const T*>(x.data);
    const P* w = static_cast<const P*>(weight);
    T* out = static_cast<T*>(const_cast<void*>(dx.data));
    P *dw = static_cast<P*>(dweight), *db = static_cast<P*>(dbias);
    if (rows || plan.one)
      with_norm_width<T>({grad, x, dx}, {}, param_type, rows, dim, [&](auto width) {
        constexpr int VE = decltype(width)::value;
        // The groups' sums, in the place of the rows under way.
        const size_t sums = std::max<size_t>((kThreads / 32) * 2 * (size_t(8) << plan.lg) * 4,
                                             VE * sizeof(T) == 16 ? kRingStages * 2 * (8 / VE) * kThreads * 16 : 0);
        if (plan.one) {
          launch_cluster(norm_grad_kernel<T, P, VE, 8 / VE, kLanes, kThreads, true>, plan.blocks, kThreads, plan.blocks,
                         sums, stream, g, grad.stride, v, x.stride, mean, rstd, rows, uint32_t(dim), w, out, dx.stride,
                         static_cast<float*>(nullptr), plan.lg, dw, db);
        } else if (plan.warp) {
          const auto kernel = plan.lg == 5 ? norm_grad_kernel<T, P, VE, 8 / VE, kWarp, kThreads>
                                           : norm_grad_kernel<T, P, VE, 8 / VE, kLanes, kThreads>;
          launch_ring(kernel, plan.blocks, plan.threads, sums, stream, g, grad.stride, v, x.stride, mean, rstd, rows,
                      uint32_t(dim), w, out, dx.stride, parts, plan.lg, static_cast<P*>(nullptr),
                      static_cast<P*>(nullptr));
        } else if (plan.ring && VE * sizeof(T) == 16) {
          if constexpr (VE * sizeof(T) == 16) {
            constexpr int R = sizeof(T) == 2 ? 4 : 2;
            const auto go = [&](auto blocks) {
              constexpr int C = decltype(blocks)::value;
              const auto kernel = dim == plan.ring_threads * 8ull * C ? norm_grad_rows_kernel<T, P, R, C, true>
                                                                     : norm_grad_rows_kernel<T, P, R, C, false>;
              const size_t shared = size_t(2) * R * 2 * 8 * sizeof(T) * plan.ring_threads;
              used = plan.ring_blocks / C;
              if (C == 1)
                launch_ring(kernel, plan.ring_blocks, plan.ring_threads, shared, stream, g, grad.stride, v, x.stride,
                            mean, rstd, uint32_t(rows), uint32_t(dim), w, out, dx.stride, parts);
              else
                launch_cluster(kernel, plan.ring_blocks, plan.ring_threads, C, shared, stream, g, grad.stride, v,
                               x.stride, mean, rstd, uint32_t(rows), uint32_t(dim), w, out, dx.stride, parts);
            };
            if (plan.ring == 1) go(std::integral_constant<int, 1>());
            else if (plan.ring == 2) go(std::integral_constant<int, 2>());
            else if (plan.ring == 4) go(std::integral_constant<int, 4>());
            else go(std::integral_constant<int, 8>());
          }
        } else if (plan.fits) {
          const auto kernel = plan.threads <= 512 ? norm_grad_kernel<T, P, VE, 8 / VE, kBlock, 512>
                                                  : norm_grad_kernel<T, P, VE, 8 / VE, kBlock, 1024>;
          kernel<<<plan.blocks, plan.threads, 0, stream>>>(
              g, grad.stride, v, x.stride, mean, rstd, rows, uint32_t(dim), w, out, dx.stride, parts, 0, nullptr,
              nullptr);
        } else {
          norm_grad_long_kernel<T, P, VE><<<unsigned(rows), 1024, 0, stream>>>(
              g, grad.stride, v, x.stride, mean, rstd, uint32_t(dim), w, out, dx.stride);
          if (params)
            norm_columns_kernel<T, VE><<<dim3(plan.blocks, blocks_for(dim, kThreads * VE)), kThreads, 0, stream>>>(
                g, grad.stride, v, x.stride, mean, rstd, rows, uint32_t(dim), parts);
        }
      });
    if (params && !plan.one)
      norm_parts_kernel<P><<<blocks_for(2 * dim, 32), 1024, 0, stream>>>(
          parts, used, uint32_t(dim), dw, db);
  });
  XGBB_CUDA(cudaGetLastError());
}

}  // namespace xgbb::nn
