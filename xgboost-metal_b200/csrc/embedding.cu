// Embedding lookup with scaling, one token or a summed bag of tokens a row,
// and the gradient of the tokens' scales. The table's gradient is in
// embedding_grad.cu.
//
//   y[r] = a * sum_t s[r][t] W[k[r][t]],    ds[r][t] = a * <dy[r], W[k[r][t]]>
//
// A token below 0 is missing and adds nothing, whatever its scale holds. A
// token past the table makes its row's result NaN: nothing is read for it.
// Sums are float32 in a fixed order, and are rounded once, when written.
#include "nn_device.cuh"

namespace xgbb::nn {

size_t type_size(int type) { return type == kF32 || type == kI32 ? 4 : type == kI64 ? 8 : 2; }

namespace {

constexpr int kThreads = 256;
const float kNaN = __builtin_nanf("");

// One token a row: a copy with a factor. Flat over the (row, piece) pairs, so
// that neighbouring threads move neighbouring pieces, four pieces in flight a
// thread.
template <class T, class O, int VE>
__global__ void __launch_bounds__(kThreads)
    lookup_kernel(Tokens k, const T* __restrict__ table, int64_t table_stride, uint64_t vocab, uint32_t pieces,
                  FastDiv div, uint64_t total, float scale, Scales s, O* __restrict__ out, int64_t out_stride,
                  float nan) {
  constexpr int U = 4;
  const uint64_t base = uint64_t(blockIdx.x) * (kThreads * U) + threadIdx.x;
  const bool wide = k.type == kI64;
  uint64_t row[U];
  uint32_t piece[U];
  int64_t token[U];
  float f[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint64_t i = base + u * kThreads;
    row[u] = total <= 0xffffffffull ? div.div(uint32_t(i)) : i / pieces;
    piece[u] = uint32_t(i - row[u] * pieces);
    token[u] = i < total ? load_token(k.data, wide, int64_t(row[u]) * k.stride_row) : -1;
    f[u] = scale;
    if (s.data && token[u] >= 0) f[u] *= s.data[int64_t(row[u]) * s.stride_row];
  }
  Pack<T, VE> v[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (uint64_t(token[u]) < vocab) v[u] = load<T, VE>(table + token[u] * table_stride + piece[u] * VE);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (base + u * kThreads >= total) break;
    float y[VE];
#pragma unroll
    for (int j = 0; j < VE; ++j)
      y[j] = uint64_t(token[u]) < vocab ? f[u] * v[u].f(j) : token[u] < 0 ? 0.0f : nan;
    store_global<O, VE>(out + int64_t(row[u]) * out_stride + piece[u] * VE, y);
  }
}

// A bag a row: 2^lg lanes own a row's columns (or a tile of them), VE values
// each; S = 2^ls such groups share a row's tokens, a contiguous span each, and
// add their sums up in shared memory, first span first. A group reads its
// tokens K to a lane, a step ahead, and hands them round by shuffles, eight
// gathers in flight.
template <class T, class O, int VE, int K, bool SCALED>
__global__ void __launch_bounds__(kThreads, (Sum<T, VE>::kPairs && K == 1 ? 4 : 2))
    bag_kernel(Tokens k, const T* __restrict__ table, int64_t table_stride, uint32_t vocab, uint32_t dim,
               float scale, Scales s, O* __restrict__ out, int64_t out_stride, int lg, int ls, float nan) {
  constexpr int U = 8;
  __shared__ float part[kThreads * VE];
  const uint32_t G = 1u << lg, lane = threadIdx.x & (G - 1), group = threadIdx.x >> lg;
  const uint32_t S = 1u << ls, span = group & (S - 1);
  const uint64_t row = uint64_t(blockIdx.x) * (kThreads >> (lg + ls)) + (group >> ls);
  const uint32_t col = (blockIdx.y * G + lane) * VE;
  const bool wide = k.type == kI64;
  const uint32_t count = uint32_t(k.per_row), per = (count + S - 1) >> ls;
  const uint32_t begin = min(count, per * span), end = row < k.rows ? min(count, begin + per) : 0;
  // Lanes past the last column read the last piece, and write nothing.
  const T* const columns = table + min(col, dim - VE);
  const char* const tokens = static_cast<const char*>(k.data) + int64_t(row) * k.stride_row * (wide ? 8 : 4);
  const float* const scales = SCALED ? s.data + int64_t(row) * s.stride_row : nullptr;
  Sum<T, VE> acc;
  acc.clear();
  bool bad = false;
  int token[K], next[K];  // -1: missing, past the table, or past the span
  float f[K], next_f[K];
  const auto fetch = [&](uint32_t t0) {
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const uint32_t t = t0 + i * G + lane;
      int64_t w = -1;
      if (t < end) w = load_token(tokens, wide, int64_t(t) * k.stride_col);
      next[i] = uint64_t(w) < vocab ? int(w) : -1;
      bad |= w >= int64_t(vocab);
      if (SCALED) next_f[i] = next[i] >= 0 ? scales[int64_t(t) * s.stride_col] : 0.0f;
    }
  };
  fetch(begin);
  for (uint32_t t0 = begin; __any_sync(0xffffffffu, t0 < end); t0 += G * K) {
    bool whole = true;
#pragma unroll
    for (int i = 0; i < K; ++i) {
      token[i] = next[i];
      whole = whole && token[i] >= 0;
      if (SCALED) f[i] = next_f[i];
    }
    whole = __all_sync(0xffffffffu, whole);
    fetch(t0 + G * K);
    const uint32_t steps = K > 1 ? 8 : G;
    for (uint32_t j = 0; j < steps; j += U) {
      Pack<T, VE> v[U];
      int at[U];
      float ff[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int slot = K > 1 ? u / (8 / K) : 0, from = K > 1 ? u % (8 / K) : int(j) + u;
        at[u] = __shfl_sync(0xffffffffu, token[slot], from, G);
        if (SCALED) ff[u] = __shfl_sync(0xffffffffu, f[slot], from, G);
      }
      if (whole) {
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = load<T, VE>(columns + at[u] * table_stride);
#pragma unroll
        for (int u = 0; u < U; ++u) acc.template add<SCALED>(v[u], SCALED ? ff[u] : 1.0f);
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (at[u] >= 0) v[u] = load<T, VE>(columns + at[u] * table_stride);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (at[u] >= 0) acc.template add<SCALED>(v[u], SCALED ? ff[u] : 1.0f);
      }
    }
  }
  // A token past the table anywhere in the group's span.
  for (uint32_t m = 1; m < G; m <<= 1) bad |= __shfl_xor_sync(0xffffffffu, int(bad), m) != 0;
  float sum[VE];
  acc.get(sum);
  if (bad)
#pragma unroll
    for (int e = 0; e < VE; ++e) sum[e] = nan;
  if (S > 1) {
#pragma unroll
    for (int e = 0; e < VE; ++e) part[threadIdx.x * VE + e] = sum[e];
    __syncthreads();
    if (span == 0)
      for (uint32_t q = 1; q < S; ++q)
#pragma unroll
        for (int e = 0; e < VE; ++e) sum[e] += part[(threadIdx.x + (q << lg)) * VE + e];
  }
  if (span == 0 && row < k.rows && col < dim) {
#pragma unroll
    for (int e = 0; e < VE; ++e) sum[e] *= scale;
    store_global<O, VE>(out + int64_t(row) * out_stride + col, sum);
  }
}

// The scales' gradient: 32 lanes a row, which hold the row's gradient in
// pieces and walk the row's tokens.
template <class T, class O, int VE>
__global__ void __launch_bounds__(kThreads)
    scale_grad_kernel(const O* __restrict__ grad, int64_t grad_stride, Tokens k, const T* __restrict__ table,
                      int64_t table_stride, uint64_t vocab, uint32_t dim, float scale, float* __restrict__ out,
                      uint64_t total, float nan) {
  const uint64_t i = (uint64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  if (i >= total) return;
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t row = i / k.per_row, t = i - row * k.per_row;
  const int64_t w =
      load_token(k.data, k.type == kI64, int64_t(row) * k.stride_row + int64_t(t) * k.stride_col);
  float acc = 0.0f;
  if (w >= 0 && w < int64_t(vocab)) {
    for (uint32_t c = lane * VE; c < dim; c += 32 * VE) {
      const auto a = load<T, VE>(table + w * table_stride + c);
      const auto b = load<O, VE>(grad + int64_t(row) * grad_stride + c);
#pragma unroll
      for (int e = 0; e < VE; ++e) acc = fmaf(a.f(e), b.f(e), acc);
    }
  }
  for (int m = 16; m; m >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, m);
  if (lane == 0) out[i] = w < int64_t(vocab) ? acc * scale : nan;
}

}  // namespace

void embedding(const Tokens& k, const Mat& table, uint64_t vocab, uint64_t dim, float scale, const Scales& s,
               const Mat& out, cudaStream_t stream) {
  if (!k.rows) return;
  with_types(table.type, out.type, [&](auto* pt, auto* po) {
    using T = std::remove_pointer_t<decltype(pt)>;
    using O = std::remove_pointer_t<decltype(po)>;
    const T* w = static_cast<const T*>(table.data);
    O* y = static_cast<O*>(const_cast<void*>(out.data));
    with_width<T>(table, vocab, out, k.rows, dim, [&](auto width) {
      constexpr int VE = decltype(width)::value;
      const uint64_t pieces = dim / VE;
      if (k.per_row == 1) {
        const uint64_t total = k.rows * pieces;
        lookup_kernel<T, O, VE><<<blocks_for(total, kThreads * 4), kThreads, 0, stream>>>(
            k, w, table.stride, vocab, uint32_t(pieces), FastDiv(uint32_t(pieces)), total, scale, s, y, out.stride,
            kNaN);
        return;
      }
      int lg = 0;
      while (lg < 5 && (1ull << lg) < pieces) ++lg;
      const uint32_t tiles = blocks_for(pieces, 1u << lg);
      // Few rows leave the card idle: their tokens are split over more groups
      // of the block, down to 8 tokens a group.
      int ls = 0;
      while (lg + ls < 8 && k.rows * tiles << (lg + ls) < 148 * 1024 && k.per_row >> (ls + 1) >= 8) ++ls;
      const dim3 grid(blocks_for(k.rows, kThreads >> (lg + ls)), tiles);
      const auto go = [&](auto kk) {
        constexpr int K = decltype(kk)::value;
        const auto kernel = s.data ? bag_kernel<T, O, VE, K, true> : bag_kernel<T, O, VE, K, false>;
        kernel<<<grid, kThreads, 0, stream>>>(k, w, table.stride, uint32_t(vocab), uint32_t(dim), scale, s, y,
                                              out.stride, lg, ls, kNaN);
      };
      if (lg >= 3) go(std::integral_constant<int, 1>());
      else if (lg == 2) go(std::integral_constant<int, 2>());
      else if (lg == 1) go(std::integral_constant<int, 4>());
      else go(std::integral_constant<int, 8>());
    });
  });
  XGBB_CUDA(cudaGetLastError());
}

void embedding_scale_backward(const Mat& grad, const Tokens& k, const Mat& table, uint64_t vocab, uint64_t dim,
                              float scale, float* out, cudaStream_t stream) {
  const uint64_t total = k.rows * k.per_row;
  if (!total) return;
  with_types(table.type, grad.type, [&](auto* pt, auto* po) {
    using T = std::remove_pointer_t<decltype(pt)>;
    using O = std::remove_pointer_t<decltype(po)>;
    with_width<T>(table, vocab, grad, k.rows, dim, [&](auto width) {
      scale_grad_kernel<T, O, decltype(width)::value><<<blocks_for(total, kThreads / 32), kThreads, 0, stream>>>(
          static_cast<const O*>(grad.data), grad.stride, k, static_cast<const T*>(table.data), table.stride, vocab,
          uint32_t(dim), scale, out, total, kNaN);
    });
  });
  XGBB_CUDA(cudaGetLastError());
}

}  // namespace xgbb::nn
