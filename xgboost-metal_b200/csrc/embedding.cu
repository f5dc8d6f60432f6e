// Embedding lookup with scaling, one token or a summed bag of tokens a row,
// and the gradient of the tokens' scales. The table's gradient is in
// embedding_grad.cu.
//
//   y[r] = a * sum_t s[r][t] W[k[r][t]],    ds[r][t] = a * <dy[r], W[k[r][t]]>
//
// A token below 0 is missing and adds nothing, whatever its scale holds. A
// token past the table makes its row's result NaN: nothing is read for it.
// Sums are float32 in a fixed order, and are rounded once, when written.
#include <cooperative_groups.h>

#include <algorithm>

#include "nn_device.cuh"

namespace xgbb::nn {

size_t type_size(int type) { return type == kF32 || type == kI32 ? 4 : type == kI64 ? 8 : 2; }

namespace {

constexpr int kThreads = 256;
const float kNaN = __builtin_nanf("");

// One token a row: a copy with a factor. Flat over the (row, piece) pairs, so
// that neighbouring threads move neighbouring pieces, four pieces in flight a
// thread. Bound by device memory: 8191 rows of 2048 bf16 take 12.0 us, 5.6 TB/s.
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
// each. SPLIT: S = 2^ls such groups share a row's tokens, a contiguous span each,
// and add their sums up in shared memory, first span first; and the blocks of a
// cluster, where there are several, share the tokens in the same way. A group
// reads its tokens K to a lane, a step ahead, and passes them on by shuffles,
// eight gathers in flight; a step without a missing token is summed without a
// look at each.
// Bound by instructions, then by the L1 cache's lines: 262144 bags of 100 x 64
// bf16 gather 3.36 GB in 269 us (12.5 TB/s, 72 % of the issue slots), where what
// they read and write once is 175 MB. 64 registers, so that an SM holds 1024
// threads: at 128 it took 493 us. Seven bags of 2000 x 33 f32 take 20.6 us in
// blocks alone and 5.0 in clusters of eight.
template <class T, class O, int VE, int K, bool SCALED, bool SPLIT>
__global__ void __launch_bounds__(kThreads, (K > 1 ? 2 : VE * sizeof(T) == 16 ? 4 : 3))
    bag_kernel(Tokens k, const T* __restrict__ table, int64_t table_stride, uint32_t vocab, uint32_t dim,
               float scale, Scales s, O* __restrict__ out, int64_t out_stride, int lg, int ls, float nan) {
  constexpr int U = 8;
  __shared__ float part[SPLIT ? kThreads * VE : 1];
  const auto cluster = cooperative_groups::this_cluster();
  const uint32_t blocks = SPLIT ? cluster.num_blocks() : 1, rank = SPLIT ? cluster.block_rank() : 0;
  const uint32_t G = 1u << lg, lane = threadIdx.x & (G - 1), group = threadIdx.x >> lg;
  if (!SPLIT) ls = 0;
  const uint32_t S = 1u << ls, span = group & (S - 1);
  const uint64_t row = uint64_t(blockIdx.x / blocks) * (kThreads >> (lg + ls)) + (group >> ls);
  const uint32_t col = (blockIdx.y * G + lane) * VE;
  const bool wide = k.type == kI64;
  const uint32_t count = uint32_t(k.per_row), per = (count + S * blocks - 1) / (S * blocks);
  const uint32_t begin = uint32_t(min(uint64_t(count), uint64_t(per) * (rank * S + span))), end = row < k.rows ? min(count, begin + per) : 0;
  // Lanes past the last column read the last piece, and write nothing.
  const T* const columns = table + min(col, dim - VE);
  const char* const tokens = static_cast<const char*>(k.data) + int64_t(row) * k.stride_row * (wide ? 8 : 4);
  const float* const scales = SCALED && (!SPLIT || s.data) ? s.data + int64_t(row) * s.stride_row : nullptr;
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
      if (SCALED) next_f[i] = SPLIT && !scales ? 1.0f : next[i] >= 0 ? scales[int64_t(t) * s.stride_col] : 0.0f;
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
  if (SPLIT && S > 1) {
#pragma unroll
    for (int e = 0; e < VE; ++e) part[threadIdx.x * VE + e] = sum[e];
    __syncthreads();
    if (span == 0)
      for (uint32_t q = 1; q < S; ++q)
#pragma unroll
        for (int e = 0; e < VE; ++e) sum[e] += part[(threadIdx.x + (q << lg)) * VE + e];
  }
  if (SPLIT && blocks > 1) {
    if (span == 0)
#pragma unroll
      for (int e = 0; e < VE; ++e) part[threadIdx.x * VE + e] = sum[e];
    cluster.sync();
    if (rank == 0 && span == 0)
      for (uint32_t q = 1; q < blocks; ++q) {
        const float* other = cluster.map_shared_rank(part, q);
#pragma unroll
        for (int e = 0; e < VE; ++e) sum[e] += other[threadIdx.x * VE + e];
      }
    cluster.sync();  // the other blocks' memory is read until here
    if (rank) return;
  }
  if (span == 0 && row < k.rows && col < dim) {
#pragma unroll
    for (int e = 0; e < VE; ++e) sum[e] *= scale;
    store_global<O, VE>(out + int64_t(row) * out_stride + col, sum);
  }
}

// The scales' gradient: 2^lg lanes own a row's columns, VE values each in as many
// tiles as it takes, and take a span of the row's tokens, eight at a time. The
// eight products are reduced together: each shuffle halves how many a lane holds,
// until the lanes hold different tokens' results. Bound by instructions: 20000
// bags of 100 x 64 bf16 gather 256 MB in 46 us; a warp a token took 96.
template <class T, class O, int VE>
__global__ void __launch_bounds__(kThreads, 3)
    scale_grad_kernel(const O* __restrict__ grad, int64_t grad_stride, Tokens k, const T* __restrict__ table,
                      int64_t table_stride, uint32_t vocab, uint32_t dim, float scale, float* __restrict__ out,
                      uint32_t span, FastDiv spans, uint64_t groups, int lg, float nan) {
  constexpr int U = 8;
  const uint32_t G = 1u << lg, lane = threadIdx.x & (G - 1);
  const uint64_t group = (uint64_t(blockIdx.x) * kThreads + threadIdx.x) >> lg;
  const bool here = group < groups;
  const uint32_t row = here ? spans.div(uint32_t(group)) : 0;
  const uint32_t begin = here ? (uint32_t(group) - row * spans.d) * span : 0;
  const uint32_t end = here ? uint32_t(min(k.per_row, uint64_t(begin) + span)) : 0;
  const bool wide = k.type == kI64;
  const char* const tokens = static_cast<const char*>(k.data) + int64_t(row) * k.stride_row * (wide ? 8 : 4);
  const O* const g_row = grad + int64_t(row) * grad_stride;
  for (uint32_t t0 = begin; __any_sync(0xffffffffu, t0 < end); t0 += U) {
    int token[U];  // -1: missing, past the table, or past the span
    if (wide) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t w =
            t0 + u < end ? reinterpret_cast<const int64_t*>(tokens)[int64_t(t0 + u) * k.stride_col] : -1;
        token[u] = uint64_t(w) < vocab ? int(w) : -1;
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int w = t0 + u < end ? reinterpret_cast<const int*>(tokens)[int64_t(t0 + u) * k.stride_col] : -1;
        token[u] = uint32_t(w) < vocab ? w : -1;
      }
    }
    Sum<float, 2> two[VE % 2 == 0 ? U : 1];
    float dot[U] = {};
    if constexpr (VE % 2 == 0)
#pragma unroll
      for (int u = 0; u < U; ++u) two[u].clear();
    for (uint32_t c = lane * VE; c < dim; c += G * VE) {
      const auto g = load<O, VE>(g_row + c);
      Pack<T, VE> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (token[u] >= 0) v[u] = load<T, VE>(table + token[u] * table_stride + c);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (token[u] >= 0) {
          if constexpr (VE % 2 == 0) {
#pragma unroll
            for (int e = 0; e < VE / 2; ++e)
              two[u].two[0] = fma2(pair_of<O, VE>(g, e), pair_of<T, VE>(v[u], e), two[u].two[0]);
          } else {
            dot[u] = fmaf(g.f(0), v[u].f(0), dot[u]);
          }
        }
    }
    if constexpr (VE % 2 == 0)
#pragma unroll
      for (int u = 0; u < U; ++u) dot[u] = two[u].two[0].x + two[u].two[0].y;
    uint32_t m = G >> 1;
#pragma unroll
    for (int n = U / 2; n >= 1; n >>= 1)
      if (m) {
        const bool upper = lane & m;
#pragma unroll
        for (int i = 0; i < n; ++i)
          dot[i] = (upper ? dot[i + n] : dot[i]) + __shfl_xor_sync(0xffffffffu, upper ? dot[i] : dot[i + n], m);
        m >>= 1;
      }
    for (; m; m >>= 1) dot[0] += __shfl_xor_sync(0xffffffffu, dot[0], m);
    // Lane l holds tokens l (8 / G) on, or token l / (G / 8).
    const uint32_t first = lg < 3 ? lane << (3 - lg) : lane >> (lg - 3);
    if (lg > 3 && (lane & ((1u << (lg - 3)) - 1))) continue;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (i >= (lg < 3 ? 8 >> lg : 1) || t0 + first + i >= end) break;
      const uint64_t at = uint64_t(row) * k.per_row + t0 + first + i;
      const int64_t w = load_token(tokens, wide, (t0 + first + i) * k.stride_col);
      out[at] = w < int64_t(vocab) ? dot[i] * scale : nan;
    }
  }
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
      const int lg = lanes_log2(pieces);
      const uint32_t tiles = blocks_for(pieces, 1u << lg);
      // Few rows leave the card idle: their tokens are split over more groups
      // of the block, down to 8 tokens a group.
      int ls = 0;
      while (lg + ls < 8 && k.rows * tiles << (lg + ls) < 148 * 1024 && k.per_row >> (ls + 1) >= 8) ++ls;
      // And over clusters, where a group still has over 16 and the clusters' blocks
      // are eight an SM at most, two to four turns of what an SM holds of them.
      // (7 bags of 2000 x 33: 20.6 us without, 5.0 in clusters; 100000 bags of 50 x 8
      // in clusters: 216 us for 33.)
      const uint64_t blocks = blocks_for(k.rows, kThreads >> (lg + ls));
      const unsigned cluster = ls && k.per_row >> ls > 16 && blocks * tiles * 8 <= 148 * 8 ? 8 : 1;
      const dim3 grid(unsigned(blocks * cluster), tiles);
      const auto go = [&](auto kk) {
        constexpr int K = decltype(kk)::value;
        const auto kernel = ls ? bag_kernel<T, O, VE, K, true, true>
                               : s.data ? bag_kernel<T, O, VE, K, true, false> : bag_kernel<T, O, VE, K, false, false>;
        cudaLaunchAttribute attribute{};
        attribute.id = cudaLaunchAttributeClusterDimension;
        attribute.val.clusterDim = {cluster, 1, 1};
        cudaLaunchConfig_t config{};
        config.gridDim = grid;
        config.blockDim = dim3(kThreads);
        config.stream = stream;
        config.attrs = &attribute;
        config.numAttrs = cluster > 1;
        XGBB_CUDA(cudaLaunchKernelEx(&config, kernel, k, w, table.stride, uint32_t(vocab), uint32_t(dim), scale, s, y,
                                     out.stride, lg, ls, kNaN));
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
      constexpr int VE = decltype(width)::value;
      int lg = 0;
      while (lg < 5 && (VE << lg) < int(std::min<uint64_t>(dim, 1024))) ++lg;
      // A span of eight tokens where that is what fills the card, longer ones where there are more.
      uint64_t span = ((total << lg) / (148 * 1024) + 7) / 8 * 8;
      span = std::min<uint64_t>(std::max<uint64_t>(span, 8), (k.per_row + 7) / 8 * 8);
      const uint64_t spans = (k.per_row + span - 1) / span, groups = k.rows * spans;
      scale_grad_kernel<T, O, VE><<<blocks_for(groups, kThreads >> lg), kThreads, 0, stream>>>(
          static_cast<const O*>(grad.data), grad.stride, k, static_cast<const T*>(table.data), table.stride,
          uint32_t(vocab), uint32_t(dim), scale, out, uint32_t(span), FastDiv(uint32_t(spans)), groups, lg, kNaN);
    });
  });
  XGBB_CUDA(cudaGetLastError());
}

}  // namespace xgbb::nn
