// The table's gradient of an embedding lookup, by sorted tokens:
//
//   dW[v] (+)= a * sum over the (r, t) with k[r][t] == v of s[r][t] dy[r]
//
// The (token, position) pairs are sorted by token with a stable radix sort,
// so that a token's positions lie side by side and in their own order. Equal
// shares of the sorted list are then summed, and a token that crosses from
// one share into the next is joined from the shares' partial sums. Every sum
// has a fixed order: equal inputs give equal bits, and a frequent token costs
// no more than many rare ones. Sums are float32, rounded once when written.
#include <algorithm>

#include "nn_device.cuh"

namespace xgbb::nn {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kItems = 16;                  // entries a thread holds of a sort tile
constexpr int kTile = kThreads * kItems;    // 4096
constexpr int kDigits = 256;
constexpr int kSortBlocks = 592;            // most blocks of a sort pass: 4 an SM
constexpr uint32_t kShare = 256;            // sorted entries that one group of lanes sums

uint32_t sort_blocks(uint64_t n) {
  const uint64_t tiles = (n + kTile - 1) / kTile;
  return uint32_t(tiles < kSortBlocks ? tiles : kSortBlocks);
}

// Where the parts of the workspace lie.
struct Layout {
  size_t keys[2], values[2], hist, totals, head, tail, bytes;
  Layout(uint64_t n, uint64_t dim) {
    size_t at = 0;
    const auto take = [&](size_t b) {
      const size_t p = at;
      at += (b + 255) / 256 * 256;
      return p;
    };
    for (int i = 0; i < 2; ++i) {
      keys[i] = take(n * 4);
      values[i] = take(n * 4);
    }
    hist = take(size_t(kDigits) * sort_blocks(n) * 4);
    totals = take(kDigits * 4);
    const uint64_t shares = (n + kShare - 1) / kShare;
    head = take(shares * dim * 4);
    tail = take(shares * dim * 4);
    bytes = at;
  }
};

// The sort's entries: pass 0 reads the tokens themselves (a token that is
// missing or past the table gets the key `vocab`, after all others; its value
// is its position in [rows][per_row]), later passes what the pass before
// wrote.
struct Source {
  Tokens k;
  FastDiv per_row;
  uint32_t vocab;
  const uint32_t* keys;
  const uint32_t* values;
  __device__ __forceinline__ uint32_t key(uint32_t i) const {
    if (keys) return keys[i];
    const uint32_t r = per_row.div(i), t = i - r * per_row.d;
    const int64_t w = load_token(k.data, k.type == kI64, int64_t(r) * k.stride_row + int64_t(t) * k.stride_col);
    return w >= 0 && w < int64_t(vocab) ? uint32_t(w) : vocab;
  }
  __device__ __forceinline__ uint32_t value(uint32_t i) const { return values ? values[i] : i; }
};

// Block b sorts the tiles [b * per, (b + 1) * per). hist[digit][block].
__global__ void __launch_bounds__(kThreads)
    sort_hist_kernel(Source src, uint32_t n, uint32_t per, int shift, uint32_t* __restrict__ hist) {
  __shared__ uint32_t count[kDigits];
  count[threadIdx.x] = 0;
  __syncthreads();
  const uint64_t begin = uint64_t(blockIdx.x) * per * kTile;
  const uint64_t end = min(uint64_t(n), begin + uint64_t(per) * kTile);
  for (uint64_t i = begin + threadIdx.x; i < end; i += kThreads)
    atomicAdd(&count[(src.key(uint32_t(i)) >> shift) & (kDigits - 1)], 1u);
  __syncthreads();
  hist[threadIdx.x * gridDim.x + blockIdx.x] = count[threadIdx.x];
}

// Exclusive sum of one value a thread over the block; `total` gets the sum.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* warp_sums, uint32_t& total) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, m);
    if (lane >= uint32_t(m)) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < int(warp)) before += warp_sums[w];
    total += warp_sums[w];
  }
  return before + x - v;
}

// Block d: the exclusive sums of digit d's counts over the sort's blocks, in
// place, and their total.
__global__ void __launch_bounds__(kThreads)
    sort_scan_kernel(uint32_t* __restrict__ hist, uint32_t blocks, uint32_t* __restrict__ totals) {
  __shared__ uint32_t warp_sums[kWarps];
  uint32_t* h = hist + size_t(blockIdx.x) * blocks;
  uint32_t before = 0;
  for (uint32_t b = 0; b < blocks; b += kThreads) {
    const uint32_t i = b + threadIdx.x;
    const uint32_t v = i < blocks ? h[i] : 0;
    uint32_t total;
    const uint32_t x = block_scan(v, warp_sums, total);
    if (i < blocks) h[i] = before + x;
    before += total;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = before;
}

// Ranks a tile's entries by digit, stably: warp w holds entries [512 w, 512
// w + 512) of it, 32 at a time; the lanes that share a digit find each other
// by ballots over its 8 bits (warp-level multisplit; Ashkiani et al., "GPU
// multisplit", 2016), and each warp counts its own digits. The tile is put in
// order in shared memory and leaves it in runs of equal digits.
__global__ void __launch_bounds__(kThreads)
    sort_scatter_kernel(Source src, uint32_t n, uint32_t per, int shift, const uint32_t* __restrict__ hist,
                        const uint32_t* __restrict__ totals, uint32_t* __restrict__ keys_out,
                        uint32_t* __restrict__ values_out) {
  __shared__ uint32_t next[kDigits];           // where the digit's next entry of this block goes
  __shared__ uint32_t local[kDigits];          // where the digit begins in the ordered tile
  __shared__ uint32_t count[kWarps][kDigits];  // the warp's entries of the digit, then those of the warps before it
  __shared__ uint32_t warp_sums[kWarps];
  __shared__ uint32_t keys[kTile], values[kTile];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = threadIdx.x;
  uint32_t unused;
  next[d] = block_scan(totals[d], warp_sums, unused) + hist[d * gridDim.x + blockIdx.x];
  const uint64_t first = uint64_t(blockIdx.x) * per;
  for (uint32_t tile = 0; tile < per; ++tile) {
    const uint64_t begin = (first + tile) * kTile;
    if (begin >= n) break;
    const uint32_t here = uint32_t(min(uint64_t(kTile), n - begin));
#pragma unroll
    for (int w = 0; w < kWarps; ++w) count[w][d] = 0;
    __syncthreads();
    uint32_t key[kItems], value[kItems], rank[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const uint32_t at = warp * (kItems * 32) + i * 32 + lane;
      key[i] = at < here ? src.key(uint32_t(begin) + at) : 0xffffffffu;
      value[i] = at < here ? src.value(uint32_t(begin) + at) : 0;
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const uint32_t at = warp * (kItems * 32) + i * 32 + lane;
      const uint32_t digit = (key[i] >> shift) & (kDigits - 1);
      uint32_t same = __ballot_sync(0xffffffffu, at < here);
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        const uint32_t set = __ballot_sync(0xffffffffu, (digit >> b) & 1u);
        same &= (digit >> b) & 1u ? set : ~set;
      }
      if (at < here) rank[i] = count[warp][digit] + __popc(same & ((1u << lane) - 1));
      __syncwarp();
      if (at < here && (same >> lane) == 1u) count[warp][digit] += __popc(same);
      __syncwarp();
    }
    __syncthreads();
    uint32_t total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const uint32_t c = count[w][d];
      count[w][d] = total;
      total += c;
    }
    local[d] = block_scan(total, warp_sums, unused);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const uint32_t at = warp * (kItems * 32) + i * 32 + lane;
      if (at < here) {
        const uint32_t digit = (key[i] >> shift) & (kDigits - 1);
        const uint32_t p = local[digit] + count[warp][digit] + rank[i];
        keys[p] = key[i];
        values[p] = value[i];
      }
    }
    __syncthreads();
    for (uint32_t p = threadIdx.x; p < here; p += kThreads) {
      const uint32_t digit = (keys[p] >> shift) & (kDigits - 1);
      const uint32_t to = next[digit] + (p - local[digit]);
      keys_out[to] = keys[p];
      values_out[to] = values[p];
    }
    __syncthreads();
    next[d] += total;
  }
}

// Groups of G = 2^lg lanes own VE columns a lane (blockIdx.y: the tile of
// columns) and sum kShare sorted entries each, eight gathers in flight. A
// token that lies in one share whole goes to its row; the sum of one that
// came in from the share before goes to head[share], of one that goes on into
// the next to tail[share] (a share inside one token has its sum in head).
template <class T, class O, int VE>
__global__ void __launch_bounds__(kThreads)
    share_sum_kernel(const T* __restrict__ grad, int64_t grad_stride, const uint32_t* __restrict__ keys,
                     const uint32_t* __restrict__ values, uint32_t n, uint32_t vocab, FastDiv per_row, Scales s,
                     float scale, uint32_t dim, O* __restrict__ out, int64_t out_stride, bool accumulate,
                     float* __restrict__ head, float* __restrict__ tail, int lg) {
  constexpr int U = 8;
  const uint32_t G = 1u << lg, lane = threadIdx.x & (G - 1);
  const uint64_t share = (uint64_t(blockIdx.x) * kThreads + threadIdx.x) >> lg;
  const uint32_t col = (blockIdx.y * G + lane) * VE;
  const uint64_t begin = share * kShare;
  const uint32_t here = begin < n ? uint32_t(min(uint64_t(kShare), n - begin)) : 0;
  const uint32_t before = here && begin ? keys[begin - 1] : 0xffffffffu;
  const uint32_t after = here && begin + here < n ? keys[begin + here] : 0xffffffffu;
  float acc[VE] = {};
  uint32_t current = 0xffffffffu;
  bool from_before = false;
  const auto finish = [&](bool goes_on) {  // the sum of token `current` is whole, or goes on
    if (current < vocab && col < dim) {
      if (from_before || goes_on) {
        float* to = (from_before ? head : tail) + share * dim + col;
        store<float, VE>(to, acc);
      } else {
        O* to = out + int64_t(current) * out_stride + col;
        float y[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) y[e] = acc[e] * scale;
        if (accumulate) {
          const auto old = load<O, VE>(to);
#pragma unroll
          for (int e = 0; e < VE; ++e) y[e] += old.f(e);
        }
        store<O, VE>(to, y);
      }
    }
  };
  for (uint32_t j0 = 0; __any_sync(0xffffffffu, j0 < here); j0 += U) {
    // Lane q of a group (of 8 lanes or more) reads entry q; narrower groups
    // read all eight in each lane.
    uint32_t key[U], row[U];
    float f[U];
    Pack<T, VE> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = j0 + u < here;
      key[u] = in ? keys[begin + j0 + u] : 0xffffffffu;
      const uint32_t value = in ? values[begin + j0 + u] : 0;
      row[u] = per_row.div(value);
      f[u] = 1.0f;
      if (s.data && key[u] < vocab)
        f[u] = s.data[int64_t(row[u]) * s.stride_row + int64_t(value - row[u] * per_row.d) * s.stride_col];
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (key[u] < vocab && col < dim) v[u] = load<T, VE>(grad + int64_t(row[u]) * grad_stride + col);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (key[u] >= vocab) continue;
      if (key[u] != current) {
        finish(false);
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[e] = 0.0f;
        current = key[u];
        from_before = j0 + u == 0 && key[u] == before;
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[e] = fmaf(f[u], v[u].f(e), acc[e]);
    }
  }
  finish(here && current == after);
}

// Block x: the token that begins in share x and goes on after it, if there is
// one: its partial sums, joined over the block's groups in a fixed order.
template <class O, int VE>
__global__ void __launch_bounds__(kThreads)
    join_kernel(const uint32_t* __restrict__ keys, uint32_t n, uint32_t vocab, float scale, uint32_t dim,
                O* __restrict__ out, int64_t out_stride, bool accumulate, const float* __restrict__ head,
                const float* __restrict__ tail, int lg) {
  __shared__ float part[kThreads * VE];
  const uint32_t share = blockIdx.x;
  const uint64_t begin = uint64_t(share) * kShare, end = begin + kShare;
  if (end >= n) return;
  const uint32_t token = keys[end - 1];
  if (token >= vocab || keys[end] != token) return;
  if (begin && keys[begin] == token && keys[begin - 1] == token) return;  // it began before
  uint32_t lo = uint32_t(end), hi = n;  // the first entry of a later token
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (keys[mid] == token) lo = mid + 1;
    else hi = mid;
  }
  const uint32_t last = (lo - 1) / kShare;
  const uint32_t G = 1u << lg, lane = threadIdx.x & (G - 1), group = threadIdx.x >> lg, groups = kThreads >> lg;
  const uint32_t col = (blockIdx.y * G + lane) * VE;
  float acc[VE] = {};
  if (col < dim) {
    if (group == 0) {
      const auto v = load<float, VE>(tail + uint64_t(share) * dim + col);
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[e] = v.f(e);
    }
    for (uint32_t q = share + 1 + group; q <= last; q += groups) {
      const auto v = load<float, VE>(head + uint64_t(q) * dim + col);
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[e] += v.f(e);
    }
  }
#pragma unroll
  for (int e = 0; e < VE; ++e) part[threadIdx.x * VE + e] = acc[e];
  __syncthreads();
  if (group != 0 || col >= dim) return;
  for (uint32_t g = 1; g < groups; ++g)
#pragma unroll
    for (int e = 0; e < VE; ++e) acc[e] += part[(threadIdx.x + (g << lg)) * VE + e];
  O* to = out + int64_t(token) * out_stride + col;
#pragma unroll
  for (int e = 0; e < VE; ++e) acc[e] *= scale;
  if (accumulate) {
    const auto old = load<O, VE>(to);
#pragma unroll
    for (int e = 0; e < VE; ++e) acc[e] += old.f(e);
  }
  store<O, VE>(to, acc);
}

// Zeros into rows of `dim` values.
template <class O, int VE>
__global__ void __launch_bounds__(kThreads)
    zero_rows_kernel(O* __restrict__ out, int64_t stride, uint32_t pieces, FastDiv div, uint64_t total) {
  const float zero[VE] = {};
  for (uint64_t i = uint64_t(blockIdx.x) * kThreads + threadIdx.x; i < total;
       i += uint64_t(gridDim.x) * kThreads) {
    const uint64_t row = total <= 0xffffffffull ? div.div(uint32_t(i)) : i / pieces;
    store<O, VE>(out + int64_t(row) * stride + (i - row * pieces) * VE, zero);
  }
}

}  // namespace

size_t embedding_backward_workspace(const Tokens& k, uint64_t, uint64_t dim) {
  return Layout(k.rows * k.per_row, dim).bytes;
}

void embedding_backward(const Mat& grad, const Tokens& k, uint64_t vocab, uint64_t dim, float scale,
                        const Scales& s, const Mat& out, bool accumulate, void* workspace,
                        cudaStream_t stream) {
  const uint32_t n = uint32_t(k.rows * k.per_row);
  const Layout at(n, dim);
  char* w = static_cast<char*>(workspace);
  const auto u32 = [&](size_t offset) { return reinterpret_cast<uint32_t*>(w + offset); };
  int from = 0;
  if (n) {
    const uint32_t blocks = sort_blocks(n), tiles = blocks_for(n, kTile), per = (tiles + blocks - 1) / blocks;
    const uint32_t grid = (tiles + per - 1) / per;
    for (int shift = 0; shift < 32 && (shift == 0 || vocab >> shift); shift += 8) {
      const Source src{k, FastDiv(uint32_t(k.per_row)), uint32_t(vocab), shift ? u32(at.keys[from]) : nullptr,
                       shift ? u32(at.values[from]) : nullptr};
      const int to = shift ? from ^ 1 : 0;
      sort_hist_kernel<<<grid, kThreads, 0, stream>>>(src, n, per, shift, u32(at.hist));
      sort_scan_kernel<<<kDigits, kThreads, 0, stream>>>(u32(at.hist), grid, u32(at.totals));
      sort_scatter_kernel<<<grid, kThreads, 0, stream>>>(src, n, per, shift, u32(at.hist), u32(at.totals),
                                                         u32(at.keys[to]), u32(at.values[to]));
      from = to;
    }
  }
  with_types(grad.type, out.type, [&](auto* pt, auto* po) {
    using T = std::remove_pointer_t<decltype(pt)>;
    using O = std::remove_pointer_t<decltype(po)>;
    O* y = static_cast<O*>(const_cast<void*>(out.data));
    with_width<T>(grad, k.rows, out, vocab, dim, [&](auto width) {
      constexpr int VE = decltype(width)::value;
      const uint64_t pieces = dim / VE;
      if (!accumulate) {
        const uint64_t total = vocab * pieces;
        zero_rows_kernel<O, VE><<<unsigned(std::min<uint64_t>(blocks_for(total, kThreads), 148 * 8)), kThreads, 0,
                                  stream>>>(y, out.stride, uint32_t(pieces), FastDiv(uint32_t(pieces)), total);
      }
      if (!n) return;
      int lg = 0;
      while (lg < 5 && (1ull << lg) < pieces) ++lg;
      const uint32_t column_tiles = blocks_for(pieces, 1u << lg), shares = blocks_for(n, kShare);
      float* head = reinterpret_cast<float*>(w + at.head);
      float* tail = reinterpret_cast<float*>(w + at.tail);
      share_sum_kernel<T, O, VE><<<dim3(blocks_for(shares, kThreads >> lg), column_tiles), kThreads, 0, stream>>>(
          static_cast<const T*>(grad.data), grad.stride, u32(at.keys[from]), u32(at.values[from]), n,
          uint32_t(vocab), FastDiv(uint32_t(k.per_row)), s, scale, uint32_t(dim), y, out.stride, accumulate, head,
          tail, lg);
      if (shares > 1)
        join_kernel<O, VE><<<dim3(shares, column_tiles), kThreads, 0, stream>>>(
            u32(at.keys[from]), n, uint32_t(vocab), scale, uint32_t(dim), y, out.stride, accumulate, head, tail, lg);
    });
  });
  XGBB_CUDA(cudaGetLastError());
}

}  // namespace xgbb::nn
