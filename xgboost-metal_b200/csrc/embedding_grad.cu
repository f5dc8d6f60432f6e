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

// Few tokens, in one launch: block (x, y) owns the table's rows [x span, x span
// + span) in a tile of columns. It picks its rows' tokens out of all n, sorts
// them, (row << kShift | position), in shared memory, zeroes the rows that have
// none, and sums the others: groups of 2^lg lanes take equal shares of the
// sorted list, and what crosses shares is joined through shared memory, in the
// shares' order. No row is written by two blocks. step: the distance of one
// token from the next where it is the same for all, else 0.
constexpr int kFewThreads = 512;
constexpr int kShift = 15;
constexpr uint32_t kFewTokens = 1u << kShift;

template <class T, class O, int VE, bool SCALED>
__global__ void __launch_bounds__(kFewThreads, 2)
    few_kernel(const T* __restrict__ grad, int64_t grad_stride, Tokens k, int64_t step, FastDiv per_row, uint32_t n,
               uint32_t vocab, uint32_t span, Scales s, float scale, uint32_t dim, O* __restrict__ out,
               int64_t out_stride, bool accumulate, int lg) {
  constexpr int U = 4, kBatch = 8;
  extern __shared__ __align__(16) uint32_t space[];
  __shared__ uint32_t total;
  __shared__ int32_t first_row[kFewThreads], last_row[kFewThreads];  // of a group's share; -1: none
  float* head = reinterpret_cast<float*>(space);  // [2][threads][VE]: sums that came in, sums that go on
  float* tail = head + kFewThreads * VE;
  uint32_t* present = space + 2 * kFewThreads * VE;  // a bit a row
  uint32_t* list = present + (span + 31) / 32;
  const uint32_t lane = threadIdx.x & 31;
  const uint32_t row0 = blockIdx.x * span, rows_here = min(span, vocab - row0);

  // The rows' tokens, in any order: all entries differ, so the sort gives one.
  for (uint32_t i = threadIdx.x; i < (span + 31) / 32; i += kFewThreads) present[i] = 0;
  if (threadIdx.x == 0) total = 0;
  __syncthreads();
  const auto where = [&](uint32_t i) {
    if (step) return int64_t(i) * step;
    const uint32_t r = per_row.div(i);
    return int64_t(r) * k.stride_row + int64_t(i - r * per_row.d) * k.stride_col;
  };
  for (uint32_t i0 = threadIdx.x - lane; i0 < n; i0 += kFewThreads * kBatch) {
    uint64_t local[kBatch];  // past rows_here: another block's token, or nobody's
    if (k.type == kI64) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const uint32_t at = i0 + i * kFewThreads + lane;
        local[i] = at < n ? uint64_t(static_cast<const int64_t*>(k.data)[where(at)]) : ~0ull;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const uint32_t at = i0 + i * kFewThreads + lane;
        local[i] = at < n ? uint64_t(int64_t(static_cast<const int32_t*>(k.data)[where(at)])) : ~0ull;
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const bool mine = local[i] - row0 < rows_here;
      const uint32_t votes = __ballot_sync(0xffffffffu, mine);
      if (!votes) continue;
      uint32_t base = 0;
      if (lane == 0) base = atomicAdd(&total, uint32_t(__popc(votes)));
      base = __shfl_sync(0xffffffffu, base, 0);
      if (mine) {
        const uint32_t r = uint32_t(local[i] - row0);
        list[base + __popc(votes & ((1u << lane) - 1))] = r << kShift | (i0 + i * kFewThreads + lane);
        atomicOr(&present[r >> 5], 1u << (r & 31));
      }
    }
  }
  __syncthreads();

  const uint32_t G = 1u << lg, me = threadIdx.x & (G - 1), group = threadIdx.x >> lg, groups = kFewThreads >> lg;
  const uint32_t col = (blockIdx.y * G + me) * VE;
  O* const mine_out = out + int64_t(row0) * out_stride + col;
  const auto zero_absent = [&] {
    const float zero[VE] = {};
    if (!accumulate && col < dim)
      for (uint32_t r = group; r < rows_here; r += groups)
        if (!(present[r >> 5] >> (r & 31) & 1)) store<O, VE>(mine_out + int64_t(r) * out_stride, zero);
  };
  // Half of the blocks zero first and half last, so that reading and writing
  // overlap on an SM that holds two.
  const bool zero_first = (blockIdx.y * gridDim.x + blockIdx.x) * 2 < gridDim.x * gridDim.y;
  if (zero_first) zero_absent();

  // By counting the smaller entries where they are few, else a bitonic network
  // whose comparators all point upwards (then what lies past the end need not
  // exist). A warp's comparators of a span of 64 or less touch its own 64
  // entries alone.
  const uint32_t count = total;
  if (count <= kFewThreads) {
    uint32_t mine = 0, rank = 0;
    if (threadIdx.x < count) {
      mine = list[threadIdx.x];
#pragma unroll 8
      for (uint32_t j = 0; j < count; ++j) rank += list[j] < mine;
    }
    __syncthreads();
    if (threadIdx.x < count) list[rank] = mine;
    __syncthreads();
  } else {
    int bits = 32 - __clz(count - 1);
    const uint32_t pairs = 1u << (bits - 1);
    const auto order = [&](uint32_t i, uint32_t j) {
      if (j < count) {
        const uint32_t a = list[i], b = list[j];
        if (a > b) {
          list[i] = b;
          list[j] = a;
        }
      }
    };
    for (int block = 1; block <= bits; ++block) {  // runs of 2^block entries
      for (uint32_t p = threadIdx.x; p < pairs; p += kFewThreads) {
        const uint32_t i = p >> (block - 1) << block | (p & ((1u << (block - 1)) - 1));
        order(i, i ^ ((1u << block) - 1));
      }
      for (int half = block - 2; half >= 0; --half) {
        if (half >= 5) __syncthreads();
        else __syncwarp();
        for (uint32_t p = threadIdx.x; p < pairs; p += kFewThreads) {
          const uint32_t i = p >> half << (half + 1) | (p & ((1u << half) - 1));
          order(i, i + (1u << half));
        }
      }
      if (block >= 6) __syncthreads();
      else __syncwarp();
    }
    __syncthreads();
  }

  const auto write = [&](int32_t local, const float(&sum)[VE]) {
    if (col >= dim) return;
    O* to = mine_out + int64_t(local) * out_stride;
    float y[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) y[e] = sum[e] * scale;
    if (accumulate) {
      const auto old = load<O, VE>(to);
#pragma unroll
      for (int e = 0; e < VE; ++e) y[e] += old.f(e);
    }
    store<O, VE>(to, y);
  };

  const uint32_t share = (count + groups - 1) / groups;
  const uint32_t begin = min(count, group * share), end = min(count, begin + share);
  const int32_t before = begin && begin < end ? int32_t(list[begin - 1] >> kShift) : -1;
  const int32_t after = begin < end && end < count ? int32_t(list[end] >> kShift) : -1;
  float acc[VE] = {};
  int32_t current = -1;
  bool from_before = false;
  for (uint32_t j = begin; j < end; j += U) {
    Pack<T, VE> v[U];
    float f[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t at = list[min(j + u, end - 1)] & (kFewTokens - 1), r = per_row.div(at);
      if (SCALED) f[u] = s.data[int64_t(r) * s.stride_row + int64_t(at - r * per_row.d) * s.stride_col];
      if (col < dim) v[u] = load<T, VE>(grad + int64_t(r) * grad_stride + col);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (j + u < end) {
        const int32_t local = int32_t(list[j + u] >> kShift);
        if (local != current) {
          if (current >= 0) {
            if (from_before) store<float, VE>(head + threadIdx.x * VE, acc);
            else write(current, acc);
          }
#pragma unroll
          for (int e = 0; e < VE; ++e) acc[e] = 0.0f;
          current = local;
          from_before = j + u == begin && local == before;
        }
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[e] = SCALED ? fmaf(f[u], v[u].f(e), acc[e]) : acc[e] + v[u].f(e);
      }
    }
  }
  const bool goes_on = current >= 0 && current == after;
  if (current >= 0) {
    if (from_before) store<float, VE>(head + threadIdx.x * VE, acc);
    else if (goes_on) store<float, VE>(tail + threadIdx.x * VE, acc);
    else write(current, acc);
  }
  if (me == 0) {
    first_row[group] = begin < end ? int32_t(list[begin] >> kShift) : -1;
    last_row[group] = goes_on ? current : -1;
  }
  __syncthreads();
  // The group in whose share a row began joins it.
  if (goes_on && !from_before) {
    for (uint32_t g = group + 1; g < groups && first_row[g] == current; ++g) {
      const auto more = load<float, VE>(head + ((g << lg) + me) * VE);
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[e] += more.v[e];
      if (last_row[g] != current) break;
    }
    write(current, acc);
  }
  if (!zero_first) zero_absent();
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

// The distance from each token to the next, or 0 where it varies.
int64_t token_step(const Tokens& k) {
  if (k.per_row == 1) return k.stride_row;
  return k.rows == 1 || k.stride_row == int64_t(k.per_row) * k.stride_col ? k.stride_col : 0;
}

// Shared memory of few_kernel, and its grid: rows of a block, blocks, column tiles.
struct FewPlan {
  int lg = 0;
  uint32_t tiles, span, blocks;
  size_t shared;
  FewPlan(uint32_t n, uint64_t vocab, uint64_t pieces, int ve) {
    while (lg < 5 && (1ull << lg) < pieces) ++lg;
    tiles = blocks_for(pieces, 1u << lg);
    // About two blocks an SM: each reads all tokens.
    const uint64_t ranges = std::max<uint64_t>(1, 296 / tiles);
    span = uint32_t(std::min<uint64_t>(std::max<uint64_t>((vocab + ranges - 1) / ranges, 1), 1u << (32 - kShift)));
    blocks = blocks_for(vocab, span);
    shared = size_t(2) * kFewThreads * ve * 4 + (span + 31) / 32 * 4 + size_t(n) * 4;
  }
};

size_t embedding_backward_workspace(const Tokens& k, uint64_t, uint64_t dim) {
  const uint64_t n = k.rows * k.per_row;
  return n <= kFewTokens ? 0 : Layout(n, dim).bytes;
}

void embedding_backward(const Mat& grad, const Tokens& k, uint64_t vocab, uint64_t dim, float scale,
                        const Scales& s, const Mat& out, bool accumulate, void* workspace,
                        cudaStream_t stream) {
  const uint32_t n = uint32_t(k.rows * k.per_row);
  if (n && n <= kFewTokens) {
    with_types(grad.type, out.type, [&](auto* pt, auto* po) {
      using T = std::remove_pointer_t<decltype(pt)>;
      using O = std::remove_pointer_t<decltype(po)>;
      with_width<T>(grad, k.rows, out, vocab, dim, [&](auto width) {
        constexpr int VE = decltype(width)::value;
        const FewPlan plan(n, vocab, dim / VE, VE);
        const auto kernel = s.data ? few_kernel<T, O, VE, true> : few_kernel<T, O, VE, false>;
        if (plan.shared > 40 * 1024)
          XGBB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(plan.shared)));
        kernel<<<dim3(plan.blocks, plan.tiles), kFewThreads, plan.shared, stream>>>(
            static_cast<const T*>(grad.data), grad.stride, k, token_step(k), FastDiv(uint32_t(k.per_row)), n,
            uint32_t(vocab), plan.span, s, scale, uint32_t(dim), static_cast<O*>(const_cast<void*>(out.data)),
            out.stride, accumulate, plan.lg);
      });
    });
    XGBB_CUDA(cudaGetLastError());
    return;
  }
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
