// The table's gradient of an embedding lookup, by sorted tokens:
//
//   dW[v] (+)= a * sum over the (r, t) with k[r][t] == v of s[r][t] dy[r]
//
// The present (token, position) pairs are sorted by token with a stable radix
// sort, so that a token's positions lie side by side and in their own order.
// Equal shares of the sorted list are then summed, and a token that crosses
// from one share into the next is joined from the shares' partial sums. Every
// sum has a fixed order: equal inputs give equal bits, and a frequent token
// costs no more than many rare ones. Sums are float32, rounded once when
// written.
#include <algorithm>

#include "nn_device.cuh"

namespace xgbb::nn {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kDigits = 256;
constexpr int kSortBlocks = 592;            // most blocks of a sort pass: 4 an SM
constexpr int kOneThreads = 1024;           // of the sort in one block
constexpr uint32_t kOneTokens = kOneThreads * 24;  // what its registers hold
constexpr uint32_t kNone = 0xffffffffu;
constexpr uint32_t kZeroBytes = 8192;              // zeros that wide rows are copied from

// Entries a thread holds of a sort tile: few, so that short lists fill the card,
// else as many as leave a block long runs of equal digits to write.
int sort_items(uint64_t n) { return n <= uint64_t(kSortBlocks) * kThreads * 4 ? 4 : 16; }
uint32_t sort_blocks(uint64_t n) {
  const uint64_t tile = kThreads * sort_items(n), tiles = (n + tile - 1) / tile;
  return uint32_t(tiles < kSortBlocks ? tiles : kSortBlocks);
}

// How the sorted list is shared out: 2^lg lanes move a row's columns, or a tile
// of them, and sum `share` entries. Long lists give each of the 1024 threads that
// an SM holds one share, short ones 8 entries a share.
struct SharePlan {
  int lg = 0;
  uint32_t tiles, share, shares;
  SharePlan(uint64_t n, uint64_t pieces) {
    lg = lanes_log2(pieces);
    tiles = blocks_for(pieces, 1u << lg);
    const uint64_t even = ((n << lg) * tiles + 148 * 1024 - 1) / (148 * 1024);
    share = uint32_t(std::min<uint64_t>(std::max<uint64_t>(8, (even + 7) / 8 * 8), 4096));
    shares = blocks_for(n, share);
  }
};

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
      keys[i] = take(n * 4 + 512);  // 32 lanes' four entries may lie past the end
      values[i] = take(n * 4 + 512);
    }
    hist = take(size_t(kDigits) * sort_blocks(n) * 4);
    totals = take((kDigits + 1) * 4);  // the digits' entries; all present entries
    // Wider pieces make fewer lanes, fewer lanes longer shares or as long ones.
    const uint64_t shares = SharePlan(n, (dim + 7) / 8).shares;
    head = take(shares * dim * 4);
    tail = take(shares * dim * 4);
    bytes = at;
  }
};

// The sort's entries. The first pass reads the tokens themselves: the key of
// one that is missing or past the table is kNone, and it is left out; the value
// is the position in [rows][per_row], or the row. `step`: the distance of one
// token from the next where it is the same for all, else 0. Later passes read
// what the pass before wrote.
enum Read { kTokens32, kTokens64, kSorted };
struct Source {
  Tokens k;
  FastDiv per_row;
  int64_t step;
  uint32_t vocab;
  bool rows;
  const uint32_t* keys;
  const uint32_t* values;
  // The keys of entries first, first + STRIDE, ..., those from `end` on none. The
  // loads are issued together: nothing asks for a value between them.
  template <int READ, int N, int STRIDE>
  __device__ __forceinline__ void load_keys(uint64_t first, uint64_t end, uint32_t (&key)[N]) const {
    if constexpr (READ == kSorted) {
      const uint32_t* from = keys + first;
#pragma unroll
      for (int i = 0; i < N; ++i) key[i] = first + i * STRIDE < end ? from[i * STRIDE] : kNone;
    } else {
      using Token = std::conditional_t<READ == kTokens64, int64_t, int32_t>;
      constexpr int BATCH = N < 8 ? N : 8;
      const Token* data = static_cast<const Token*>(k.data);
#pragma unroll
      for (int i0 = 0; i0 < N; i0 += BATCH) {
        Token w[BATCH];
        if (step) {
          const Token* from = data + int64_t(first + i0 * STRIDE) * step;
#pragma unroll
          for (int i = 0; i < BATCH; ++i)
            if (i0 + i < N)
              w[i] = first + (i0 + i) * STRIDE < end ? from[i * (STRIDE * step)] : Token(-1);
        } else {
#pragma unroll
          for (int i = 0; i < BATCH; ++i) {
            const uint32_t at = uint32_t(first) + (i0 + i) * STRIDE;
            const uint32_t r = per_row.div(at);
            if (i0 + i < N)
              w[i] = first + (i0 + i) * STRIDE < end
                         ? data[int64_t(r) * k.stride_row + int64_t(at - r * per_row.d) * k.stride_col]
                         : Token(-1);
          }
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
          if (i0 + i < N) key[i0 + i] = uint64_t(int64_t(w[i])) < vocab ? uint32_t(w[i]) : kNone;
      }
    }
  }
  template <int READ>
  __device__ __forceinline__ uint32_t value(uint32_t i) const {
    if constexpr (READ == kSorted) return values[i];
    else return rows ? per_row.div(i) : i;
  }
};

// Exclusive sum of one value a thread over the block; `total` gets the sum.
template <int WARPS>
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
  for (int w = 0; w < WARPS; ++w) {
    if (w < int(warp)) before += warp_sums[w];
    total += warp_sums[w];
  }
  return before + x - v;
}

// A warp's next 32 entries: each one's rank among the warp's entries of its digit
// so far, which `count` holds. The lanes of a digit find each other by the bits
// that they set in mask[digit], zero before and after (warp-level multisplit;
// Ashkiani et al., "GPU multisplit", 2016).
template <class C>
__device__ __forceinline__ uint32_t next_rank(uint32_t digit, bool in, uint32_t* mask, C* count) {
  const uint32_t bit = 1u << (threadIdx.x & 31);
  if (in) atomicOr(&mask[digit], bit);
  __syncwarp();
  uint32_t same = 0, rank = 0;
  if (in) {
    same = mask[digit];
    rank = count[digit] + __popc(same & (bit - 1));
  }
  __syncwarp();
  if (same >> 1 < bit && in) {  // the digit's highest lane
    count[digit] = C(rank + 1);
    mask[digit] = 0;
  }
  __syncwarp();
  return rank;
}

// Block b sorts the entries [b * per, (b + 1) * per). hist[digit][block].
template <int READ>
__global__ void __launch_bounds__(kThreads)
    sort_hist_kernel(Source src, const uint32_t* __restrict__ present, uint32_t n, uint32_t per, int shift,
                     uint32_t* __restrict__ hist) {
  constexpr int U = 8;
  __shared__ uint32_t count[kDigits];
  count[threadIdx.x] = 0;
  __syncthreads();
  if (READ == kSorted) n = *present;
  const uint64_t begin = uint64_t(blockIdx.x) * per, end = min(uint64_t(n), begin + per);
  for (uint64_t i = begin + threadIdx.x; i < end; i += kThreads * U) {
    uint32_t key[U];
    src.load_keys<READ, U, kThreads>(i, end, key);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (key[u] != kNone) atomicAdd(&count[(key[u] >> shift) & (kDigits - 1)], 1u);
  }
  __syncthreads();
  hist[threadIdx.x * gridDim.x + blockIdx.x] = count[threadIdx.x];
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
    const uint32_t x = block_scan<kWarps>(v, warp_sums, total);
    if (i < blocks) h[i] = before + x;
    before += total;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = before;
}

// Ranks a tile's entries by digit, stably: each warp holds an equal part of it,
// 32 entries at a time, and counts its own digits. The tile is put in
// order in shared memory and leaves it in runs of equal digits, while the next
// tile's keys are on their way. The first pass tells how many entries are
// present. Bound by shared memory (77 % of its wavefronts): 26.2 M entries take
// 195 us in the first pass and 145 in the second, after 32 and 27 us for the
// counts. With the lanes of a digit found by ballots it took 284 and 210 us, by
// match.any 448 and 252.
template <int READ, int kItems>
__global__ void __launch_bounds__(kThreads, 4)
    sort_scatter_kernel(Source src, uint32_t* __restrict__ present, uint32_t n, uint32_t per, int shift,
                        const uint32_t* __restrict__ hist, const uint32_t* __restrict__ totals,
                        uint32_t* __restrict__ keys_out, uint32_t* __restrict__ values_out) {
  constexpr int kTile = kThreads * kItems;
  __shared__ uint32_t to[kDigits];            // where the digit's entries go, less their place in the ordered tile
  __shared__ uint32_t count[kWarps][kDigits];  // the warp's entries of the digit, then where they begin in the tile
  __shared__ uint32_t warp_sums[kWarps];
  __shared__ uint32_t keys[kTile < kWarps * kDigits ? kWarps * kDigits : kTile], values[kTile];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = threadIdx.x;
  if (READ == kSorted) n = *present;
  uint32_t all, before = 0, digits = 0;
  if (totals) {
    digits = totals[d];
    before = hist[d * gridDim.x + blockIdx.x];
  } else {  // few blocks, whose counts nobody has added up
    const uint32_t* h = hist + d * gridDim.x;
#pragma unroll 8
    for (uint32_t b = 0; b < gridDim.x; ++b) {
      if (b < blockIdx.x) before += h[b];
      digits += h[b];
    }
  }
  uint32_t next = block_scan<kWarps>(digits, warp_sums, all) + before;
  if (READ != kSorted && blockIdx.x == 0 && d == 0) *present = all;
  uint32_t* const masks = keys;  // [warps][digits], while the tile is ranked
  const uint32_t mine = warp * (kItems * 32) + lane;
  uint64_t begin = uint64_t(blockIdx.x) * per;
  const uint64_t end = min(uint64_t(n), begin + per);
  uint32_t key[kItems], rank[kItems];
  src.load_keys<READ, kItems, 32>(begin + mine, end, key);
  for (; begin < end; begin += kTile) {
#pragma unroll
    for (int w = 0; w < kWarps; ++w) count[w][d] = masks[w * kDigits + d] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i)
      rank[i] = next_rank((key[i] >> shift) & (kDigits - 1), key[i] != kNone, masks + warp * kDigits, count[warp]);
    __syncthreads();
    uint32_t total = 0, tile_total;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) total += count[w][d];
    const uint32_t local = block_scan<kWarps>(total, warp_sums, tile_total);
    uint32_t at = local;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const uint32_t c = count[w][d];
      count[w][d] = at;
      at += c;
    }
    to[d] = next - local;
    next += total;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i)
      if (key[i] != kNone) {
        const uint32_t p = count[warp][(key[i] >> shift) & (kDigits - 1)] + rank[i];
        keys[p] = key[i];
        values[p] = src.value<READ>(uint32_t(begin) + mine + i * 32);
      }
    src.load_keys<READ, kItems, 32>(begin + kTile + mine, end, key);
    __syncthreads();
    for (uint32_t p = threadIdx.x; p < tile_total; p += kThreads) {
      const uint32_t k = keys[p], q = to[(k >> shift) & (kDigits - 1)] + p;
      keys_out[q] = k;
      values_out[q] = values[p];
    }
    __syncthreads();
  }
}

// The rows without a token, for blocks beside a block that sorts: block b of
// `blocks` looks through all tokens for those of its equal share of the rows and
// zeroes the others: wide rows by copies behind the threads' backs, narrow ones
// by plain stores.
struct Rows {
  char* data;
  int64_t stride;  // bytes
  uint32_t bytes, item;
  bool bulk;
};
template <int READ>
__device__ __forceinline__ void zero_rows_beside(const Source& src, uint32_t n, const Rows& rows, uint32_t block,
                                                 uint32_t blocks, uint32_t* space) {
  constexpr int U = 8;
  const uint32_t first = uint32_t(uint64_t(src.vocab) * block / blocks);
  const uint32_t here = uint32_t(uint64_t(src.vocab) * (block + 1) / blocks) - first;
  uint32_t* zeros = space;
  uint32_t* present = space + kZeroBytes / 4;  // a bit a row
  const uint32_t batch_rows = 32 * 1024;       // rows that the bits are for at a time
  for (uint32_t i = threadIdx.x; i < kZeroBytes / 4; i += kOneThreads) zeros[i] = 0;
  bulk_fence();
  for (uint32_t r0 = 0; r0 < here; r0 += batch_rows) {
    const uint32_t count = min(batch_rows, here - r0), row0 = first + r0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < (count + 31) / 32; i += kOneThreads) present[i] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kOneThreads * U) {
      uint32_t key[U];
      src.load_keys<READ, U, kOneThreads>(i, n, key);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (key[u] - row0 < count) atomicOr(&present[(key[u] - row0) >> 5], 1u << ((key[u] - row0) & 31));
    }
    __syncthreads();
    if (rows.bulk) {
      for (uint32_t r = threadIdx.x; r < count; r += kOneThreads)
        if (!(present[r >> 5] >> (r & 31) & 1)) {
          char* to = rows.data + int64_t(row0 + r) * rows.stride;
          for (uint32_t at = 0; at < rows.bytes; at += kZeroBytes)
            bulk_store(to + at, zeros, min(kZeroBytes, rows.bytes - at));
        }
    } else {
      const uint32_t items = rows.bytes / rows.item, lane = threadIdx.x & 31;
      for (uint32_t r = threadIdx.x >> 5; r < count; r += kOneThreads / 32)
        if (!(present[r >> 5] >> (r & 31) & 1)) {
          char* to = rows.data + int64_t(row0 + r) * rows.stride;
          for (uint32_t i = lane; i < items; i += 32) {
            if (rows.item == 4) reinterpret_cast<uint32_t*>(to)[i] = 0;
            else reinterpret_cast<uint16_t*>(to)[i] = 0;
          }
        }
    }
  }
  bulk_wait_all();
}

// The whole sort of up to 1024 ITEMS entries in one block, which holds them in
// registers, (key, position) with 16-bit positions and ranks, and passes them
// through shared memory after each pass. The other blocks zero the rows that
// have no token meanwhile: of 16411 tokens' gradient of 65536 x 2048 f32 the sort
// takes 30 us, the zeros 80, and all 116 (166 with the zeros beside the sums),
// where its 604 MB take 92 at the copy rate.
template <int READ, int ITEMS>
__global__ void __launch_bounds__(kOneThreads)
    sort_one_kernel(Source src, uint32_t n, int passes, uint32_t* __restrict__ present,
                    uint32_t* __restrict__ keys_out, uint32_t* __restrict__ values_out, Rows rows) {
  constexpr int kOneWarps = kOneThreads / 32;
  extern __shared__ __align__(16) uint32_t space[];
  if (blockIdx.x) return zero_rows_beside<READ>(src, n, rows, blockIdx.x - 1, gridDim.x - 1, space);
  uint32_t* keys = space;                                                       // [1024 ITEMS]
  uint16_t* at = reinterpret_cast<uint16_t*>(keys + kOneThreads * ITEMS);       // [1024 ITEMS]
  uint16_t* count = at + kOneThreads * ITEMS;                                   // [warps][digits]
  uint32_t* mask = reinterpret_cast<uint32_t*>(count + kOneWarps * kDigits);    // [warps][digits]
  __shared__ uint32_t warp_sums[kOneWarps];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t turns = (n + kOneThreads - 1) / kOneThreads;  // at most ITEMS
  const uint32_t mine = warp * (turns * 32) + lane;
  uint32_t key[ITEMS], both[ITEMS];  // both: rank << 16 | position
  src.load_keys<READ, ITEMS, 32>(mine, min(n, (warp + 1) * turns * 32), key);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) both[i] = mine + i * 32;
  for (uint32_t i = threadIdx.x; i < kOneWarps * kDigits; i += kOneThreads) mask[i] = 0;
  uint32_t all = n;
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * 8;
    if (pass) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const uint32_t p = mine + i * 32;
        const bool in = i < turns && p < all;
        key[i] = in ? keys[p] : kNone;
        both[i] = in ? at[p] : 0;
      }
    }
    for (uint32_t i = threadIdx.x; i < kOneWarps * kDigits / 2; i += kOneThreads)
      reinterpret_cast<uint32_t*>(count)[i] = 0;
    __syncthreads();
    uint16_t* const own = count + warp * kDigits;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (i < turns)
        both[i] |= next_rank((key[i] >> shift) & (kDigits - 1), key[i] != kNone, mask + warp * kDigits, own) << 16;
    __syncthreads();
    // A digit's warps, eight to a thread: their counts' sums, then their places.
    const uint32_t digit = threadIdx.x >> 2, w0 = (threadIdx.x & 3) * 8;
    uint32_t c[8], eight = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      c[w] = count[(w0 + w) * kDigits + digit];
      eight += c[w];
    }
    uint32_t place = block_scan<kOneWarps>(eight, warp_sums, all);
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      count[(w0 + w) * kDigits + digit] = uint16_t(place);
      place += c[w];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (key[i] != kNone) {
        const uint32_t p = own[(key[i] >> shift) & (kDigits - 1)] + (both[i] >> 16);
        keys[p] = key[i];
        at[p] = uint16_t(both[i]);
      }
    __syncthreads();
  }
  if (threadIdx.x == 0) *present = all;
  for (uint32_t p = threadIdx.x; p < all; p += kOneThreads) {
    keys_out[p] = keys[p];
    values_out[p] = src.value<READ>(at[p]);
  }
}

// scale times a row's sum, into the row.
template <class O, int VE>
__device__ __forceinline__ void write_row(O* to, const float (&sum)[VE], float scale, bool accumulate) {
  float y[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) y[e] = sum[e] * scale;
  if (accumulate) {
    const auto old = load<O, VE>(to);
#pragma unroll
    for (int e = 0; e < VE; ++e) y[e] += old.f(e);
  }
  store_global<O, VE>(to, y);
}

// Rows without a token, in front of the others' sums: block b looks up the rows
// [b 256, b 256 + 256) in the sorted keys, a row a thread, and zeroes the absent
// ones: wide ones by copies behind the threads' backs, narrow ones together.
template <class O, int VE>
__device__ __forceinline__ void zero_absent(const uint32_t* __restrict__ keys, uint32_t n, uint32_t vocab, uint32_t dim,
                                            O* __restrict__ out, int64_t out_stride, bool bulk, uint32_t block,
                                            uint4* zeros) {
  __shared__ uint32_t absent[kWarps];
  const uint32_t row = block * kThreads + threadIdx.x;
  if (bulk) {
    for (uint32_t i = threadIdx.x; i < kZeroBytes / 16; i += kThreads) zeros[i] = make_uint4(0, 0, 0, 0);
    bulk_fence();
  }
  uint32_t lo = 0, hi = n;
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (keys[mid] < row) lo = mid + 1;
    else hi = mid;
  }
  const bool none = row < vocab && (lo == n || keys[lo] != row);
  if (bulk) {
    __syncthreads();
    const uint32_t row_bytes = dim * sizeof(O);
    if (none) {
      char* to = reinterpret_cast<char*>(out + int64_t(row) * out_stride);
      for (uint32_t at = 0; at < row_bytes; at += kZeroBytes) bulk_store(to + at, zeros, min(kZeroBytes, row_bytes - at));
    }
    bulk_wait_all();
    return;
  }
  const uint32_t votes = __ballot_sync(0xffffffffu, none);
  if ((threadIdx.x & 31) == 0) absent[threadIdx.x >> 5] = votes;
  __syncthreads();
  const float zero[VE] = {};
  const uint32_t pieces = dim / VE;
  for (uint64_t i = threadIdx.x; i < uint64_t(pieces) * kThreads; i += kThreads) {
    const uint32_t r = uint32_t(i / pieces);
    if (absent[r >> 5] >> (r & 31) & 1)
      store_global<O, VE>(out + int64_t(block * kThreads + r) * out_stride + (i - uint64_t(r) * pieces) * VE, zero);
  }
}

// Groups of G = 2^lg lanes own VE columns a lane (blockIdx.y: the tile of
// columns) and sum `share` sorted entries each. The lanes read four entries
// each, a turn ahead, and pass them on by shuffles; a turn that lies in one
// token, as most do where tokens are frequent, is summed without a look at its
// keys. A token that lies in one share whole goes to its row; the sum of one
// that came in from the share before goes to head[share], of one that goes on
// into the next to tail[share] (a share inside one token has its sum in head).
// The first `zero_blocks` blocks zero the rows without a token.
// Bound by the latency of gathers from the L2 cache: 26.2 M rows of 64 bf16, 3.36
// GB, in 355 us (9.5 TB/s). With the keys of a step read by every lane, and
// registers for the next step's, it took 540 us at three blocks an SM and 810,
// spilling, at four; five and six blocks spill as well (405 and 415).
template <class T, class O, int VE, bool SCALED>
__global__ void __launch_bounds__(kThreads, 4)
    share_sum_kernel(const T* __restrict__ grad, int64_t grad_stride, const uint32_t* __restrict__ keys,
                     const uint32_t* __restrict__ values, const uint32_t* __restrict__ present, uint32_t share_size,
                     uint32_t vocab, FastDiv per_row, Scales s, float scale, uint32_t dim, O* __restrict__ out,
                     int64_t out_stride, bool accumulate, float* __restrict__ head, float* __restrict__ tail, int lg,
                     uint32_t zero_blocks, bool bulk) {
  __shared__ uint4 zeros[kZeroBytes / 16];
  const uint32_t n = *present;
  if (blockIdx.x < zero_blocks) {
    if (blockIdx.y == 0) zero_absent<O, VE>(keys, n, vocab, dim, out, out_stride, bulk, blockIdx.x, zeros);
    return;
  }
  const uint32_t G = 1u << lg, lane = threadIdx.x & (G - 1), E = 4 * G;
  const uint32_t mask = (G == 32 ? ~0u : (1u << G) - 1) << (threadIdx.x & 31 & ~(G - 1));
  const uint64_t share = (uint64_t(blockIdx.x - zero_blocks) * kThreads + threadIdx.x) >> lg;
  const uint32_t col = (blockIdx.y * G + lane) * VE;
  const uint64_t begin = share * share_size;
  if (begin >= n) return;  // the whole group
  const uint32_t here = uint32_t(min(uint64_t(share_size), n - begin));
  const uint32_t before = begin ? keys[begin - 1] : kNone;
  const uint32_t after = begin + here < n ? keys[begin + here] : kNone;
  // Lanes past the last column read the last piece, and write nothing.
  const T* const columns = grad + min(col, dim - VE);
  Sum<T, VE> acc;
  acc.clear();
  uint32_t current = kNone;
  bool from_before = false;
  const auto finish = [&](bool goes_on) {
    if (current == kNone || col >= dim) return;
    float y[VE];
    acc.get(y);
    if (from_before || goes_on) store_global<float, VE>((from_before ? head : tail) + share * dim + col, y);
    else write_row<O, VE>(out + int64_t(current) * out_stride + col, y, scale, accumulate);
  };
  // What a turn reads past the list's end is not used.
  const uint4* key4 = reinterpret_cast<const uint4*>(keys + begin) + lane;
  const uint4* value4 = reinterpret_cast<const uint4*>(values + begin) + lane;
  uint4 next_key = *key4, next_value = *value4;
  for (uint32_t r0 = 0; r0 < here; r0 += E) {
    const uint4 key = next_key;
    uint4 row = next_value;
    float4 f = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
    if (r0 + E < here) {
      key4 += G;
      value4 += G;
      next_key = *key4;
      next_value = *value4;
    }
    if (SCALED) {
      const auto look = [&](uint32_t i, uint32_t& value) {
        float v = 0.0f;
        if (r0 + lane * 4 + i < here) {
          const uint32_t r = per_row.div(value);
          v = s.data[int64_t(r) * s.stride_row + int64_t(value - r * per_row.d) * s.stride_col];
          value = r;
        }
        return v;
      };
      f.x = look(0, row.x);
      f.y = look(1, row.y);
      f.z = look(2, row.z);
      f.w = look(3, row.w);
    }
    const bool one = r0 + E <= here && __shfl_sync(mask, key.w, G - 1, G) == current;
    if (one) {
#pragma unroll 2
      for (uint32_t q = 0; q < G; ++q) {
        const uint32_t at[4] = {__shfl_sync(mask, row.x, q, G), __shfl_sync(mask, row.y, q, G),
                                __shfl_sync(mask, row.z, q, G), __shfl_sync(mask, row.w, q, G)};
        float g[4] = {1.0f, 1.0f, 1.0f, 1.0f};
        if (SCALED) {
          g[0] = __shfl_sync(mask, f.x, q, G);
          g[1] = __shfl_sync(mask, f.y, q, G);
          g[2] = __shfl_sync(mask, f.z, q, G);
          g[3] = __shfl_sync(mask, f.w, q, G);
        }
        Pack<T, VE> v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = load<T, VE>(columns + int64_t(at[u]) * grad_stride);
#pragma unroll
        for (int u = 0; u < 4; ++u) acc.template add<SCALED>(v[u], g[u]);
      }
      continue;
    }
    for (uint32_t q = 0; q < G && r0 + q * 4 < here; ++q) {
      const uint32_t k[4] = {__shfl_sync(mask, key.x, q, G), __shfl_sync(mask, key.y, q, G),
                             __shfl_sync(mask, key.z, q, G), __shfl_sync(mask, key.w, q, G)};
      const uint32_t at[4] = {__shfl_sync(mask, row.x, q, G), __shfl_sync(mask, row.y, q, G),
                              __shfl_sync(mask, row.z, q, G), __shfl_sync(mask, row.w, q, G)};
      float g[4] = {1.0f, 1.0f, 1.0f, 1.0f};
      if (SCALED) {
        g[0] = __shfl_sync(mask, f.x, q, G);
        g[1] = __shfl_sync(mask, f.y, q, G);
        g[2] = __shfl_sync(mask, f.z, q, G);
        g[3] = __shfl_sync(mask, f.w, q, G);
      }
      const uint32_t left = here - (r0 + q * 4);
      Pack<T, VE> v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (u < left) v[u] = load<T, VE>(columns + int64_t(at[u]) * grad_stride);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (u < left) {
          if (k[u] != current) {
            finish(false);
            acc.clear();
            current = k[u];
            from_before = r0 + q + u == 0 && k[u] == before;
          }
          acc.template add<SCALED>(v[u], g[u]);
        }
    }
  }
  finish(current == after);
}

// Tokens that cross shares. A warp looks at one share: of the token that begins
// in it and goes on after it, if there is one, the partial sums are added up in
// the shares' order by the warp, or by the block's warps together (each every
// eighth share, then the warps in order) where there are over 32. blockIdx.y: 32
// pieces of the columns.
constexpr uint32_t kLongRun = 32;
template <class O, int VE>
__global__ void __launch_bounds__(kThreads)
    join_kernel(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ present, uint32_t share_size,
                float scale, uint32_t dim, O* __restrict__ out, int64_t out_stride, bool accumulate,
                const float* __restrict__ head, const float* __restrict__ tail) {
  constexpr int U = 8;
  __shared__ uint32_t long_share[kWarps], long_last[kWarps];
  __shared__ float part[kWarps][32 * VE];
  const uint32_t n = *present, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t share = blockIdx.x * kWarps + warp, c = (blockIdx.y * 32 + lane) * VE;
  if (uint64_t(blockIdx.x * kWarps + 1) * share_size >= n) return;  // no share of the block goes on
  uint32_t last = share, token = kNone;  // the share that the token's last entry is in
  if (uint64_t(share + 1) * share_size < n) {
    const uint32_t begin = share * share_size, end = begin + share_size;
    token = keys[end];
    const bool begun = keys[end - 1] == token;
    const bool earlier = begin && keys[begin] == token && keys[begin - 1] == token;
    if (begun && !earlier) {
      // The next shares that begin with the token, 32 at a look.
      uint32_t same;
      do {
        const uint64_t at = uint64_t(last + 1 + lane) * share_size;
        same = __ballot_sync(0xffffffffu, at < n && keys[at] == token);
        last += same == ~0u ? 32 : __ffs(~same) - 1;
      } while (same == ~0u);
    } else {
      token = kNone;
    }
  }
  const bool is_long = last - share > kLongRun;
  if (lane == 0) {
    long_share[warp] = is_long ? share : kNone;
    long_last[warp] = last;
  }
  const auto add = [&](float(&acc)[VE], const float* from) {
    const auto v = load<float, VE>(from);
#pragma unroll
    for (int e = 0; e < VE; ++e) acc[e] += v.v[e];
  };
  if (token != kNone && !is_long && c < dim) {
    float acc[VE] = {};
    add(acc, tail + uint64_t(share) * dim + c);
#pragma unroll 8
    for (uint32_t q = share + 1; q <= last; ++q) add(acc, head + uint64_t(q) * dim + c);
    write_row<O, VE>(out + int64_t(token) * out_stride + c, acc, scale, accumulate);
  }
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) {
    const uint32_t from = long_share[i], to = long_last[i];
    if (from == kNone) continue;
    float acc[VE] = {};
    if (c < dim) {
      if (warp == 0) add(acc, tail + uint64_t(from) * dim + c);
      for (uint32_t q = from + 1 + warp; q <= to; q += kWarps * U) {
        Pack<float, VE> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (q + u * kWarps <= to) v[u] = load<float, VE>(head + uint64_t(q + u * kWarps) * dim + c);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (q + u * kWarps <= to)
#pragma unroll
            for (int e = 0; e < VE; ++e) acc[e] += v[u].v[e];
      }
    }
#pragma unroll
    for (int e = 0; e < VE; ++e) part[warp][lane * VE + e] = acc[e];
    __syncthreads();
    if (warp == 0 && c < dim) {
      for (int w = 1; w < kWarps; ++w)
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[e] += part[w][lane * VE + e];
      write_row<O, VE>(out + int64_t(keys[uint64_t(from + 1) * share_size]) * out_stride + c, acc, scale, accumulate);
    }
    __syncthreads();
  }
}

// Zeros into rows of `dim` values, where there is no token at all.
template <class O, int VE>
__global__ void __launch_bounds__(kThreads)
    zero_rows_kernel(O* __restrict__ out, int64_t stride, uint32_t pieces, FastDiv div, uint64_t total) {
  const float zero[VE] = {};
  for (uint64_t i = uint64_t(blockIdx.x) * kThreads + threadIdx.x; i < total;
       i += uint64_t(gridDim.x) * kThreads) {
    const uint64_t row = total <= 0xffffffffull ? div.div(uint32_t(i)) : i / pieces;
    store_global<O, VE>(out + int64_t(row) * stride + (i - row * pieces) * VE, zero);
  }
}

// Few tokens, in one launch: of N x M blocks, block (x, y) owns the table's rows
// x, x + N, ... in a tile of columns (neighbours apart, since the frequent tokens
// of many vocabularies lie together). It picks its rows' tokens out of all n, in
// their order, sorts them by row in shared memory, zeroes the rows that have
// none, and sums the others: groups of 2^lg lanes take equal shares of the sorted
// list, and what crosses shares is joined through shared memory, in the shares'
// order. No row is written by two blocks. An entry is its row's number among the
// block's rows << kShift | position. Bound by latency: 4100 tokens of 96 f32 take
// 8 us, 8000 of 32 bf16 8 to 13, where the sort's launches alone take 20; from 8193
// tokens on, each block's look at all of them costs more than the sort.
constexpr int kFewThreads = 512;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kShift = 13;
constexpr uint32_t kFewTokens = 1u << kShift;
constexpr int kFewTurns = kFewTokens / kFewThreads;  // entries a lane sorts
constexpr uint32_t kFewCounts = kFewWarps * kDigits * 4;

template <class T, class O, int VE, bool SCALED>
__global__ void __launch_bounds__(kFewThreads, 2)
    few_kernel(const T* __restrict__ grad, int64_t grad_stride, Source src, uint32_t n, FastDiv blocks, Scales s,
               float scale, uint32_t dim, O* __restrict__ out, int64_t out_stride, bool accumulate, bool bulk, int lg) {
  constexpr int U = 4, kBatch = 8;
  extern __shared__ __align__(16) uint32_t space[];
  __shared__ uint32_t warp_sums[kFewWarps];
  // While sorting, counts and masks; then the sums that came in from the group before, [threads][VE].
  uint32_t* const counts = space;
  uint32_t* const masks = space + kFewCounts / 4;
  float* const head = reinterpret_cast<float*>(space);
  static_assert(kFewThreads * VE * 4 <= 2 * kFewCounts, "head in the place of counts and masks");
  uint32_t* const zeros = space + 2 * kFewCounts / 4;
  const uint32_t span = (src.vocab + blocks.d - 1) / blocks.d;  // rows of a block, at most
  const uint32_t rows_here = (src.vocab - blockIdx.x + blocks.d - 1) / blocks.d;
  uint32_t* const present = zeros + (bulk ? kZeroBytes / 4 : 0);  // a bit a row
  uint32_t* list = present + (span + 31) / 32;
  const uint32_t turns = (n + kFewThreads - 1) / kFewThreads, per = turns * 32;
  uint32_t* other = list + kFewWarps * per;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

  // Warp w looks at the tokens [w per, w per + per) and keeps its rows' there.
  for (uint32_t i = threadIdx.x; i < (span + 31) / 32; i += kFewThreads) present[i] = 0;
  if (bulk)
    for (uint32_t i = threadIdx.x; i < kZeroBytes / 4; i += kFewThreads) zeros[i] = 0;
  bulk_fence();
  __syncthreads();
  uint32_t own = 0;
  const uint32_t from = warp * per, to = min(n, from + per);
  for (uint32_t i0 = from; i0 < to; i0 += 32 * kBatch) {
    uint32_t key[kBatch];
    if (src.k.type == kI64) src.load_keys<kTokens64, kBatch, 32>(i0 + lane, to, key);
    else src.load_keys<kTokens32, kBatch, 32>(i0 + lane, to, key);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const uint32_t r = blocks.div(key[i]);
      const bool mine = key[i] != kNone && key[i] - r * blocks.d == blockIdx.x;
      const uint32_t votes = __ballot_sync(0xffffffffu, mine);
      if (mine) {
        list[from + own + __popc(votes & ((1u << lane) - 1))] = r << kShift | (i0 + i * 32 + lane);
        atomicOr(&present[r >> 5], 1u << (r & 31));
      }
      own += __popc(votes);
    }
  }
  __syncthreads();

  const uint32_t G = 1u << lg, me = threadIdx.x & (G - 1), group = threadIdx.x >> lg, groups = kFewThreads >> lg;
  const uint32_t col = (blockIdx.y * G + me) * VE;
  const int64_t row_stride = int64_t(blocks.d) * out_stride;
  O* const mine_out = out + int64_t(blockIdx.x) * out_stride + col;
  // Absent rows: wide ones whole, a share of the block's rows for each column
  // tile, written behind the threads' backs while they sort and sum; narrow ones
  // by plain stores.
  if (!accumulate && bulk) {
    const uint32_t row_bytes = dim * sizeof(O);
    const uint32_t last = uint32_t(uint64_t(rows_here) * (blockIdx.y + 1) / gridDim.y);
    for (uint32_t r = uint32_t(uint64_t(rows_here) * blockIdx.y / gridDim.y) + threadIdx.x; r < last; r += kFewThreads)
      if (!(present[r >> 5] >> (r & 31) & 1)) {
        char* row = reinterpret_cast<char*>(out + int64_t(blockIdx.x) * out_stride + r * row_stride);
        for (uint32_t at = 0; at < row_bytes; at += kZeroBytes) bulk_store(row + at, zeros, min(kZeroBytes, row_bytes - at));
      }
  } else if (!accumulate && col < dim) {
    const float zero[VE] = {};
    for (uint32_t r = group; r < rows_here; r += groups)
      if (!(present[r >> 5] >> (r & 31) & 1)) store_global<O, VE>(mine_out + r * row_stride, zero);
  }

  // In the order of rows and, within a row, of positions.
  if (lane == 0) warp_sums[warp] = own;
  __syncthreads();
  uint32_t count = 0, earlier = 0;
#pragma unroll
  for (int w = 0; w < kFewWarps; ++w) {
    if (w < int(warp)) earlier += warp_sums[w];
    count += warp_sums[w];
  }
  const bool by_counting = count <= kFewThreads / 2;
  if (by_counting) {  // few entries: each one's place is the number of smaller ones
    for (uint32_t i = lane; i < own; i += 32) other[earlier + i] = list[from + i];
    __syncthreads();
    if (threadIdx.x < count) {
      const uint32_t mine = other[threadIdx.x];
      uint32_t place = 0;
#pragma unroll 8
      for (uint32_t j = 0; j < count; ++j) place += other[j] < mine;
      list[place] = mine;
    }
    __syncthreads();
  }
  // Else stably by the row's digits, the first pass out of each warp's own part.
  uint32_t begin_here = from, end_here = from + own;
  for (int shift = kShift; !by_counting && (shift == kShift || (rows_here - 1) >> (shift - kShift)); shift += 8) {
    uint32_t* const my_counts = counts + warp * kDigits;
    for (uint32_t i = threadIdx.x; i < kFewCounts / 4; i += kFewThreads) counts[i] = masks[i] = 0;
    if (shift > kShift) {
      const uint32_t each = (count + kFewThreads - 1) / kFewThreads * 32;
      begin_here = min(count, warp * each);
      end_here = min(count, begin_here + each);
    }
    __syncthreads();
    uint32_t entry[kFewTurns], rank[kFewTurns];
#pragma unroll
    for (int i = 0; i < kFewTurns; ++i)
      if (begin_here + i * 32 < end_here) {
        const bool in = begin_here + i * 32 + lane < end_here;
        entry[i] = in ? list[begin_here + i * 32 + lane] : 0;
        rank[i] = next_rank((entry[i] >> shift) & (kDigits - 1), in, masks + warp * kDigits, my_counts);
      }
    __syncthreads();
    const uint32_t digit = threadIdx.x >> 1, w0 = (threadIdx.x & 1) * 8;
    uint32_t c[8], eight = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      c[w] = counts[(w0 + w) * kDigits + digit];
      eight += c[w];
    }
    uint32_t place = block_scan<kFewWarps>(eight, warp_sums, count);
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      counts[(w0 + w) * kDigits + digit] = place;
      place += c[w];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kFewTurns; ++i)
      if (begin_here + i * 32 + lane < end_here)
        other[my_counts[(entry[i] >> shift) & (kDigits - 1)] + rank[i]] = entry[i];
    __syncthreads();
    uint32_t* const sorted = other;
    other = list;
    list = sorted;
  }

  const auto write = [&](int32_t local, const float(&sum)[VE]) {
    if (col < dim) write_row<O, VE>(mine_out + local * row_stride, sum, scale, accumulate);
  };
  const uint32_t share = max((count + groups - 1) / groups, uint32_t(U));
  const uint32_t begin = min(count, group * share), end = min(count, begin + share);
  const int32_t before = begin && begin < end ? int32_t(list[begin - 1] >> kShift) : -1;
  const int32_t after = begin < end && end < count ? int32_t(list[end] >> kShift) : -1;
  Sum<T, VE> acc;
  acc.clear();
  float sum[VE];
  int32_t current = -1;
  bool from_before = false;
  const T* const columns = grad + min(col, dim - VE);
  for (uint32_t j = begin; j < end; j += U) {
    Pack<T, VE> v[U];
    float f[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t at = list[min(j + u, end - 1)] & (kFewTokens - 1), r = src.per_row.div(at);
      if (SCALED) f[u] = s.data[int64_t(r) * s.stride_row + int64_t(at - r * src.per_row.d) * s.stride_col];
      v[u] = load<T, VE>(columns + int64_t(r) * grad_stride);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (j + u < end) {
        const int32_t local = int32_t(list[j + u] >> kShift);
        if (local != current) {
          if (current >= 0) {
            acc.get(sum);
            if (from_before) store<float, VE>(head + threadIdx.x * VE, sum);
            else write(current, sum);
          }
          acc.clear();
          current = local;
          from_before = j + u == begin && local == before;
        }
        acc.template add<SCALED>(v[u], SCALED ? f[u] : 1.0f);
      }
    }
  }
  acc.get(sum);
  const bool goes_on = current >= 0 && current == after;
  if (current >= 0) {
    if (from_before) store<float, VE>(head + threadIdx.x * VE, sum);
    else if (!goes_on) write(current, sum);
  }
  __syncthreads();
  // The group in whose share a row began joins it, from what it holds of it.
  if (goes_on && !from_before) {
    uint32_t lo = end, hi = count;  // the first entry of a later row
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (int32_t(list[mid] >> kShift) == current) lo = mid + 1;
      else hi = mid;
    }
    const uint32_t last = (lo - 1) / share;
#pragma unroll 8
    for (uint32_t g = group + 1; g <= last; ++g) {
      const auto more = load<float, VE>(head + ((g << lg) + me) * VE);
#pragma unroll
      for (int e = 0; e < VE; ++e) sum[e] += more.v[e];
    }
    write(current, sum);
  }
  if (bulk) bulk_wait_all();
}

// The distance from each token to the next, or 0 where it varies.
int64_t token_step(const Tokens& k) {
  if (k.per_row == 1) return k.stride_row;
  return k.rows == 1 || k.stride_row == int64_t(k.per_row) * k.stride_col ? k.stride_col : 0;
}

// Shared memory of few_kernel, and its grid: blocks and column tiles.
struct FewPlan {
  // Of the most tokens and 65536 rows a block.
  static constexpr size_t kMostShared = 2 * kFewCounts + kZeroBytes + 65536 / 8 + size_t(2) * 4 * kFewTokens;
  int lg = 0;
  uint32_t tiles, blocks;
  size_t shared;
  FewPlan(uint32_t n, uint64_t vocab, uint64_t pieces, bool bulk) {
    while (lg < 5 && (1ull << lg) < pieces) ++lg;
    tiles = blocks_for(pieces, 1u << lg);
    // About two blocks an SM, which all read all tokens; a row's number takes 16 bits.
    const uint64_t want = std::max<uint64_t>(std::max<uint64_t>(1, 296 / tiles), (vocab + 65535) / 65536);
    blocks = uint32_t(std::min(want, vocab));
    const uint64_t span = (vocab + blocks - 1) / blocks;
    shared = 2 * kFewCounts + (bulk ? kZeroBytes : 0) + (span + 31) / 32 * 4 +
             size_t(2) * 4 * ((n + kFewThreads - 1) / kFewThreads * kFewThreads);
  }
};

// Whether whole rows can be zeroed by copies of 16-byte multiples, and are wide
// enough for it.
bool bulk_rows(const Mat& out, uint64_t vocab, uint64_t dim) {
  const size_t e = type_size(out.type);
  return dim * e >= 512 && dim * e % 16 == 0 && row_aligned(out.data, out.stride, vocab, e, 16 / e);
}

}  // namespace

size_t embedding_backward_workspace(const Tokens& k, uint64_t, uint64_t dim) {
  const uint64_t n = k.rows * k.per_row;
  return n <= kFewTokens ? 0 : Layout(n, dim).bytes;
}

void embedding_backward(const Mat& grad, const Tokens& k, uint64_t vocab, uint64_t dim, float scale,
                        const Scales& s, const Mat& out, bool accumulate, void* workspace,
                        cudaStream_t stream) {
  const uint32_t n = uint32_t(k.rows * k.per_row);
  const FastDiv per_row(uint32_t(n ? k.per_row : 1));
  const Layout at(n, dim);
  char* w = static_cast<char*>(workspace);
  const auto u32 = [&](size_t offset) { return reinterpret_cast<uint32_t*>(w + offset); };
  int sorted = 0;
  Source src{k, per_row, token_step(k), uint32_t(vocab), s.data == nullptr, nullptr, nullptr};
  // One block sorts where the others have rows to zero meanwhile, for longer than
  // it takes.
  const bool beside = n <= kOneTokens && !accumulate && vocab * dim * type_size(out.type) >= 128u << 20;
  if (n > kFewTokens) {
    uint32_t* present = u32(at.totals) + kDigits;
    int passes = 1;
    while (passes < 4 && (vocab - 1) >> (8 * passes)) ++passes;
    const auto first_read = [&](auto&& f) {
      if (k.type == kI64) f(std::integral_constant<int, kTokens64>());
      else f(std::integral_constant<int, kTokens32>());
    };
    if (beside) {
      first_read([&](auto read) {
        const auto go = [&](auto items) {
          constexpr int ITEMS = decltype(items)::value;
          const auto kernel = sort_one_kernel<decltype(read)::value, ITEMS>;
          const size_t shared = size_t(kOneThreads) * ITEMS * 6 + kOneThreads / 32 * kDigits * 6;
          allow_shared(kernel, shared, shared);
          const size_t e = type_size(out.type);
          const Rows rows{static_cast<char*>(const_cast<void*>(out.data)), out.stride * int64_t(e), uint32_t(dim * e),
                          uint32_t(e), bulk_rows(out, vocab, dim)};
          kernel<<<unsigned(1 + std::min<uint64_t>(147, vocab)), kOneThreads, shared, stream>>>(
              src, n, passes, present, u32(at.keys[0]), u32(at.values[0]), rows);
        };
        if (n <= kOneThreads * 12) go(std::integral_constant<int, 12>());
        else go(std::integral_constant<int, 24>());
      });
    } else {
      const uint32_t tile = kThreads * sort_items(n), blocks = sort_blocks(n);
      const uint32_t per = blocks_for(blocks_for(n, tile), blocks) * tile, grid = blocks_for(n, per);
      for (int pass = 0; pass < passes; ++pass) {
        const auto go = [&](auto read) {
          constexpr int READ = decltype(read)::value;
          const int to = pass ? sorted ^ 1 : 0;
          sort_hist_kernel<READ><<<grid, kThreads, 0, stream>>>(src, present, n, per, pass * 8, u32(at.hist));
          // Up to 64 blocks add the counts up themselves: a launch less.
          if (grid > 64) sort_scan_kernel<<<kDigits, kThreads, 0, stream>>>(u32(at.hist), grid, u32(at.totals));
          const auto scatter = tile == kThreads * 4 ? sort_scatter_kernel<READ, 4> : sort_scatter_kernel<READ, 16>;
          scatter<<<grid, kThreads, 0, stream>>>(src, present, n, per, pass * 8, u32(at.hist),
                                                 grid > 64 ? u32(at.totals) : nullptr,
                                                 u32(at.keys[to]), u32(at.values[to]));
          sorted = to;
        };
        if (pass) go(std::integral_constant<int, kSorted>());
        else first_read(go);
        src.keys = u32(at.keys[sorted]);
        src.values = u32(at.values[sorted]);
      }
    }
  }
  with_types(grad.type, out.type, [&](auto* pt, auto* po) {
    using T = std::remove_pointer_t<decltype(pt)>;
    using O = std::remove_pointer_t<decltype(po)>;
    const T* g = static_cast<const T*>(grad.data);
    O* y = static_cast<O*>(const_cast<void*>(out.data));
    with_width<T>(grad, k.rows, out, vocab, dim, [&](auto width) {
      constexpr int VE = decltype(width)::value;
      const uint64_t pieces = dim / VE;
      if (!n) {
        const uint64_t total = vocab * pieces;
        if (!accumulate)
          zero_rows_kernel<O, VE><<<unsigned(std::min<uint64_t>((total + kThreads - 1) / kThreads, 148 * 8)), kThreads,
                                    0, stream>>>(y, out.stride, uint32_t(pieces), FastDiv(uint32_t(pieces)), total);
        return;
      }
      const bool bulk = !accumulate && bulk_rows(out, vocab, dim);
      if (n <= kFewTokens) {
        const FewPlan plan(n, vocab, pieces, bulk);
        const auto kernel = s.data ? few_kernel<T, O, VE, true> : few_kernel<T, O, VE, false>;
        allow_shared(kernel, plan.shared, FewPlan::kMostShared);
        kernel<<<dim3(plan.blocks, plan.tiles), kFewThreads, plan.shared, stream>>>(
            g, grad.stride, src, n, FastDiv(plan.blocks), s, scale, uint32_t(dim), y, out.stride, accumulate, bulk,
            plan.lg);
        return;
      }
      const SharePlan plan(n, pieces);
      const uint32_t* present = u32(at.totals) + kDigits;
      float* head = reinterpret_cast<float*>(w + at.head);
      float* tail = reinterpret_cast<float*>(w + at.tail);
      const uint32_t zero_blocks = accumulate || beside ? 0 : blocks_for(vocab, kThreads);
      const auto kernel = s.data ? share_sum_kernel<T, O, VE, true> : share_sum_kernel<T, O, VE, false>;
      kernel<<<dim3(zero_blocks + blocks_for(plan.shares, kThreads >> plan.lg), plan.tiles), kThreads, 0, stream>>>(
          g, grad.stride, u32(at.keys[sorted]), u32(at.values[sorted]), present, plan.share, uint32_t(vocab), per_row,
          s, scale, uint32_t(dim), y, out.stride, accumulate, head, tail, plan.lg, zero_blocks, bulk);
      constexpr int JOIN = VE >= 4 ? 4 : VE;
      if (plan.shares > 1)
        join_kernel<O, JOIN><<<dim3(blocks_for(plan.shares, kWarps), blocks_for(dim, 32 * JOIN)), kThreads, 0,
                               stream>>>(
            u32(at.keys[sorted]), present, plan.share, scale, uint32_t(dim), y, out.stride, accumulate, head, tail);
    });
  });
  XGBB_CUDA(cudaGetLastError());
}

}  // namespace xgbb::nn
