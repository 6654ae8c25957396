// Stable counting / radix sort of row numbers (see keysort.h).
//
// place(i) = #{j : key_j < key_i} + #{j < i : key_j = key_i}: unique, so the result does not depend on how threads are
// scheduled and everything summed in this order repeats bit for bit.  Up to kSmallItems items one CTA does the whole
// sort (by counting pairs up to kPairItems, by radix passes in shared memory above); beyond, each pass is three
// kernels: digit counts of every tile, a scan of those counts over the tiles, and the scatter.
#include "keysort.h"

#include "core.cuh"
#include "plan.h"

namespace thcb {
namespace {

constexpr int kTileThreads = 256;
constexpr int kTileItems = 2048;      // per CTA of the tiled passes: 8 rounds of a warp
constexpr int kTileWarps = kTileThreads / 32;
constexpr int kWarpItems = kTileItems / kTileWarps;
constexpr int kMaxDigitBits = 9;      // tiled radix passes: 8 warps x 512 counters = 16 KiB of shared memory

struct KeySource {
  const int64_t *index;               // pass 0
  int64_t stride, limit, skip;
  int zero_is_none;
  unsigned int *errors;               // null: not counted (a second look at the same items)
  const uint32_t *key, *pos;          // later passes
};

__device__ __forceinline__ uint32_t source_key(const KeySource &s, int64_t i) {
  if (s.key) return s.key[i];
  const int64_t raw = s.index[i * s.stride];
  const int64_t k = raw - 1;          // positions are 1-based (TH_INDEX_BASE)
  const bool row = (uint64_t)k < (uint64_t)s.limit;
  if (!row && s.errors && !(raw == 0 && s.zero_is_none) && !(raw == s.skip && s.skip != 0)) atomicAdd(s.errors, 1u);
  return (row && !(raw == s.skip && s.skip != 0)) ? (uint32_t)k : (uint32_t)s.limit;
}

// Counts of every digit in a tile: hist[tile][bin].
__global__ void __launch_bounds__(kTileThreads)
tile_hist_kernel(KeySource src, uint32_t *hist, int64_t n, int shift, uint32_t bins) {
  pdl_prologue();
  extern __shared__ uint32_t sm[];
  for (uint32_t b = threadIdx.x; b < bins; b += kTileThreads) sm[b] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kTileItems;
#pragma unroll
  for (int r = 0; r < kTileItems / kTileThreads; ++r) {
    const int64_t i = base + r * kTileThreads + threadIdx.x;
    if (i < n) atomicAdd(&sm[(source_key(src, i) >> shift) & (bins - 1)], 1u);
  }
  __syncthreads();
  for (uint32_t b = threadIdx.x; b < bins; b += kTileThreads) hist[(size_t)blockIdx.x * bins + b] = sm[b];
}

// hist[tile][bin] -> items of the bin in earlier tiles; totals[bin] = items of the bin.  A CTA takes 32 bins, one to a
// lane, and splits the tiles over its 32 warps.
__global__ void __launch_bounds__(1024)
tile_scan_kernel(uint32_t *hist, uint32_t *totals, int tiles, uint32_t bins) {
  pdl_prologue();
  __shared__ uint32_t part[32][33];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t b = blockIdx.x * 32 + lane;
  const int per = (tiles + 31) / 32, lo = min((int)warp * per, tiles), hi = min(lo + per, tiles);
  uint32_t sum = 0;
  if (b < bins) {
#pragma unroll 4
    for (int t = lo; t < hi; ++t) sum += hist[(size_t)t * bins + b];
  }
  part[warp][lane] = sum;
  __syncthreads();
  uint32_t run = 0, all = 0;
#pragma unroll
  for (int w = 0; w < 32; ++w) {
    if (w < (int)warp) run += part[w][lane];
    all += part[w][lane];
  }
  if (b >= bins) return;
#pragma unroll 4
  for (int t = lo; t < hi; ++t) {
    const uint32_t c = hist[(size_t)t * bins + b];
    hist[(size_t)t * bins + b] = run;
    run += c;
  }
  if (warp == 0) totals[b] = all;
}

// Exclusive scan of v[0 .. count) in shared memory by one CTA of `threads` threads (a multiple of 32, at most 1024).
__device__ __forceinline__ void cta_exclusive_scan(uint32_t *v, uint32_t count, uint32_t threads, uint32_t *warp_sums) {
  const uint32_t per = (count + threads - 1) / threads;
  const uint32_t lo = min(threadIdx.x * per, count), hi = min(lo + per, count);
  uint32_t sum = 0;
  for (uint32_t i = lo; i < hi; ++i) sum += v[i];
  uint32_t incl = sum;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t o = __shfl_up_sync(~0u, incl, d);
    if (lane >= (uint32_t)d) incl += o;
  }
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  uint32_t before = 0;
  for (uint32_t w = 0; w < warp; ++w) before += warp_sums[w];
  uint32_t run = before + incl - sum;
  for (uint32_t i = lo; i < hi; ++i) {
    const uint32_t c = v[i];
    v[i] = run;
    run += c;
  }
  __syncthreads();
}

// A warp's stable ranks: item r of lane l (item number base + r * 32 + l) gets the count of equal digits in front of it
// among the warp's items.  `count` holds the warp's counters, zero at the start.
template <int ROUNDS>
__device__ __forceinline__ void warp_ranks(const uint32_t (&digit)[ROUNDS], const bool (&live)[ROUNDS], uint32_t (&rank)[ROUNDS], uint32_t *count) {
  const uint32_t lane = threadIdx.x & 31, below = (1u << lane) - 1;
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const uint32_t peers = __match_any_sync(~0u, live[r] ? digit[r] : 0xffffffffu);
    uint32_t seen = 0;
    if (live[r]) seen = count[digit[r]];
    __syncwarp();
    if (live[r]) {
      rank[r] = seen + __popc(peers & below);
      if ((peers & below) == 0) count[digit[r]] = seen + __popc(peers);
    }
    __syncwarp();
  }
}

// Moves a tile's items to their places.  SLOTS: the single pass of sort_to_slots; otherwise a radix pass.
template <bool SLOTS>
__global__ void __launch_bounds__(kTileThreads)
tile_scatter_kernel(KeySource src, const uint32_t *hist, const uint32_t *totals, uint32_t *out_key, uint32_t *out_pos,
                    int64_t *slot, int64_t *order, int64_t *offsets, int64_t n, int shift, uint32_t bins, int last) {
  pdl_prologue();
  extern __shared__ uint32_t sm[];
  __shared__ uint32_t warp_sums[32];
  uint32_t *start = sm;               // [bins]: place of the tile's first item of the bin
  uint32_t *count = sm + bins;        // [warps][bins]
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (uint32_t b = threadIdx.x; b < bins; b += kTileThreads) start[b] = totals[b];
  for (uint32_t i = threadIdx.x; i < kTileWarps * bins; i += kTileThreads) count[i] = 0;
  __syncthreads();
  cta_exclusive_scan(start, bins, kTileThreads, warp_sums);
  if constexpr (SLOTS) {
    if (blockIdx.x == 0)
      for (uint32_t b = threadIdx.x; b <= (uint32_t)src.limit; b += kTileThreads) offsets[b] = (int64_t)start[b];
  }
  const uint32_t none = SLOTS ? start[src.limit] : 0;   // items with a key
  constexpr int R = kWarpItems / 32;
  const int64_t base = (int64_t)blockIdx.x * kTileItems + warp * kWarpItems + lane;
  uint32_t key[R], pos[R], digit[R], rank[R];
  bool live[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t i = base + r * 32;
    live[r] = i < n;
    key[r] = live[r] ? source_key(src, i) : 0;
    pos[r] = live[r] && src.pos ? src.pos[i] : (uint32_t)i;
    digit[r] = (key[r] >> shift) & (bins - 1);
  }
  warp_ranks<R>(digit, live, rank, count + warp * bins);
  __syncthreads();
  for (uint32_t b = threadIdx.x; b < bins; b += kTileThreads) {
    uint32_t run = start[b] + hist[(size_t)blockIdx.x * bins + b];
#pragma unroll
    for (int w = 0; w < kTileWarps; ++w) {
      const uint32_t c = count[w * bins + b];
      count[w * bins + b] = run;
      run += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (!live[r]) continue;
    const uint32_t p = count[warp * bins + digit[r]] + rank[r];
    if constexpr (SLOTS) {
      const bool routed = p < none;
      slot[base + r * 32] = routed ? (int64_t)p + 1 : 0;
      order[p] = routed ? base + r * 32 + 1 : 0;
    } else {
      out_key[p] = key[r];
      out_pos[p] = pos[r];
    }
  }
  if (!SLOTS && last && blockIdx.x == 0 && threadIdx.x == 0) out_key[n] = 0xffffffffu;
}

// ---- one CTA -----------------------------------------------------------------------------------
constexpr int kPairItems = 256;
constexpr int kSmallThreads = 1024;
constexpr int kSmallItems = 4096;     // 4 rounds of 32 warps; 32 x 256 counters = 32 KiB of shared memory
constexpr int kSmallBins = 256;
constexpr int kSmallRounds = kSmallItems / kSmallThreads;

// Up to kPairItems items: each thread counts the pairs its item comes after.
template <bool SLOTS>
__global__ void __launch_bounds__(kPairItems)
pair_sort_kernel(KeySource src, uint32_t *out_key, uint32_t *out_pos, int64_t *slot, int64_t *order, int64_t *offsets, uint32_t n) {
  pdl_prologue();
  __shared__ uint32_t keys[kPairItems];
  const uint32_t i = threadIdx.x;
  const uint32_t mine = i < n ? source_key(src, i) : 0xffffffffu;
  keys[i] = mine;
  __syncthreads();
  uint32_t p = 0;
  for (uint32_t j = 0; j < n; ++j) {
    const uint32_t k = keys[j];
    p += (k < mine || (k == mine && j < i)) ? 1u : 0u;
  }
  if (i < n) {
    if constexpr (SLOTS) {
      const bool routed = mine < (uint32_t)src.limit;
      slot[i] = routed ? (int64_t)p + 1 : 0;
      order[p] = routed ? (int64_t)i + 1 : 0;
    } else {
      out_key[p] = mine;
      out_pos[p] = i;
    }
  }
  if constexpr (SLOTS) {
    for (uint32_t e = threadIdx.x; e <= (uint32_t)src.limit; e += blockDim.x) {
      uint32_t c = 0;
      for (uint32_t j = 0; j < n; ++j) c += keys[j] < e ? 1u : 0u;
      offsets[e] = (int64_t)c;
    }
  } else {
    if (threadIdx.x == 0) out_key[n] = 0xffffffffu;
  }
}

// Up to kSmallItems items: radix passes inside one CTA, items in shared memory between the passes.
template <bool SLOTS>
__global__ void __launch_bounds__(kSmallThreads)
small_sort_kernel(KeySource src, uint32_t *out_key, uint32_t *out_pos, int64_t *slot, int64_t *order, int64_t *offsets, uint32_t n,
                  int passes, int digit_bits) {
  pdl_prologue();
  extern __shared__ uint32_t sm[];
  __shared__ uint32_t warp_sums[32];
  const uint32_t bins = 1u << digit_bits;
  uint32_t *skey = sm, *spos = sm + kSmallItems;
  uint32_t *count = spos + kSmallItems;      // [bins][warps]: in this order the scan runs over the bins, then the warps
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, below = (1u << lane) - 1;
  constexpr uint32_t W = kSmallThreads / 32;
  uint32_t key[kSmallRounds], pos[kSmallRounds], rank[kSmallRounds];
  // a warp's items are consecutive
  const uint32_t base = warp * (kSmallRounds * 32) + lane;
#pragma unroll
  for (int r = 0; r < kSmallRounds; ++r) {
    const uint32_t i = base + r * 32;
    pos[r] = i;
    key[r] = i < n ? source_key(src, i) : 0;
  }
  for (int p = 0; p < passes; ++p) {
    const int shift = p * digit_bits;
    for (uint32_t i = threadIdx.x; i < bins * W; i += kSmallThreads) count[i] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSmallRounds; ++r) {
      const bool live = base + r * 32 < n;
      const uint32_t d = (key[r] >> shift) & (bins - 1);
      const uint32_t peers = __match_any_sync(~0u, live ? d : 0xffffffffu);
      uint32_t seen = 0;
      if (live) seen = count[d * W + warp];
      __syncwarp();
      if (live) {
        rank[r] = seen + __popc(peers & below);
        if ((peers & below) == 0) count[d * W + warp] = seen + __popc(peers);
      }
      __syncwarp();
    }
    __syncthreads();
    cta_exclusive_scan(count, bins * W, kSmallThreads, warp_sums);
    const bool last = p == passes - 1;
    if (SLOTS && last)
      for (uint32_t e = threadIdx.x; e <= (uint32_t)src.limit; e += kSmallThreads) offsets[e] = (int64_t)count[e * W];
#pragma unroll
    for (int r = 0; r < kSmallRounds; ++r) {
      if (base + r * 32 >= n) continue;
      const uint32_t q = count[((key[r] >> shift) & (bins - 1)) * W + warp] + rank[r];
      if (!last) {
        skey[q] = key[r];
        spos[q] = pos[r];
      } else if constexpr (SLOTS) {
        const bool routed = key[r] < (uint32_t)src.limit;
        slot[pos[r]] = routed ? (int64_t)q + 1 : 0;
        order[q] = routed ? (int64_t)pos[r] + 1 : 0;
      } else {
        out_key[q] = key[r];
        out_pos[q] = pos[r];
      }
    }
    if (last) break;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSmallRounds; ++r) {
      const uint32_t i = base + r * 32;
      if (i < n) { key[r] = skey[i]; pos[r] = spos[i]; }
    }
  }
  if (!SLOTS && threadIdx.x == 0) out_key[n] = 0xffffffffu;
}

int bits_of(int64_t max_key) {
  int b = 1;
  while (max_key >> b) ++b;
  return b;
}

KeySource first_source(const SortInput &in, bool count_errors) {
  KeySource s;
  s.index = in.index;
  s.stride = in.stride;
  s.limit = in.limit;
  s.skip = in.skip;
  s.zero_is_none = in.zero_is_none;
  s.errors = count_errors ? in.errors : nullptr;
  s.key = s.pos = nullptr;
  return s;
}

uint32_t pow2_at_least(uint32_t v) {
  uint32_t b = 1;
  while (b < v) b <<= 1;
  return b;
}

size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }
int64_t tiles_of(int64_t n) { return (n + kTileItems - 1) / kTileItems; }

template <bool SLOTS>
int launch_small(const SortInput &in, uint32_t *out_key, uint32_t *out_pos, int64_t *slot, int64_t *order, int64_t *offsets, int passes,
                 int digit_bits, cudaStream_t st) {
  const size_t smem = (size_t)(2 * kSmallItems + (kSmallThreads / 32) * (1 << digit_bits)) * sizeof(uint32_t);
  if (smem + 256 > 48 * 1024) THCB_CUDA_TRY(cudaFuncSetAttribute(small_sort_kernel<SLOTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  launch_pdl(small_sort_kernel<SLOTS>, 1, kSmallThreads, smem, st, first_source(in, true), out_key, out_pos, slot, order, offsets,
             (uint32_t)in.n, passes, digit_bits);
  count_launch();
  THCB_CUDA_TRY(cudaGetLastError());
  return 0;
}

}  // namespace

size_t sort_by_key_bytes(int64_t n, int64_t limit) {
  if (n <= kSmallItems) return 0;
  (void)limit;
  const size_t bins = 1u << kMaxDigitBits;
  return align256((size_t)tiles_of(n) * bins * 4) + align256(bins * 4) + 2 * align256(((size_t)n + 1) * 4);
}

int sort_by_key(const SortInput &in, uint32_t *out_key, uint32_t *out_pos, void *ws, cudaStream_t st) {
  const int bits = bits_of(in.limit);   // keys 0 .. limit
  if (in.n <= kPairItems) {
    launch_pdl(pair_sort_kernel<false>, 1, kPairItems, 0, st, first_source(in, true), out_key, out_pos, (int64_t *)nullptr, (int64_t *)nullptr,
               (int64_t *)nullptr, (uint32_t)in.n);
    count_launch();
    THCB_CUDA_TRY(cudaGetLastError());
    return 0;
  }
  if (in.n <= kSmallItems) {
    const int passes = (bits + 7) / 8;
    return launch_small<false>(in, out_key, out_pos, nullptr, nullptr, nullptr, passes, (bits + passes - 1) / passes, st);
  }
  const int passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits, digit_bits = (bits + passes - 1) / passes;
  const uint32_t bins = 1u << digit_bits;
  const int64_t tiles = tiles_of(in.n);
  char *w = (char *)ws;
  uint32_t *hist = (uint32_t *)w;
  w += align256((size_t)tiles * (1u << kMaxDigitBits) * 4);
  uint32_t *totals = (uint32_t *)w;
  w += align256((1u << kMaxDigitBits) * 4);
  uint32_t *tkey = (uint32_t *)w;
  w += align256(((size_t)in.n + 1) * 4);
  uint32_t *tpos = (uint32_t *)w;
  KeySource src = first_source(in, true);
  for (int p = 0; p < passes; ++p) {
    // the last pass ends in the output, the ones before alternate with it
    const bool to_out = ((passes - 1 - p) & 1) == 0;
    uint32_t *dk = to_out ? out_key : tkey, *dp = to_out ? out_pos : tpos;
    const int shift = p * digit_bits;
    launch_pdl(tile_hist_kernel, (unsigned)tiles, kTileThreads, bins * 4, st, src, hist, in.n, shift, bins);
    launch_pdl(tile_scan_kernel, (bins + 31) / 32, 1024, 0, st, hist, totals, (int)tiles, bins);
    src.errors = nullptr;
    launch_pdl(tile_scatter_kernel<false>, (unsigned)tiles, kTileThreads, (1 + kTileWarps) * bins * 4, st, src, (const uint32_t *)hist,
               (const uint32_t *)totals, dk, dp, (int64_t *)nullptr, (int64_t *)nullptr, (int64_t *)nullptr, in.n, shift, bins, p == passes - 1 ? 1 : 0);
    count_launch(3);
    THCB_CUDA_TRY(cudaGetLastError());
    src.key = dk;
    src.pos = dp;
  }
  return 0;
}

size_t sort_to_slots_bytes(int64_t n, int64_t limit) {
  if (n <= kPairItems || (n <= kSmallItems && limit < kSmallBins)) return 0;
  const size_t bins = pow2_at_least((uint32_t)limit + 1);
  return align256((size_t)tiles_of(n) * bins * 4) + align256(bins * 4);
}

int sort_to_slots(const SortInput &in, int64_t *slot, int64_t *order, int64_t *offsets, void *ws, cudaStream_t st) {
  if (in.n <= kPairItems) {
    launch_pdl(pair_sort_kernel<true>, 1, kPairItems, 0, st, first_source(in, true), (uint32_t *)nullptr, (uint32_t *)nullptr, slot, order, offsets,
               (uint32_t)in.n);
    count_launch();
    THCB_CUDA_TRY(cudaGetLastError());
    return 0;
  }
  const int bits = bits_of(in.limit);
  if (in.n <= kSmallItems && in.limit < kSmallBins) return launch_small<true>(in, nullptr, nullptr, slot, order, offsets, 1, bits, st);
  const uint32_t bins = pow2_at_least((uint32_t)in.limit + 1);
  const int64_t tiles = tiles_of(in.n);
  uint32_t *hist = (uint32_t *)ws, *totals = (uint32_t *)((char *)ws + align256((size_t)tiles * bins * 4));
  KeySource src = first_source(in, true);
  launch_pdl(tile_hist_kernel, (unsigned)tiles, kTileThreads, bins * 4, st, src, hist, in.n, 0, bins);
  launch_pdl(tile_scan_kernel, (bins + 31) / 32, 1024, 0, st, hist, totals, (int)tiles, bins);
  src.errors = nullptr;
  const size_t smem = (size_t)(1 + kTileWarps) * bins * 4;
  if (smem + 256 > 48 * 1024) THCB_CUDA_TRY(cudaFuncSetAttribute(tile_scatter_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  launch_pdl(tile_scatter_kernel<true>, (unsigned)tiles, kTileThreads, smem, st, src, (const uint32_t *)hist, (const uint32_t *)totals,
             (uint32_t *)nullptr, (uint32_t *)nullptr, slot, order, offsets, in.n, 0, bins, 1);
  count_launch(3);
  THCB_CUDA_TRY(cudaGetLastError());
  return 0;
}

}  // namespace thcb
