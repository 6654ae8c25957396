// Stable counting / radix sort of row numbers (see keysort.h).
//
// place(i) = #{j : key_j < key_i} + #{j < i : key_j = key_i}: unique, so the result does not depend on how threads are
// scheduled and everything summed in this order repeats bit for bit.  Up to kPairItems items one CTA counts pairs; up to
// kClusterItems one cluster does all radix passes in one launch; beyond, each pass is three kernels: digit counts of
// every tile, a scan of those counts over the tiles, and the scatter.  One pass, B200, us back to back in a graph:
//   items        300   4096   8192  16384  32768  65536  131072  262144
//   cluster      3.2    3.5    4.4    5.0    5.9    8.1                    (64 keys; 500 keys: 4.0 .. 10.4)
//   tiles                           10.8   10.6   10.9    11.7    15.7    (500 keys: 12 .. 17)
// (one CTA's shared memory instead of the cluster: 5.4 at 300 items, 10.8 at 4096.)
#include "keysort.h"

#include <cooperative_groups.h>

#include <atomic>

#include "core.cuh"
#include "plan.h"

namespace thcb {
namespace {

// launch_pdl for clusters of `cluster` CTAs.
template <typename... KArgs, typename... Args>
cudaError_t launch_pdl_cluster(void (*kernel)(KArgs...), unsigned cluster, dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args &&...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

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

__device__ __forceinline__ uint32_t key_of(const KeySource &s, int64_t raw) {
  const int64_t k = raw - 1;          // positions are 1-based (TH_INDEX_BASE)
  const bool row = (uint64_t)k < (uint64_t)s.limit;
  if (!row && s.errors && !(raw == 0 && s.zero_is_none) && !(raw == s.skip && s.skip != 0)) atomicAdd(s.errors, 1u);
  return (row && !(raw == s.skip && s.skip != 0)) ? (uint32_t)k : (uint32_t)s.limit;
}
__device__ __forceinline__ uint32_t source_key(const KeySource &s, int64_t i) { return s.key ? s.key[i] : key_of(s, s.index[i * s.stride]); }
// A thread's items first, first + step, ... below n, all loads in flight together; 0 for the others.
template <int ROUNDS>
__device__ __forceinline__ void source_keys(uint32_t (&key)[ROUNDS], const KeySource &s, int64_t first, int64_t step, int64_t n) {
  if (s.key) {
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) key[r] = first + r * step < n ? __ldcg(s.key + first + r * step) : 0;
    return;
  }
  constexpr int B = ROUNDS < 8 ? ROUNDS : 8;
#pragma unroll
  for (int r0 = 0; r0 < ROUNDS; r0 += B) {
    int64_t raw[B];
#pragma unroll
    for (int u = 0; u < B; ++u) raw[u] = first + (r0 + u) * step < n ? s.index[(first + (r0 + u) * step) * s.stride] : 0;
#pragma unroll
    for (int u = 0; u < B; ++u) key[r0 + u] = first + (r0 + u) * step < n ? key_of(s, raw[u]) : 0;
  }
}

// Counts of every digit in a tile: hist[tile][bin].
__global__ void __launch_bounds__(kTileThreads)
tile_hist_kernel(KeySource src, uint32_t *hist, int64_t n, int shift, uint32_t bins) {
  pdl_prologue();
  extern __shared__ uint32_t sm[];
  for (uint32_t b = threadIdx.x; b < bins; b += kTileThreads) sm[b] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kTileItems;
  uint32_t key[kTileItems / kTileThreads];
  source_keys<kTileItems / kTileThreads>(key, src, base + threadIdx.x, kTileThreads, n);
#pragma unroll
  for (int r = 0; r < kTileItems / kTileThreads; ++r)
    if (base + r * kTileThreads + threadIdx.x < n) atomicAdd(&sm[(key[r] >> shift) & (bins - 1)], 1u);
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

// Lanes of the warp with the same digit, among the live ones.  One vote per bit: the match instruction serves one distinct
// value after the other and took 160 cycles a warp here, 8 bits of votes take about 35 issue slots.
template <int BITS>
__device__ __forceinline__ uint32_t lanes_with(uint32_t digit, bool live) {
  uint32_t peers = __ballot_sync(~0u, live);
#pragma unroll
  for (int b = 0; b < BITS; ++b) {
    const uint32_t mine = (uint32_t)((int32_t)(digit << (31 - b)) >> 31);   // all ones or none
    peers &= ~(__ballot_sync(~0u, mine != 0) ^ mine);
  }
  return peers;
}

// A warp's stable ranks: item r of lane l (item number first + r * 32 + l) gets the count of equal digits in front of it
// among the warp's items.  `count` holds the warp's counters, `stride` apart and zero at the start.
template <int BITS, int ROUNDS, typename C>
__device__ __forceinline__ void warp_ranks_of(const uint32_t (&key)[ROUNDS], int shift, int64_t first, int64_t n, uint32_t (&rank)[ROUNDS], C *count,
                                              uint32_t stride) {
  const uint32_t lane = threadIdx.x & 31, below = (1u << lane) - 1;
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const bool live = first + r * 32 < n;
    const uint32_t d = (key[r] >> shift) & ((1u << BITS) - 1);
    const uint32_t peers = lanes_with<BITS>(d, live);
    uint32_t seen = 0;
    if (live) seen = count[d * stride];
    __syncwarp();
    rank[r] = seen + __popc(peers & below);
    if (live && (peers & below) == 0) count[d * stride] = (C)(seen + __popc(peers));
    __syncwarp();
  }
}
// One unrolled form for each width of a digit (2^11 = kSortMaxBins).
template <int ROUNDS, typename C>
__device__ __forceinline__ void warp_ranks(const uint32_t (&key)[ROUNDS], int shift, int bits, int64_t first, int64_t n, uint32_t (&rank)[ROUNDS], C *count,
                                           uint32_t stride) {
  switch (bits) {
#define THCB_RANKS(B) case B: warp_ranks_of<B, ROUNDS, C>(key, shift, first, n, rank, count, stride); break;
    THCB_RANKS(1) THCB_RANKS(2) THCB_RANKS(3) THCB_RANKS(4) THCB_RANKS(5) THCB_RANKS(6) THCB_RANKS(7) THCB_RANKS(8) THCB_RANKS(9) THCB_RANKS(10)
    THCB_RANKS(11)
#undef THCB_RANKS
  }
}

// Moves a tile's items to their places.  SLOTS: the single pass of sort_to_slots; otherwise a radix pass.
template <bool SLOTS>
__global__ void __launch_bounds__(kTileThreads)
tile_scatter_kernel(KeySource src, const uint32_t *hist, const uint32_t *totals, uint32_t *out_key, uint32_t *out_pos,
                    uint32_t *zero, int64_t *slot, int64_t *order, int64_t *offsets, int64_t n, int shift, uint32_t bins, int last) {
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
  uint32_t key[R], rank[R];
  source_keys<R>(key, src, base, 32, n);
  warp_ranks<R>(key, shift, 31 - __clz(bins), base, n, rank, count + warp * bins, 1);
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
    const int64_t i = base + r * 32;
    if (i >= n) continue;
    const uint32_t p = count[warp * bins + ((key[r] >> shift) & (bins - 1))] + rank[r];
    if constexpr (SLOTS) {
      const bool routed = p < none;
      slot[i] = routed ? (int64_t)p + 1 : 0;
      order[p] = routed ? i + 1 : 0;
    } else {
      out_key[p] = key[r];
      out_pos[p] = src.pos ? src.pos[i] : (uint32_t)i;
    }
  }
  if (!SLOTS && last && blockIdx.x == 0 && threadIdx.x == 0) {
    out_key[n] = 0xffffffffu;
    *zero = 0;
  }
}

// ---- one CTA -----------------------------------------------------------------------------------
constexpr int kPairItems = 256;
// Up to kPairItems items: each thread counts the pairs its item comes after.
template <bool SLOTS>
__global__ void __launch_bounds__(kPairItems)
pair_sort_kernel(KeySource src, uint32_t *out_key, uint32_t *out_pos, uint32_t *zero, int64_t *slot, int64_t *order, int64_t *offsets, uint32_t n) {
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
    if (threadIdx.x == 0) {
      out_key[n] = 0xffffffffu;
      *zero = 0;
    }
  }
}

// ---- one cluster -------------------------------------------------------------------------------
// Up to kClusterItems items: eight or sixteen CTAs that wait for one another in hardware, so that all passes fit one launch.
// Sixteen (more than every GPU grants a cluster, hence the function attribute) where eight would take a second round: a pass is
// bound by its instructions, about 100 per warp and round.  Each CTA holds an equal share of the items; between the passes
// they go straight to the shared memory of the CTA that holds their place, digit counts are read from there as well.  (With
// the items in global memory between the passes, and 1024 to a CTA however few there were, lookup gradients took 19.1 us in place
// of 16.8 for 1419 tokens of 3008 halves, 29.2 in place of 27.8 for 5003 of 1001 floats.)
// In the last pass a CTA first puts its items in order in its own shared memory and then writes each digit's run side by
// side: with eight or sixteen SMs the rate of scattered stores is part of what a pass waits for.
constexpr int kClusterFew = 8, kClusterMany = 16;
constexpr int kClusterThreads = 1024;      // or half as many, where they have no more items than that
constexpr int kClusterMaxRounds = 4;
constexpr int64_t kClusterItems = (int64_t)kClusterMany * kClusterThreads * kClusterMaxRounds;
constexpr int kClusterBins = 1 << kMaxDigitBits;
static_assert(kClusterBins <= kClusterThreads / 2, "a thread per bin");

template <bool SLOTS, int ROUNDS>
__global__ void __launch_bounds__(kClusterThreads)
cluster_sort_kernel(KeySource src, uint32_t *out_key, uint32_t *out_pos, uint32_t *zero, int64_t *slot, int64_t *order, int64_t *offsets, uint32_t n,
                    FastDiv32 share, int passes, int digit_bits) {
  pdl_prologue();
  cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  extern __shared__ uint4 cluster_smem[];
  const uint32_t threads = blockDim.x, warps = threads >> 5, per_cta = share.d;
  uint64_t *const held = reinterpret_cast<uint64_t *>(cluster_smem);          // items that came from the pass before: position above key
  uint32_t *const skey = reinterpret_cast<uint32_t *>(held + (SLOTS ? 0 : ROUNDS * threads)), *const spos = skey + ROUNDS * threads;
  __shared__ __align__(16) uint16_t count[kClusterThreads / 32 * kClusterBins];   // at most 4096 equal digits in a CTA
  __shared__ uint32_t total[kClusterBins], base[kClusterBins], local[kClusterBins], warp_sums[2][32];
  const uint32_t cta = cluster.block_rank(), ctas = cluster.num_blocks(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t bins = 1u << digit_bits;
  const uint32_t begin = min(cta * per_cta, n), end = min(begin + per_cta, n);
  const uint32_t first = begin + warp * (ROUNDS * 32) + lane;                  // a warp's items are consecutive
  for (int p = 0;; ++p) {
    const int shift = p * digit_bits;
    const bool last = p == passes - 1;
    uint32_t key[ROUNDS], pos[ROUNDS], rank[ROUNDS];
    if (p == 0) {
      source_keys<ROUNDS>(key, src, first, 32, end);
#pragma unroll
      for (int r = 0; r < ROUNDS; ++r) pos[r] = first + r * 32;
    } else {
#pragma unroll
      for (int r = 0; r < ROUNDS; ++r) {
        const uint64_t x = first + r * 32 < end ? held[first - begin + r * 32] : 0;
        key[r] = (uint32_t)x;
        pos[r] = (uint32_t)(x >> 32);
      }
    }
    for (uint32_t i = threadIdx.x; i < warps * bins / 8; i += threads) reinterpret_cast<uint4 *>(count)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    uint16_t *mine = count + warp * bins;
    warp_ranks<ROUNDS>(key, shift, digit_bits, first, end, rank, mine, 1);
    __syncthreads();
    const uint32_t b = threadIdx.x;
    if (b < bins) {
      uint32_t run = 0;
#pragma unroll 8
      for (uint32_t w = 0; w < warps; ++w) {
        const uint32_t c = count[w * bins + b];
        count[w * bins + b] = (uint16_t)run;
        run += c;
      }
      total[b] = run;
    }
    cluster.sync();                 // totals are there, and what each CTA held is in its registers
    uint32_t before = 0, all = 0, here = 0;
    if (b < bins) {
      here = total[b];
      for (uint32_t c0 = 0; c0 < ctas; c0 += kClusterFew) {
        uint32_t t[kClusterFew];
#pragma unroll
        for (int u = 0; u < kClusterFew; ++u) t[u] = cluster.map_shared_rank(total, c0 + u)[b];
#pragma unroll
        for (int u = 0; u < kClusterFew; ++u) {
          if (c0 + u < cta) before += t[u];
          all += t[u];
        }
      }
    }
    // exclusive scans of the bins' totals, of the cluster and of this CTA: one bin a thread
    uint32_t incl = all, incl_here = here;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(~0u, incl, d), h = __shfl_up_sync(~0u, incl_here, d);
      if (lane >= (uint32_t)d) {
        incl += o;
        incl_here += h;
      }
    }
    if (lane == 31) {
      warp_sums[0][warp] = incl;
      warp_sums[1][warp] = incl_here;
    }
    __syncthreads();
    if (last) cluster.barrier_arrive();             // nobody reads the others' totals any more
    uint32_t front = 0, front_here = 0;
#pragma unroll
    for (int w = 0; w < kClusterBins / 32; ++w) {
      front += w < (int)warp ? warp_sums[0][w] : 0;
      front_here += w < (int)warp ? warp_sums[1][w] : 0;
    }
    if (b < bins) {
      const uint32_t start = front + incl - all;
      local[b] = front_here + incl_here - here;
      base[b] = start + before - (last ? local[b] : 0);   // place of the CTA's first item of this bin; last: less its place here
      if (SLOTS && cta == 0 && b <= (uint32_t)src.limit) offsets[b] = (int64_t)start;
    }
    __syncthreads();
    if (!last) {
#pragma unroll
      for (int r = 0; r < ROUNDS; ++r) {
        if (first + r * 32 >= end) continue;
        const uint32_t d = (key[r] >> shift) & (bins - 1);
        uint32_t owner, at;
        share.divmod(base[d] + mine[d] + rank[r], owner, at);
        cluster.map_shared_rank(held, owner)[at] = (uint64_t)pos[r] << 32 | key[r];
      }
      cluster.sync();               // everything is in place for the next pass, and nobody reads this CTA's totals any more
      continue;
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const uint32_t i = first + r * 32;
      if (i >= end) continue;
      const uint32_t d = (key[r] >> shift) & (bins - 1), x = local[d] + mine[d] + rank[r];
      skey[x] = key[r];
      spos[x] = pos[r];
      if constexpr (SLOTS) slot[i] = key[r] < (uint32_t)src.limit ? (int64_t)(base[d] + x) + 1 : 0;   // a single pass: item i is choice i
    }
    __syncthreads();
    for (uint32_t x = threadIdx.x; x < end - begin; x += threads) {
      const uint32_t k = skey[x], q = base[(k >> shift) & (bins - 1)] + x;
      if constexpr (SLOTS) {
        order[q] = k < (uint32_t)src.limit ? (int64_t)spos[x] + 1 : 0;
      } else {
        out_key[q] = k;
        out_pos[q] = spos[x];
      }
    }
    break;
  }
  if (!SLOTS && cta == 0 && threadIdx.x == 0) {
    out_key[n] = 0xffffffffu;
    *zero = 0;
  }
  cluster.barrier_wait();
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
int launch_cluster(const SortInput &in, uint32_t *out_key, uint32_t *out_pos, uint32_t *zero, int64_t *slot, int64_t *order, int64_t *offsets, int passes,
                   int digit_bits, cudaStream_t st) {
  const KeySource src = first_source(in, true);
  const uint32_t n = (uint32_t)in.n, ctas = n <= kClusterFew * kClusterThreads ? kClusterFew : kClusterMany;
  const uint32_t each = (n + ctas - 1) / ctas, threads = each <= kClusterThreads / 2 ? kClusterThreads / 2 : kClusterThreads;
  auto launch = [&](auto kernel, uint32_t rounds) -> int {
    const uint32_t share = (each + 32 * rounds - 1) / (32 * rounds) * (32 * rounds);
    const size_t smem = (size_t)rounds * threads * (SLOTS ? 8 : 16);
    if (smem + 40960 > 48 * 1024) THCB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    if (ctas > kClusterFew) THCB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    THCB_CUDA_TRY(launch_pdl_cluster(kernel, ctas, ctas, threads, smem, st, src, out_key, out_pos, zero, slot, order, offsets, n, FastDiv32(share), passes,
                                     digit_bits));
    return 0;
  };
  const int rc = each <= kClusterThreads ? launch(cluster_sort_kernel<SLOTS, 1>, 1) : each <= 2 * kClusterThreads ? launch(cluster_sort_kernel<SLOTS, 2>, 2)
                                                                                                            : launch(cluster_sort_kernel<SLOTS, 4>, 4);
  if (rc) return rc;
  count_launch();
  THCB_CUDA_TRY(cudaGetLastError());
  return 0;
}

}  // namespace

// Items that one cluster takes on the current device: all kClusterItems where it grants clusters of kClusterMany CTAs, which
// not every partition of a GPU need do; the portable size otherwise.
static int64_t cluster_items() {
  static std::atomic<int> granted[64];              // per device: 0 not asked, 1 yes, 2 no
  int d = 0;
  if (cudaGetDevice(&d) != cudaSuccess || d < 0 || d >= 64) { cudaGetLastError(); return kClusterFew * kClusterThreads; }
  int g = granted[d].load(std::memory_order_relaxed);
  if (g == 0) {
    auto kernel = cluster_sort_kernel<false, kClusterMaxRounds>;
    const size_t smem = (size_t)kClusterMaxRounds * kClusterThreads * 16;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = kClusterMany;
    cfg.blockDim = kClusterThreads;
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kClusterMany;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    const bool ok = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) == cudaSuccess &&
                    cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                    cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) == cudaSuccess && clusters > 0;
    if (!ok) cudaGetLastError();
    g = ok ? 1 : 2;
    granted[d].store(g, std::memory_order_relaxed);
  }
  return g == 1 ? kClusterItems : (int64_t)kClusterFew * kClusterThreads;
}

size_t sort_by_key_bytes(int64_t n, int64_t) {
  if (n <= kPairItems) return 0;
  const size_t bins = 1u << kMaxDigitBits;
  return n <= cluster_items() ? 0 : align256((size_t)tiles_of(n) * bins * 4) + align256(bins * 4) + 2 * align256(((size_t)n + 1) * 4);
}

int sort_by_key(const SortInput &in, uint32_t *out_key, uint32_t *out_pos, uint32_t *zero, void *ws, cudaStream_t st) {
  const int bits = bits_of(in.limit);   // keys 0 .. limit
  if (in.n <= kPairItems) {
    launch_pdl(pair_sort_kernel<false>, 1, kPairItems, 0, st, first_source(in, true), out_key, out_pos, zero, (int64_t *)nullptr, (int64_t *)nullptr,
               (int64_t *)nullptr, (uint32_t)in.n);
    count_launch();
    THCB_CUDA_TRY(cudaGetLastError());
    return 0;
  }
  const int passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits, digit_bits = (bits + passes - 1) / passes;
  const uint32_t bins = 1u << digit_bits;
  const int64_t tiles = tiles_of(in.n);
  char *w = (char *)ws;
  if (in.n <= cluster_items()) return launch_cluster<false>(in, out_key, out_pos, zero, nullptr, nullptr, nullptr, passes, digit_bits, st);
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
               (const uint32_t *)totals, dk, dp, zero, (int64_t *)nullptr, (int64_t *)nullptr, (int64_t *)nullptr, in.n, shift, bins, p == passes - 1 ? 1 : 0);
    count_launch(3);
    THCB_CUDA_TRY(cudaGetLastError());
    src.key = dk;
    src.pos = dp;
  }
  return 0;
}

size_t sort_to_slots_bytes(int64_t n, int64_t limit) {
  if (n <= kPairItems || (n <= cluster_items() && limit < kClusterBins)) return 0;
  const size_t bins = pow2_at_least((uint32_t)limit + 1);
  return align256((size_t)tiles_of(n) * bins * 4) + align256(bins * 4);
}

int sort_to_slots(const SortInput &in, int64_t *slot, int64_t *order, int64_t *offsets, void *ws, cudaStream_t st) {
  if (in.n <= kPairItems) {
    launch_pdl(pair_sort_kernel<true>, 1, kPairItems, 0, st, first_source(in, true), (uint32_t *)nullptr, (uint32_t *)nullptr, (uint32_t *)nullptr, slot, order, offsets,
               (uint32_t)in.n);
    count_launch();
    THCB_CUDA_TRY(cudaGetLastError());
    return 0;
  }
  const int bits = bits_of(in.limit);
  if (in.n <= cluster_items() && in.limit < kClusterBins)
    return launch_cluster<true>(in, nullptr, nullptr, nullptr, slot, order, offsets, 1, bits, st);
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
             (uint32_t *)nullptr, (uint32_t *)nullptr, (uint32_t *)nullptr, slot, order, offsets, in.n, 0, bins, 1);
  count_launch(3);
  THCB_CUDA_TRY(cudaGetLastError());
  return 0;
}

}  // namespace thcb
