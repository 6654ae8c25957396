// Tokens sorted by the experts they are routed to, and back.
//
//   sort      expert[t, k] in 1..E (0: not routed) -> slot[t, k], order[p], offsets[e], stable by (expert, t, k)
//   dispatch  rows[slot[t, k], :] = (w[t, k] *) x[t, :]
//   combine   y[t, :] = sum over k of (w[t, k] *) rows[slot[t, k], :]
//   gradient  grad_rows[slot[t, k], :] = w[t, k] * grad_y[t, :],  grad_w[t, k] = <grad_y[t, :], rows[slot[t, k], :]>
//
// Combine without weights is the gradient of dispatch, and dispatch with weights the row part of combine's gradient.
// All four walk the tokens, not the sorted places: a token's row is read once for its k copies, sums run over k in order
// (no atomics, results repeat bit for bit), and every access to the sorted side is a whole row.  They are bound by HBM.
#include <cuda_fp16.h>

#include "context.h"
#include "core.cuh"
#include "keysort.h"
#include "plan.h"
#include "rows.cuh"

namespace thcb {
namespace {

constexpr int kRowThreads = 256;

// Routing weights and sums over k: float beside half and float, double beside double; sums as the library's reductions.
template <typename T> struct Weight { using type = float; };
template <> struct Weight<double> { using type = double; };

template <typename T> struct RouteArgs {
  T *dst;
  const T *src;            // token rows (dispatch) or sorted rows (combine)
  const int64_t *slot;     // [tokens][chosen]
  const typename Weight<T>::type *weight;
  int64_t vecs;            // vectors per row
  uint64_t per, items;     // items per token (dispatch of vectors: vectors; otherwise stretches of a row); tokens * per
  uint32_t team;           // lanes that take a stretch together: 32, or 8 or 16 where a row has no more vectors
  FastDiv32 per32;
  int chosen;
  int64_t places;          // rows on the sorted side
  int64_t dst_stride, src_stride, src_col;
  unsigned int *errors;
};

template <typename T>
__device__ __forceinline__ void split_item(const RouteArgs<T> &a, uint64_t i, int64_t *token, int64_t *part) {
  if (a.items <= 0xffffffffull) {
    uint32_t q, r;
    a.per32.divmod((uint32_t)i, q, r);
    *token = q;
    *part = r;
  } else {
    *token = (int64_t)(i / a.per);
    *part = (int64_t)(i - (uint64_t)*token * a.per);
  }
}

// Place of a slot on the sorted side, or -1; a slot that is neither 0 nor a place is counted once.
__device__ __forceinline__ int64_t place_of(int64_t slot, int64_t places, bool count, unsigned int *errors) {
  const int64_t p = slot - 1;
  if ((uint64_t)p < (uint64_t)places) return p;
  if (slot != 0 && count) atomicAdd(errors, 1u);
  return -1;
}

template <typename T, int V>
__global__ void __launch_bounds__(kRowThreads)
dispatch_kernel(RouteArgs<T> a) {
  pdl_prologue();
  const uint64_t i = (uint64_t)blockIdx.x * kRowThreads + threadIdx.x;
  if (i >= a.items) return;
  int64_t token, vec;
  split_item(a, i, &token, &vec);
  const Pack<T, V> x = load_pack<T, V>(a.src + token * a.src_stride + vec * V * a.src_col);
  for (int k = 0; k < a.chosen; ++k) {
    const int64_t p = place_of(a.slot[token * a.chosen + k], a.places, vec == 0, a.errors);
    if (p < 0) continue;
    T *q = a.dst + p * a.dst_stride + vec * V;
    if (a.weight) {
      using Math = typename TypeTraits<T>::Math;
      const Math w = (Math)a.weight[token * a.chosen + k];
      Pack<T, V> y;
#pragma unroll
      for (int e = 0; e < V; ++e) y.e[e] = from_math<T>(to_math(x.e[e]) * w);
      store_pack<T, V>(q, y);
    } else {
      store_pack<T, V>(q, x);
    }
  }
}

// Rows of single elements: a warp takes kLaneItems elements per lane, 32 apart, of a token's row, and its lanes read the
// token's slots and weights, one each: 1003 x 3 of 1021 floats 5.8 us with one element and its own slots per thread, 3.9 us so.
// Halves go by 8, as a lane moves few bytes otherwise (4 and 8: dispatch of 20000 x 2 of 2047 halves 72 and 62 us, 29625 x 2 of 151
// 13.1 and 9.9 us, combine 103 and 95, 15.6 and 13.9 us); 8 floats are too many (3.9 and 4.7 us; combine of 20000 x 4 of 2047 182 and
// 198 us).
template <typename T> constexpr int kLaneItems = sizeof(T) == 2 ? 8 : 4;
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
dispatch_single_kernel(RouteArgs<T> a) {
  using Math = typename TypeTraits<T>::Math;
  constexpr int G = kLaneItems<T>;
  pdl_prologue();
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t unit = (uint64_t)blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5);
  if (unit >= a.items) return;
  int64_t token, stretch;
  split_item(a, unit, &token, &stretch);
  const int32_t col0 = (int32_t)stretch * (32 * G) + (int32_t)lane, width = (int32_t)a.vecs;
  const T *src = a.src + token * a.src_stride + col0 * a.src_col;
  const int64_t step = 32 * a.src_col;
  T x[G];
#pragma unroll
  for (int g = 0; g < G; ++g)
    if (col0 + 32 * g < width) x[g] = src[g * step];
  for (int k0 = 0; k0 < a.chosen; k0 += 32) {
    const int k = k0 + (int)lane;
    int64_t slot = 0;
    Math weight = 1;
    if (k < a.chosen) {
      slot = a.slot[token * a.chosen + k];
      if (a.weight) weight = (Math)a.weight[token * a.chosen + k];
    }
    const int64_t place = place_of(slot, a.places, stretch == 0, a.errors);
    for (int u = 0; u < min(32, a.chosen - k0); ++u) {
      const int64_t p = __shfl_sync(~0u, place, u);
      const Math w = __shfl_sync(~0u, weight, u);
      if (p < 0) continue;
      T *q = a.dst + p * a.dst_stride + col0;
#pragma unroll
      for (int g = 0; g < G; ++g)
        if (col0 + 32 * g < width) q[32 * g] = a.weight ? from_math<T>(to_math(x[g]) * w) : x[g];
    }
  }
}

// Rows made of 16-byte vectors.  A warp (for narrow rows, a team of 8 or 16 lanes) takes stretches of tokens' rows, one after
// the other; its lanes read a token's slots and weights, one each, and hand them round.  The rows' vectors come by asynchronous
// copies into places of shared memory that belong to the lane that asked for them (no barrier), the copies of one stretch on
// their way while the one before is summed and the slots of the one after are read: 64 to 128 KiB per SM in flight without a
// register for them.  Held in registers instead, 4 rows at a time took 112 us and 8 rows (100 registers) 139 us where this takes
// 90 us (16384 tokens, 8 rows of 2048 halves each, 604 MB: 6.7 TB/s); 66 us against 49 us with 4 rows.
// BATCH rows of G vectors, a team's width apart, in a stretch: 8 vectors per lane.
constexpr int kRingSlots = 8, kRingStages = 2;
constexpr size_t kRingBytes = (size_t)kRingStages * kRingSlots * kRowThreads * 16;

template <typename T, int BATCH>
__global__ void __launch_bounds__(kRowThreads)
combine_ring_kernel(RouteArgs<T> a) {
  using Acc = typename TypeTraits<T>::Acc;
  using W = typename Weight<T>::type;
  constexpr int V = 16 / sizeof(T), G = kRingSlots / BATCH;
  extern __shared__ Bytes16 ring[];        // [stage][slot][thread]
  pdl_prologue();
  const uint32_t team = a.team, lane = threadIdx.x & (team - 1), teams = 32 / team;
  const uint64_t stride = (uint64_t)gridDim.x * (kRowThreads / 32) * teams;
  struct Item {                            // a batch of choices of a stretch
    uint64_t unit;
    int64_t token, stretch;
    int k0;
    uint32_t valid;                        // choices of the batch that have a place
    int64_t slot;                          // the lane's choice
    W weight;
  };
  auto read = [&](Item &x) {               // the item's slots and weights; nothing behind the last item
    x.slot = 0;
    x.weight = 1;
    x.token = x.stretch = 0;
    if (x.unit >= a.items) return;
    split_item(a, x.unit, &x.token, &x.stretch);
    const int k = x.k0 + (int)lane;
    if (lane < BATCH && k < a.chosen) {
      x.slot = a.slot[x.token * a.chosen + k];
      if (a.weight) x.weight = a.weight[x.token * a.chosen + k];
    }
  };
  auto after = [&](const Item &x) {
    Item y;
    y.unit = x.unit;
    y.k0 = x.k0 + BATCH;
    if (y.k0 >= a.chosen) {
      y.unit += stride;
      y.k0 = 0;
    }
    read(y);
    return y;
  };
  auto copy = [&](Item &x, int stage) {
    const int place = (int)place_of(x.slot, a.places, x.stretch == 0, a.errors);      // no slot behind the last item
    x.valid = __ballot_sync(~0u, place >= 0) >> (threadIdx.x & 31 & ~(team - 1));
    const int64_t vec0 = x.stretch * (team * G) + lane;
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int p = __shfl_sync(~0u, place, u, team);
      if (p < 0) continue;
      const T *row = a.src + p * a.src_stride + vec0 * V;
#pragma unroll
      for (int g = 0; g < G; ++g)
        if (vec0 + team * g < a.vecs)
          copy_async<T, V>(&ring[(stage * kRingSlots + u * G + g) * kRowThreads + threadIdx.x], row + team * g * V);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  Acc acc[G][V];
  auto sum = [&](const Item &x, int stage) {
    if (x.k0 == 0) {
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int e = 0; e < V; ++e) acc[g][e] = 0;
    }
    const int64_t vec0 = x.stretch * (team * G) + lane;
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const Acc w = (Acc)__shfl_sync(~0u, x.weight, u, team);
      if (!(x.valid >> u & 1)) continue;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (vec0 + team * g >= a.vecs) continue;
        const Bytes16 b = ring[(stage * kRingSlots + u * G + g) * kRowThreads + threadIdx.x];
        Pack<T, V> v;
        memcpy(&v, &b, 16);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[g][e] += (Acc)to_math(v.e[e]) * w;
      }
    }
    if (x.k0 + BATCH < a.chosen || x.unit >= a.items) return;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (vec0 + team * g >= a.vecs) continue;
      Pack<T, V> y;
#pragma unroll
      for (int e = 0; e < V; ++e) y.e[e] = round_from<T>(acc[g][e]);
      store_pack<T, V>(a.dst + x.token * a.dst_stride + (vec0 + team * g) * V, y);
    }
  };
  Item now, next;
  now.unit = ((uint64_t)blockIdx.x * kRowThreads + threadIdx.x) / team;
  now.k0 = 0;
  read(now);
  copy(now, 0);
  next = after(now);
  // all teams of a warp go as far as its first, which never has fewer items than they
  for (int stage = 0; __shfl_sync(~0u, now.unit, 0) < a.items; stage ^= 1) {
    copy(next, stage ^ 1);
    const Item third = after(next);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    sum(now, stage);
    now = next;
    next = third;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Other rows: single elements, G per lane and row, 32 apart, of BATCH rows at a time.
// UNIT: neighbouring columns, whose addresses are constants apart (20000 x 2 of 2047 halves 95 -> 71 us, 29625 x 2 of 151 13.9 -> 9.3 us).
template <typename T, int BATCH, bool UNIT>
__global__ void __launch_bounds__(kRowThreads)
combine_kernel(RouteArgs<T> a) {
  using Acc = typename TypeTraits<T>::Acc;
  constexpr int G = kLaneItems<T>;
  pdl_prologue();
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t unit = (uint64_t)blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5);
  if (unit >= a.items) return;
  int64_t token, stretch;
  split_item(a, unit, &token, &stretch);
  const int32_t col0 = (int32_t)stretch * (32 * G) + (int32_t)lane, width = (int32_t)a.vecs;
  const T *src = a.src + (UNIT ? (int64_t)col0 : col0 * a.src_col);
  const int64_t step = UNIT ? 32 : 32 * a.src_col;
  Acc acc[G];
#pragma unroll
  for (int g = 0; g < G; ++g) acc[g] = 0;
  for (int k0 = 0; k0 < a.chosen; k0 += BATCH) {
    const int k = k0 + (int)lane;
    const bool mine = lane < BATCH && k < a.chosen;
    const int64_t slot = mine ? a.slot[token * a.chosen + k] : 0;
    const typename Weight<T>::type weight = mine && a.weight ? a.weight[token * a.chosen + k] : 1;
    const int place = (int)place_of(slot, a.places, stretch == 0, a.errors);
    T x[BATCH][G];
    int p[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      p[u] = __shfl_sync(~0u, place, u);
      if (p[u] < 0) continue;
      const T *row = src + p[u] * a.src_stride;
#pragma unroll
      for (int g = 0; g < G; ++g)
        if (col0 + 32 * g < width) x[u][g] = row[g * step];
    }
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const Acc w = (Acc)__shfl_sync(~0u, weight, u);
      if (p[u] < 0) continue;
#pragma unroll
      for (int g = 0; g < G; ++g) acc[g] += (Acc)to_math(x[u][g]) * w;
    }
  }
  T *dst = a.dst + token * a.dst_stride + col0;
#pragma unroll
  for (int g = 0; g < G; ++g)
    if (col0 + 32 * g < width) dst[32 * g] = round_from<T>(acc[g]);
}

template <typename T> struct CombineGradArgs {
  T *grad_rows;                                // may be null
  typename Weight<T>::type *grad_weight;       // may be null
  const T *grad, *rows;
  const int64_t *slot;
  const typename Weight<T>::type *weight;      // may be null: ones
  uint64_t pairs;
  int64_t vecs;
  FastDiv32 chosen;
  uint32_t team_bits;                          // 2^team_bits lanes take a pair together
  int64_t places;
  int64_t out_stride, grad_stride, grad_col, rows_stride, rows_col;
  unsigned int *errors;
};

// A single element by a load that stays where it is written: the compiler otherwise sinks a batch's loads to their uses.
template <typename T> __device__ __forceinline__ T load_single(const T *p) {
  T x;
  if constexpr (sizeof(T) == 2) {
    uint16_t b;
    asm volatile("ld.global.u16 %0, [%1];" : "=h"(b) : "l"(p));
    memcpy(&x, &b, 2);
  } else if constexpr (sizeof(T) == 4) {
    uint32_t b;
    asm volatile("ld.global.u32 %0, [%1];" : "=r"(b) : "l"(p));
    memcpy(&x, &b, 4);
  } else {
    uint64_t b;
    asm volatile("ld.global.u64 %0, [%1];" : "=l"(b) : "l"(p));
    memcpy(&x, &b, 8);
  }
  return x;
}

// A warp (for narrow rows, a team of 4, 8 or 16 lanes) per (token, choice): the token's gradient row is read by the warps of its
// choices, which sit side by side in the CTA, so all but the first find it in the L1.  16384 tokens x 4 of 2048 halves, 577 MB:
// 88 us, 6.5 TB/s (116 us while the compiler kept two vectors in flight).  Rows of single elements are bound by instructions: a
// step between loads that is added, not multiplied out in 64 bits, took 29625 x 2 x 151 halves from 72 to 36 us.
// Of those, rows of more than 8 elements per lane have 8 in flight: 4 and 8 take 8.5 and 6.7 us (1003 x 3 x 1021 floats), 112.5 and
// 98 us (20000 x 2 x 2047 halves), but 18.4 and 21.0 us (29625 x 2 x 151 halves); doubles 51.0 and 56.8 us (5000 x 4 x 777).
template <typename T, int V, bool ROWS, bool DOT, bool TEAMS, bool LONG>
__global__ void __launch_bounds__(kRowThreads)
combine_grad_kernel(CombineGradArgs<T> a) {
  using Acc = typename TypeTraits<T>::Acc;
  using Math = typename TypeTraits<T>::Math;
  // vectors of each row in flight per lane (2 of 32 bytes 140 us, 4 157 us, 16384 x 4 x 2048 half; doubles, whose few pairs leave
  // few warps, 127 us with 4 and 140 us with 2 at 567 x 8 x 5632)
  constexpr int B = LONG ? 8 : V == 1 || (V * sizeof(T) == 32 && sizeof(T) == 8) ? 4 : 2;
  pdl_prologue();
  const uint32_t team_bits = TEAMS ? a.team_bits : 5, team = 1u << team_bits, lane = threadIdx.x & (team - 1);
  const uint64_t pair = ((uint64_t)blockIdx.x * kRowThreads + threadIdx.x) >> team_bits;
  if (((uint64_t)blockIdx.x * kRowThreads + (threadIdx.x & ~31u)) >> team_bits >= a.pairs) return;   // whole warps
  const bool there = pair < a.pairs;
  const int64_t token = there ? a.chosen.div((uint32_t)pair) : 0;
  const int64_t p = there ? place_of(a.slot[pair], a.places, lane == 0, a.errors) : -1;
  Acc dot = 0;
  if (p >= 0) {
    const Math w = a.weight ? (Math)a.weight[pair] : (Math)1;
    const T *g = a.grad + token * a.grad_stride + (int64_t)lane * V * a.grad_col, *r = a.rows + p * a.rows_stride + (int64_t)lane * V * a.rows_col;
    T *o = ROWS ? a.grad_rows + p * a.out_stride + lane * V : nullptr;
    const int64_t g_step = (int64_t)team * V * a.grad_col, r_step = (int64_t)team * V * a.rows_col;
    for (int32_t left = (int32_t)a.vecs - (int32_t)lane; left > 0; left -= (int32_t)team * B) {
      Pack<T, V> x[B], y[DOT ? B : 1];
#pragma unroll
      for (int u = 0; u < B; ++u) {
        if (left <= (int32_t)team * u) continue;
        if constexpr (V == 1) {
          x[u].e[0] = load_single(g + u * g_step);
          if (DOT) y[u].e[0] = load_single(r + u * r_step);
        } else {
          x[u] = load_kept<T, V>(g + u * g_step);
          if (DOT) y[u] = load_pack<T, V>(r + u * r_step);
        }
      }
#pragma unroll
      for (int u = 0; u < B; ++u) {
        if (left <= (int32_t)team * u) continue;
        if (DOT) {
#pragma unroll
          for (int e = 0; e < V; ++e) dot += (Acc)to_math(x[u].e[e]) * (Acc)to_math(y[u].e[e]);
        }
        if (ROWS) {
          Pack<T, V> z;
#pragma unroll
          for (int e = 0; e < V; ++e) z.e[e] = from_math<T>(to_math(x[u].e[e]) * w);
          store_pack<T, V>(o + u * team * V, z);
        }
      }
      g += B * g_step;
      if (DOT) r += B * r_step;
      if (ROWS) o += (int64_t)B * team * V;
    }
  }
  if (!DOT) return;
#pragma unroll
  for (uint32_t d = 16; d > 0; d >>= 1)
    if (d < team) dot += __shfl_xor_sync(~0u, dot, d);
  if (lane == 0 && there) a.grad_weight[pair] = (typename Weight<T>::type)dot;
}

// ---- host --------------------------------------------------------------------------------------
struct SlotView {
  const int64_t *data;
  int64_t tokens, chosen;
};

bool dense(const HostView &v) {
  int64_t run = 1;
  for (int d = v.ndim - 1; d >= 0; --d) {
    if (v.sizes[d] != 1 && v.strides[d] != run) return false;
    run *= v.sizes[d];
  }
  return true;
}

int slot_view(const thcb200_tensor *t, SlotView *s, const char *what) {
  HostView v;
  const int rc = to_host_view(t, &v, what);
  if (rc) return rc;
  if (v.dtype != THCB200_I64 || v.ndim != 2 || !dense(v)) { set_error("%s: expected a contiguous matrix of I64", what); return THCB200_ERR_ARG; }
  s->data = (const int64_t *)v.data;
  s->tokens = v.sizes[0];
  s->chosen = v.sizes[1];
  if (s->chosen > kSortMaxItems || (s->chosen > 0 && s->tokens > kSortMaxItems / s->chosen)) { set_error("%s: more than 2^31 choices", what); return THCB200_ERR_LIMIT; }
  return 0;
}

// A routing weight matrix shaped like the slots, in the type that goes with the rows' type.
int weight_view(const thcb200_tensor *t, int rows_dtype, const SlotView &s, void **data, const char *what) {
  *data = nullptr;
  if (!t) return 0;
  HostView v;
  const int rc = to_host_view(t, &v, what);
  if (rc) return rc;
  if (v.dtype != (rows_dtype == THCB200_F64 ? THCB200_F64 : THCB200_F32)) { set_error("%s: weights are F32, or F64 beside F64 rows", what); return THCB200_ERR_ARG; }
  if (v.ndim != 2 || !dense(v)) { set_error("%s: expected a contiguous matrix", what); return THCB200_ERR_ARG; }
  if (v.sizes[0] != s.tokens || v.sizes[1] != s.chosen) { set_error("%s: weights and slots differ in size", what); return THCB200_ERR_SIZE; }
  *data = v.data;
  return 0;
}

template <typename T>
int run_route(thcb200_ctx *ctx, bool dispatch, const MatView &dst, const MatView &src, const SlotView &s, const void *weight, cudaStream_t st) {
  constexpr int VB = 16 / sizeof(T);
  const bool vec = mat_vec(dst, sizeof(T), 16) && mat_vec(src, sizeof(T), 16);
  RouteArgs<T> a;
  a.dst = (T *)dst.data;
  a.src = (const T *)src.data;
  a.slot = s.data;
  a.weight = (const typename Weight<T>::type *)weight;
  a.vecs = vec ? dst.cols / VB : dst.cols;
  const int batch = s.chosen <= 1 ? 1 : s.chosen <= 2 ? 2 : s.chosen <= 4 ? 4 : 8;
  a.team = vec && a.vecs <= 8 ? 8 : vec && a.vecs <= 16 ? 16 : 32;
  const int64_t lane_vecs = vec ? kRingSlots / batch : kLaneItems<T>;     // G of the combine kernels
  const bool by_vector = dispatch && vec;
  a.per = by_vector ? (uint64_t)a.vecs : (uint64_t)((a.vecs + a.team * lane_vecs - 1) / (a.team * lane_vecs));
  a.items = a.per * (uint64_t)s.tokens;
  const uint64_t per_cta = by_vector ? kRowThreads : kRowThreads / a.team, blocks = (a.items + per_cta - 1) / per_cta;
  if (blocks >= (1ull << 31) || a.vecs >= (1ll << 31) - 1024 || src.rows >= (1ll << 31)) { set_error("expert rows: tensor too large"); return THCB200_ERR_LIMIT; }
  a.per32 = FastDiv32((uint32_t)a.per);
  a.chosen = (int)s.chosen;
  a.places = dispatch ? dst.rows : src.rows;
  a.dst_stride = dst.row_stride;
  a.src_stride = src.row_stride;
  a.src_col = vec ? 1 : src.col_stride;
  a.errors = index_errors(ctx);
  if (dispatch) {
    if (vec) launch_pdl(dispatch_kernel<T, VB>, (unsigned)blocks, kRowThreads, 0, st, a);
    else launch_pdl(dispatch_single_kernel<T>, (unsigned)blocks, kRowThreads, 0, st, a);
  } else {
    if (vec) {
      const unsigned grid = (unsigned)(blocks < 3 * kNumSM_B200 ? blocks : 3 * kNumSM_B200);
      auto launch = [&](auto kernel) -> int {
        THCB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kRingBytes));
        launch_pdl(kernel, grid, kRowThreads, kRingBytes, st, a);
        return 0;
      };
      const int rc = batch == 1 ? launch(combine_ring_kernel<T, 1>) : batch == 2 ? launch(combine_ring_kernel<T, 2>)
                   : batch == 4 ? launch(combine_ring_kernel<T, 4>) : launch(combine_ring_kernel<T, 8>);
      if (rc) return rc;
    } else {
      auto launch = [&](auto kernel) { launch_pdl(kernel, (unsigned)blocks, kRowThreads, 0, st, a); };
      const bool unit = a.src_col == 1;
      if (batch <= 2) launch(unit ? combine_kernel<T, 2, true> : combine_kernel<T, 2, false>);
      else if (batch == 4) launch(unit ? combine_kernel<T, 4, true> : combine_kernel<T, 4, false>);
      else launch(unit ? combine_kernel<T, 8, true> : combine_kernel<T, 8, false>);
    }
  }
  count_launch();
  THCB_CUDA_TRY(cudaGetLastError());
  return 0;
}

template <typename T>
int run_combine_grad(thcb200_ctx *ctx, const MatView *out, void *grad_weight, const MatView &grad, const MatView &rows, const SlotView &s,
                     const void *weight, cudaStream_t st) {
  auto made_of = [&](size_t bytes) { return (!out || mat_vec(*out, sizeof(T), bytes)) && mat_vec(grad, sizeof(T), bytes) && mat_vec(rows, sizeof(T), bytes); };
  const int bytes = made_of(32) && grad.cols * (int64_t)sizeof(T) >= 32 * 32 ? 32 : made_of(16) ? 16 : (int)sizeof(T);
  const bool vec = bytes > (int)sizeof(T);
  CombineGradArgs<T> a;
  a.grad_rows = out ? (T *)out->data : nullptr;
  a.grad_weight = (typename Weight<T>::type *)grad_weight;
  a.grad = (const T *)grad.data;
  a.rows = (const T *)rows.data;
  a.slot = s.data;
  a.weight = (const typename Weight<T>::type *)weight;
  a.pairs = (uint64_t)(s.tokens * s.chosen);
  a.vecs = grad.cols * (int64_t)sizeof(T) / bytes;
  if (a.vecs >= (1ll << 31) - 1024) { set_error("expert rows: tensor too large"); return THCB200_ERR_LIMIT; }
  a.chosen = FastDiv32((uint32_t)s.chosen);
  a.places = rows.rows;
  a.out_stride = out ? out->row_stride : 0;
  a.grad_stride = grad.row_stride;
  a.grad_col = vec ? 1 : grad.col_stride;
  a.rows_stride = rows.row_stride;
  a.rows_col = vec ? 1 : rows.col_stride;
  a.errors = index_errors(ctx);
  a.team_bits = 5;
  while (a.team_bits > 2 && (1 << (a.team_bits - 1)) >= a.vecs) --a.team_bits;
  const uint64_t per_cta = kRowThreads >> a.team_bits;
  const unsigned blocks = (unsigned)((a.pairs + per_cta - 1) / per_cta);
  auto launch = [&](auto kernel) { launch_pdl(kernel, blocks, kRowThreads, 0, st, a); };
#define THCB_GRAD(V, TEAMS, LONG) \
  do { \
    if (out && grad_weight) launch(combine_grad_kernel<T, V, true, true, TEAMS, LONG>); \
    else if (out) launch(combine_grad_kernel<T, V, true, false, TEAMS, LONG>); \
    else launch(combine_grad_kernel<T, V, false, true, TEAMS, LONG>); \
  } while (0)
  if (bytes == 32) THCB_GRAD(32 / sizeof(T), false, false);
  else if (bytes == 16) THCB_GRAD(16 / sizeof(T), true, false);
  else if (sizeof(T) == 8 || a.vecs <= 8 * 32) THCB_GRAD(1, true, false);
  else THCB_GRAD(1, false, sizeof(T) < 8);
#undef THCB_GRAD
  count_launch();
  THCB_CUDA_TRY(cudaGetLastError());
  return 0;
}

int route(thcb200_ctx *ctx, bool dispatch, const thcb200_tensor *dst_t, const thcb200_tensor *src_t, const thcb200_tensor *slot,
          const thcb200_tensor *weight, void *stream) {
  const char *name = dispatch ? "expert_dispatch" : "expert_combine";
  if (!ctx) { set_error("%s: null context", name); return THCB200_ERR_ARG; }
  MatView dst, src;
  SlotView s;
  void *w = nullptr;
  int rc = to_mat_view(dst_t, &dst, name);
  if (!rc) rc = to_mat_view(src_t, &src, name);
  if (!rc) rc = slot_view(slot, &s, name);
  if (!rc && (!floating(dst.dtype) || src.dtype != dst.dtype)) { set_error("%s: both matrices must be of one floating-point type", name); rc = THCB200_ERR_ARG; }
  if (!rc) rc = weight_view(weight, dst.dtype, s, &w, name);
  if (rc) return rc;
  if (dst.cols != src.cols || (dispatch ? src.rows : dst.rows) != s.tokens) { set_error("%s: sizes do not match", name); return THCB200_ERR_SIZE; }
  if (!dense_rows(dst)) { set_error("%s: the result must have dense rows that do not overlap", name); return THCB200_ERR_ARG; }
  if (s.tokens == 0 || dst.cols == 0 || (dispatch && s.chosen == 0)) return THCB200_OK;
  cudaStream_t st = (cudaStream_t)stream;
  set_plan_name(name);
  switch (dst.dtype) {
    case THCB200_F16: return run_route<__half>(ctx, dispatch, dst, src, s, w, st);
    case THCB200_F32: return run_route<float>(ctx, dispatch, dst, src, s, w, st);
    default: return run_route<double>(ctx, dispatch, dst, src, s, w, st);
  }
}

}  // namespace
}  // namespace thcb

using namespace thcb;

extern "C" {

int thcb200_expert_sort(thcb200_ctx *ctx, const thcb200_tensor *slot, const thcb200_tensor *order, const thcb200_tensor *offsets,
                        const thcb200_tensor *expert, void *stream) {
  if (!ctx) { set_error("expert_sort: null context"); return THCB200_ERR_ARG; }
  HostView vs, vo, vf, ve;
  int rc = to_host_view(slot, &vs, "expert_sort slots");
  if (!rc) rc = to_host_view(order, &vo, "expert_sort order");
  if (!rc) rc = to_host_view(offsets, &vf, "expert_sort offsets");
  if (!rc) rc = to_host_view(expert, &ve, "expert_sort experts");
  if (rc) return rc;
  for (const HostView *v : {&vs, &vo, &vf, &ve})
    if (v->dtype != THCB200_I64 || !dense(*v)) { set_error("expert_sort: every argument is a contiguous I64 tensor"); return THCB200_ERR_ARG; }
  if (vs.numel != ve.numel || vo.numel != ve.numel || vf.ndim != 1) { set_error("expert_sort: sizes do not match"); return THCB200_ERR_SIZE; }
  const int64_t experts = vf.sizes[0] - 1;
  if (experts < 1 || experts >= kSortMaxBins) { set_error("expert_sort: between 1 and %d experts", kSortMaxBins - 1); return THCB200_ERR_LIMIT; }
  if (ve.numel > kSortMaxItems) { set_error("expert_sort: more than 2^31 choices"); return THCB200_ERR_LIMIT; }
  THCB_CTX_LOCK(ctx);
  SortInput in;
  in.index = (const int64_t *)ve.data;
  in.stride = 1;
  in.n = ve.numel;
  in.limit = experts;
  in.skip = 0;
  in.zero_is_none = 1;
  in.errors = index_errors(ctx);
  cudaStream_t st = (cudaStream_t)stream;
  set_plan_name("expert_sort");
  Workspace ws(ctx, sort_to_slots_bytes(in.n, in.limit), st);
  if (!ws.ok) return THCB200_ERR_NOMEM;
  return sort_to_slots(in, (int64_t *)vs.data, (int64_t *)vo.data, (int64_t *)vf.data, ws.data, st);
}

int thcb200_expert_dispatch(thcb200_ctx *ctx, const thcb200_tensor *rows, const thcb200_tensor *src, const thcb200_tensor *slot,
                            const thcb200_tensor *weight, void *stream) {
  return route(ctx, true, rows, src, slot, weight, stream);
}

int thcb200_expert_combine(thcb200_ctx *ctx, const thcb200_tensor *result, const thcb200_tensor *rows, const thcb200_tensor *slot,
                           const thcb200_tensor *weight, void *stream) {
  return route(ctx, false, result, rows, slot, weight, stream);
}

int thcb200_expert_combine_grad(thcb200_ctx *ctx, const thcb200_tensor *grad_rows, const thcb200_tensor *grad_weight,
                                const thcb200_tensor *grad_result, const thcb200_tensor *rows, const thcb200_tensor *slot,
                                const thcb200_tensor *weight, void *stream) {
  const char *name = "expert_combine_grad";
  if (!ctx) { set_error("%s: null context", name); return THCB200_ERR_ARG; }
  MatView out, grad, r;
  SlotView s;
  void *w = nullptr, *gw = nullptr;
  int rc = grad_rows ? to_mat_view(grad_rows, &out, name) : 0;
  if (!rc) rc = to_mat_view(grad_result, &grad, name);
  if (!rc) rc = to_mat_view(rows, &r, name);
  if (!rc) rc = slot_view(slot, &s, name);
  if (!rc && (!floating(grad.dtype) || r.dtype != grad.dtype || (grad_rows && out.dtype != grad.dtype))) {
    set_error("%s: the matrices must be of one floating-point type", name);
    rc = THCB200_ERR_ARG;
  }
  if (!rc) rc = weight_view(weight, grad.dtype, s, &w, name);
  if (!rc) rc = weight_view(grad_weight, grad.dtype, s, &gw, name);
  if (rc) return rc;
  if (grad.rows != s.tokens || r.cols != grad.cols || (grad_rows && (out.cols != r.cols || out.rows != r.rows))) {
    set_error("%s: sizes do not match", name);
    return THCB200_ERR_SIZE;
  }
  if (grad_rows && !dense_rows(out)) { set_error("%s: the rows' gradient must have dense rows that do not overlap", name); return THCB200_ERR_ARG; }
  if (s.tokens == 0 || s.chosen == 0 || (!grad_rows && !grad_weight)) return THCB200_OK;
  cudaStream_t st = (cudaStream_t)stream;
  set_plan_name(name);
  const MatView *o = grad_rows ? &out : nullptr;
  switch (grad.dtype) {
    case THCB200_F16: return run_combine_grad<__half>(ctx, o, gw, grad, r, s, w, st);
    case THCB200_F32: return run_combine_grad<float>(ctx, o, gw, grad, r, s, w, st);
    default: return run_combine_grad<double>(ctx, o, gw, grad, r, s, w, st);
  }
}

}  // extern "C"
