// One AdamW step over a list of tensors, and the values that 8-bit moments stand for.
//
// With g = grad_scale * gradient, t = step:
//   m = beta1 m + (1 - beta1) g          v = beta2 v + (1 - beta2) g^2
//   p = p (1 - lr weight_decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
// All of it in float (double for double parameters), one rounding when a half parameter is stored; with a master the new
// value is computed from the float master and the parameter is its rounding.
//
// 8-bit moments.  256 neighbouring elements of a tensor share a float unit.  A signed code c of the first moment stands for
// c|c| * unit with unit = max|m| / 127^2, a code c of 0..255 of the second for c^4 * unit with unit = max v / 255^4: codes
// are dense near zero, where most moments of a block lie.  Steps of moments are far smaller than the distance of two codes
// (1 - beta2 = 0.001 against 1.6 % at the top of a block), so rounding to the nearest code would hold an average in place;
// a value between two codes instead takes the upper one with the probability that keeps its expectation, by a dither that
// is a hash of the element's place and the step (multiplicative hashing, Knuth, The Art of Computer Programming 6.4):
// nothing is drawn, the same call gives the same codes.  A second moment that is not zero never takes code 0: a zero
// below the root would blow its element's step up.
//
// Every step here is one IEEE operation (the library is compiled without contraction), so codes do not depend on the
// compiler's choice of fused operations.
#include <cuda_fp16.h>
#include <math.h>

#include <algorithm>
#include <new>
#include <vector>

#include "context.h"
#include "core.cuh"
#include "plan.h"
#include "rows.cuh"

namespace thcb {
namespace {

constexpr int kStepThreads = 256;
constexpr int kStepItems = 8;                                 // elements per thread
constexpr int kStepTile = kStepThreads * kStepItems;          // elements per CTA
constexpr int kUnitItems = THCB200_ADAMW_BLOCK;               // elements that share a unit: a warp's
static_assert(kUnitItems == 32 * kStepItems, "a warp holds one block of codes");

template <typename T> struct State { using type = float; };
template <> struct State<double> { using type = double; };

struct StepEntry {
  void *param;
  const void *grad;
  void *m, *v, *master;
  float *m_unit, *v_unit;
  int64_t n;
  uint32_t first_tile;
  uint32_t wide;        // every array starts on a vector boundary
};
// The list travels in the kernel's arguments: no table to upload, and a captured graph holds it by value.
template <int N> struct StepTable {
  int count;
  StepEntry e[N];
};
constexpr int kFewTensors = 16, kManyTensors = 320;           // 1 KiB / 22.5 KiB of arguments

template <typename A> struct StepScalars { A beta1, one_minus_beta1, beta2, one_minus_beta2, keep, size, root, eps, grad_scale; uint32_t dither; };

// The entry a tile belongs to: the last one whose first tile is not behind it.
template <int N> __device__ __forceinline__ const StepEntry &entry_of(const StepTable<N> &t, uint32_t tile) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.e[mid].first_tile <= tile) lo = mid; else hi = mid - 1;
  }
  return t.e[lo];
}

// Eight elements of a thread: neighbours of a vector, or for tensors off the vector grid and the ragged end one in
// every 32 (32 threads then read neighbouring elements).
template <typename T> struct Eight { T e[kStepItems]; };

template <typename T> __device__ __forceinline__ void load_wide(Eight<T> &x, const T *p) {
  constexpr int bytes = sizeof(T) * kStepItems;
  char *d = reinterpret_cast<char *>(&x);
  if constexpr (bytes == 8) {
    const uint2 b = *reinterpret_cast<const uint2 *>(p);
    memcpy(d, &b, 8);
  } else if constexpr (bytes == 16) {
    const Bytes16 b = ld16_stream(p);
    memcpy(d, &b, 16);
  } else {
#pragma unroll
    for (int k = 0; k < bytes / 32; ++k) {
      const Bytes32 b = ld32_stream(reinterpret_cast<const char *>(p) + 32 * k);
      memcpy(d + 32 * k, &b, 32);
    }
  }
}
template <typename T> __device__ __forceinline__ void store_wide(T *p, const Eight<T> &x) {
  constexpr int bytes = sizeof(T) * kStepItems;
  const char *s = reinterpret_cast<const char *>(&x);
  if constexpr (bytes == 8) {
    uint2 b;
    memcpy(&b, s, 8);
    *reinterpret_cast<uint2 *>(p) = b;
  } else if constexpr (bytes == 16) {
    Bytes16 b;
    memcpy(&b, s, 16);
    st16(p, b);
  } else {
#pragma unroll
    for (int k = 0; k < bytes / 32; ++k) {
      Bytes32 b;
      memcpy(&b, s + 32 * k, 32);
      st32(reinterpret_cast<char *>(p) + 32 * k, b);
    }
  }
}

// Where a thread's elements lie: base + j (wide) or base + 32 j.
struct Place {
  int64_t base, n;
  bool wide;
  __device__ __forceinline__ int64_t at(int j) const { return wide ? base + j : base + 32 * j; }
};
template <typename T> __device__ __forceinline__ void load_eight(Eight<T> &x, const T *p, const Place &q) {
  if (q.wide) {
    load_wide(x, p + q.base);
  } else {
#pragma unroll
    for (int j = 0; j < kStepItems; ++j)
      if (q.at(j) < q.n) x.e[j] = p[q.at(j)]; else x.e[j] = T();
  }
}
template <typename T> __device__ __forceinline__ void store_eight(T *p, const Eight<T> &x, const Place &q) {
  if (q.wide) {
    store_wide(p + q.base, x);
  } else {
#pragma unroll
    for (int j = 0; j < kStepItems; ++j)
      if (q.at(j) < q.n) p[q.at(j)] = x.e[j];
  }
}
__device__ __forceinline__ Place place_of(const StepEntry &e, uint32_t tile) {
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t block = (int64_t)(tile - e.first_tile) * kStepTile + (int64_t)warp * kUnitItems;
  Place q;
  q.n = e.n;
  q.wide = e.wide && block + kUnitItems <= e.n;
  q.base = q.wide ? block + lane * kStepItems : block + lane;
  return q;
}

template <typename A> __device__ __forceinline__ A root_of(A v);
template <> __device__ __forceinline__ float root_of<float>(float v) { return sqrtf(v); }
template <> __device__ __forceinline__ double root_of<double>(double v) { return sqrt(v); }

template <typename T, bool MASTER>
__device__ __forceinline__ void load_param(Eight<typename State<T>::type> &p, const StepEntry &e, const Place &q) {
  using A = typename State<T>::type;
  if constexpr (MASTER) {
    load_eight(p, (const A *)e.master, q);
  } else {
    Eight<T> x;
    load_eight(x, (const T *)e.param, q);
#pragma unroll
    for (int j = 0; j < kStepItems; ++j) p.e[j] = (A)to_math(x.e[j]);
  }
}
template <typename T, bool MASTER>
__device__ __forceinline__ void store_param(const Eight<typename State<T>::type> &p, const StepEntry &e, const Place &q) {
  using A = typename State<T>::type;
  if constexpr (MASTER) store_eight((A *)e.master, p, q);
  Eight<T> x;
#pragma unroll
  for (int j = 0; j < kStepItems; ++j) x.e[j] = from_math<T>(p.e[j]);
  store_eight((T *)e.param, x, q);
}

template <typename A>
__device__ __forceinline__ void advance(A &p, A &m, A &v, A g, const StepScalars<A> &s) {
  g = g * s.grad_scale;
  m = m * s.beta1 + g * s.one_minus_beta1;
  v = v * s.beta2 + g * s.one_minus_beta2 * g;
  p = p * s.keep - s.size * (m / (root_of(v) * s.root + s.eps));
}

template <typename T, bool MASTER, int N>
__global__ void __launch_bounds__(kStepThreads)
adamw_kernel(const __grid_constant__ StepTable<N> table, const StepScalars<typename State<T>::type> s) {
  using A = typename State<T>::type;
  pdl_prologue();
  const StepEntry &e = entry_of(table, blockIdx.x);
  const Place q = place_of(e, blockIdx.x);
  if (q.base >= q.n) return;
  Eight<A> p, m, v;
  Eight<T> g;
  load_param<T, MASTER>(p, e, q);
  load_eight(g, (const T *)e.grad, q);
  load_eight(m, (const A *)e.m, q);
  load_eight(v, (const A *)e.v, q);
#pragma unroll
  for (int j = 0; j < kStepItems; ++j) advance<A>(p.e[j], m.e[j], v.e[j], (A)to_math(g.e[j]), s);
  store_param<T, MASTER>(p, e, q);
  store_eight((A *)e.m, m, q);
  store_eight((A *)e.v, v, q);
}

// ---- 8-bit codes ---------------------------------------------------------------------------------
__device__ __forceinline__ float first_value(int c) { return (float)(c * abs(c)); }
__device__ __forceinline__ float second_value(int c) { const float f = (float)(c * c); return f * f; }
__device__ __forceinline__ uint32_t dither_of(uint32_t place, uint32_t step) {
  uint32_t h = place * 0x9E3779B9u + step;
  h = (h ^ h >> 16) * 0x9E3779B9u;
  h = (h ^ h >> 15) * 0x9E3779B9u;
  return h ^ h >> 16;
}
// The last code of 0..TOP whose value is at most x, or by the dither the next.
template <int TOP, float VALUE(int)>
__device__ __forceinline__ int code_of(float x, float guess, float dither) {
  int k = min(max((int)guess, 0), TOP);
  if (VALUE(k) > x) --k;
  else if (k < TOP && VALUE(k + 1) <= x) ++k;
  if (k < TOP && dither * (VALUE(k + 1) - VALUE(k)) < x - VALUE(k)) ++k;
  return k;
}
// Largest of non-negative floats over a warp; a NaN, whose bits are above infinity's, wins.
__device__ __forceinline__ float warp_most(float x) { return __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(x) & 0x7fffffffu)); }

constexpr float kFirstTop = (float)(1.0 / 16129.0), kSecondTop = (float)(1.0 / (255.0 * 255.0 * 255.0 * 255.0));
// Blocks whose largest value is below these (where a unit would leave the normal floats) are stored as zero.
constexpr float kFirstLeast = 1e-30f, kSecondLeast = 1e-28f;

template <typename T, bool MASTER, int N>
__global__ void __launch_bounds__(kStepThreads)
adamw8_kernel(const __grid_constant__ StepTable<N> table, const StepScalars<float> s) {
  pdl_prologue();
  const StepEntry &e = entry_of(table, blockIdx.x);
  const Place q = place_of(e, blockIdx.x);
  const int64_t block = (int64_t)(blockIdx.x - e.first_tile) * (kStepThreads / 32) + (threadIdx.x >> 5);
  if (block * kUnitItems >= e.n) return;      // whole warps
  Eight<float> p, m, v;
  Eight<T> g;
  Eight<int8_t> cm;
  Eight<uint8_t> cv;
  load_param<T, MASTER>(p, e, q);
  load_eight(g, (const T *)e.grad, q);
  load_eight(cm, (const int8_t *)e.m, q);
  load_eight(cv, (const uint8_t *)e.v, q);
  const float mu = e.m_unit[block], vu = e.v_unit[block];
  float mm = 0, vm = 0;
  bool mnan = false;
#pragma unroll
  for (int j = 0; j < kStepItems; ++j) {
    m.e[j] = first_value(cm.e[j]) * mu;
    v.e[j] = second_value(cv.e[j]) * vu;
    advance<float>(p.e[j], m.e[j], v.e[j], to_math(g.e[j]), s);
    if (!q.wide && q.at(j) >= q.n) m.e[j] = v.e[j] = 0;
    mnan = mnan || !(m.e[j] == m.e[j]) || !(v.e[j] == v.e[j]);
    mm = fmaxf(mm, fabsf(m.e[j]));
    vm = fmaxf(vm, v.e[j]);
  }
  store_param<T, MASTER>(p, e, q);
  if (mnan) mm = vm = __int_as_float(0x7fffffff);
  mm = warp_most(mm);
  vm = warp_most(vm);
  // not (x < least): a NaN stays
  const float nmu = mm < kFirstLeast ? 0.0f : mm * kFirstTop, nvu = vm < kSecondLeast ? 0.0f : vm * kSecondTop;
  const float mi = nmu > 0 ? 1.0f / nmu : 0.0f, vi = nvu > 0 ? 1.0f / nvu : 0.0f;
#pragma unroll
  for (int j = 0; j < kStepItems; ++j) {
    const uint32_t h = dither_of((uint32_t)q.at(j), s.dither);
    const float xm = fabsf(m.e[j]) * mi, xv = v.e[j] * vi;
    const int km = code_of<127, first_value>(xm, sqrtf(xm), (float)(h >> 16) * (1.0f / 65536.0f));
    int kv = code_of<255, second_value>(xv, sqrtf(sqrtf(xv)), (float)(h & 0xffffu) * (1.0f / 65536.0f));
    if (v.e[j] > 0 && kv == 0) kv = 1;
    cm.e[j] = (int8_t)(m.e[j] < 0 ? -km : km);
    cv.e[j] = (uint8_t)kv;
  }
  store_eight((int8_t *)e.m, cm, q);
  store_eight((uint8_t *)e.v, cv, q);
  if ((threadIdx.x & 31) == 0) {
    e.m_unit[block] = nmu;
    e.v_unit[block] = nvu;
  }
}

// What the codes stand for: param and master of the entry are the float results for the first and second moment.
template <int N>
__global__ void __launch_bounds__(kStepThreads)
adamw_values_kernel(const __grid_constant__ StepTable<N> table) {
  pdl_prologue();
  const StepEntry &e = entry_of(table, blockIdx.x);
  const Place q = place_of(e, blockIdx.x);
  const int64_t block = (int64_t)(blockIdx.x - e.first_tile) * (kStepThreads / 32) + (threadIdx.x >> 5);
  if (block * kUnitItems >= e.n) return;
  Eight<int8_t> cm;
  Eight<uint8_t> cv;
  Eight<float> m, v;
  load_eight(cm, (const int8_t *)e.m, q);
  load_eight(cv, (const uint8_t *)e.v, q);
  const float mu = e.m_unit[block], vu = e.v_unit[block];
#pragma unroll
  for (int j = 0; j < kStepItems; ++j) {
    m.e[j] = first_value(cm.e[j]) * mu;
    v.e[j] = second_value(cv.e[j]) * vu;
  }
  store_eight((float *)e.param, m, q);
  store_eight((float *)e.master, v, q);
}

// ---- host --------------------------------------------------------------------------------------
bool on_grid(const void *p, size_t esz) {
  const size_t bytes = esz * kStepItems > 32 ? 32 : esz * kStepItems;
  return (uintptr_t)p % bytes == 0;
}

// Two arrays that share memory, one of them written, would make the step depend on the order of threads.  Lists of
// pieces of one buffer come in address order; anything else is sorted.
struct Range { uintptr_t lo, hi; };
bool overlap(std::vector<Range> &r) {
  if (!std::is_sorted(r.begin(), r.end(), [](const Range &a, const Range &b) { return a.lo < b.lo; }))
    std::sort(r.begin(), r.end(), [](const Range &a, const Range &b) { return a.lo < b.lo; });
  for (size_t i = 1; i < r.size(); ++i)
    if (r[i].lo < r[i - 1].hi) return true;
  return false;
}

enum StepKind { kStep32, kStep8, kStepValues };

template <int N, typename L>
int launch_table(const thcb200_adamw_tensor *t, int count, size_t esz, StepKind kind, L launch) {
  // entries are taken in turn until the table is full or the tiles run out of grid
  StepTable<N> table;
  int i = 0;
  while (i < count) {
    table.count = 0;
    uint64_t tiles = 0;
    for (; i < count && table.count < N; ++i) {
      if (t[i].numel == 0) continue;
      const uint64_t need = ((uint64_t)t[i].numel + kStepTile - 1) / kStepTile;
      if (need >= (1ull << 31)) { set_error("adamw: tensor %d is too large", i); return THCB200_ERR_LIMIT; }
      if (tiles + need >= (1ull << 31)) break;
      StepEntry &e = table.e[table.count++];
      e.param = t[i].param;
      e.grad = t[i].grad;
      e.m = t[i].m;
      e.v = t[i].v;
      e.master = t[i].master;
      e.m_unit = t[i].m_unit;
      e.v_unit = t[i].v_unit;
      e.n = t[i].numel;
      e.first_tile = (uint32_t)tiles;
      const size_t msz = kind == kStep32 ? (esz == 8 ? 8 : 4) : 1, psz = kind == kStepValues ? 4 : esz, wsz = esz == 8 ? 8 : 4;
      e.wide = on_grid(e.param, psz) && (!e.grad || on_grid(e.grad, psz)) && on_grid(e.m, msz) && on_grid(e.v, msz) &&
               (!e.master || on_grid(e.master, wsz));
      tiles += need;
    }
    if (table.count == 0) break;
    launch(table, (unsigned)tiles);
    count_launch();
    THCB_CUDA_TRY(cudaGetLastError());
  }
  return 0;
}

template <typename T, bool MASTER, int N>
int run_step(const thcb200_adamw_tensor *t, int count, int bits, const thcb200_adamw_args &a, cudaStream_t st) {
  using A = typename State<T>::type;
  StepScalars<A> s;
  s.beta1 = (A)a.beta1;
  s.one_minus_beta1 = (A)(1 - a.beta1);
  s.beta2 = (A)a.beta2;
  s.one_minus_beta2 = (A)(1 - a.beta2);
  s.keep = (A)(1 - a.lr * a.weight_decay);
  s.size = (A)(a.lr / (1 - pow(a.beta1, (double)a.step)));
  s.root = (A)(1 / sqrt(1 - pow(a.beta2, (double)a.step)));
  s.eps = (A)a.eps;
  s.grad_scale = (A)a.grad_scale;
  s.dither = (uint32_t)((uint64_t)a.step * 0x7F4A7C15ull);
  if (bits == 32)
    return launch_table<N>(t, count, sizeof(T), kStep32, [&](const StepTable<N> &table, unsigned tiles) {
      launch_pdl(adamw_kernel<T, MASTER, N>, tiles, kStepThreads, 0, st, table, s);
    });
  if constexpr (sizeof(T) < 8)
    return launch_table<N>(t, count, sizeof(T), kStep8, [&](const StepTable<N> &table, unsigned tiles) {
      launch_pdl(adamw8_kernel<T, MASTER, N>, tiles, kStepThreads, 0, st, table, s);
    });
  return THCB200_ERR_UNSUPPORTED;
}

template <typename T>
int run_step_typed(const thcb200_adamw_tensor *t, int count, int bits, bool master, const thcb200_adamw_args &a, cudaStream_t st) {
  const bool few = count <= kFewTensors;
  if constexpr (sizeof(T) == 2) {
    if (master) return few ? run_step<T, true, kFewTensors>(t, count, bits, a, st) : run_step<T, true, kManyTensors>(t, count, bits, a, st);
  }
  return few ? run_step<T, false, kFewTensors>(t, count, bits, a, st) : run_step<T, false, kManyTensors>(t, count, bits, a, st);
}

int check_list(const thcb200_adamw_tensor *t, int n, size_t esz, StepKind kind, bool master, const char *name) {
  const size_t wsz = esz == 8 ? 8 : 4, msz = kind == kStep32 ? wsz : 1;
  std::vector<Range> ranges;
  ranges.reserve((size_t)n * (master ? 6 : 5) + 1);
  auto add = [&](const void *p, size_t bytes) { ranges.push_back(Range{(uintptr_t)p, (uintptr_t)p + bytes}); };
  for (int pass = 0; pass < 6; ++pass) {
    for (int i = 0; i < n; ++i) {
      const size_t k = (size_t)t[i].numel, blocks = (k + kUnitItems - 1) / kUnitItems;
      if (k == 0) continue;
      switch (pass) {
        case 0: add(t[i].param, k * (kind == kStepValues ? 4 : esz)); break;
        case 1: add(t[i].m, k * msz); break;
        case 2: add(t[i].v, k * msz); break;
        case 3: if (master || kind == kStepValues) add(t[i].master, k * (kind == kStepValues ? 4 : wsz)); break;
        case 4: if (kind != kStep32) add(t[i].m_unit, blocks * 4); break;
        default: if (kind != kStep32) add(t[i].v_unit, blocks * 4); break;
      }
    }
  }
  if (overlap(ranges)) { set_error("%s: two of the tensors share memory (a tensor may be listed once)", name); return THCB200_ERR_ARG; }
  return 0;
}

}  // namespace
}  // namespace thcb

using namespace thcb;

extern "C" {

int thcb200_adamw(thcb200_ctx *ctx, int dtype, int bits, const thcb200_adamw_tensor *tensors, int n, const thcb200_adamw_args *args, void *stream) {
  if (!ctx || !args || n < 0 || (n > 0 && !tensors)) { set_error("adamw: null argument"); return THCB200_ERR_ARG; }
  if (!floating(dtype)) { set_error("adamw: parameters are of a floating-point type"); return THCB200_ERR_ARG; }
  if (bits != 32 && bits != 8) { set_error("adamw: moments have 32 or 8 bits"); return THCB200_ERR_ARG; }
  if (bits == 8 && dtype == THCB200_F64) { set_error("adamw: 8-bit moments go with half and float parameters"); return THCB200_ERR_UNSUPPORTED; }
  const thcb200_adamw_args &a = *args;
  if (!(a.beta1 >= 0 && a.beta1 < 1 && a.beta2 >= 0 && a.beta2 < 1)) { set_error("adamw: beta1 and beta2 lie in [0, 1)"); return THCB200_ERR_ARG; }
  if (!(a.eps >= 0) || !(a.lr >= 0)) { set_error("adamw: lr and eps are not negative"); return THCB200_ERR_ARG; }
  if (a.step < 1) { set_error("adamw: steps count from 1"); return THCB200_ERR_ARG; }
  bool master = false;
  for (int i = 0; i < n; ++i) {
    const thcb200_adamw_tensor &t = tensors[i];
    if (t.numel < 0) { set_error("adamw: tensor %d has a negative size", i); return THCB200_ERR_SIZE; }
    if (t.master) master = true;
    if (t.numel == 0) continue;
    if (!t.param || !t.grad || !t.m || !t.v || (bits == 8 && (!t.m_unit || !t.v_unit))) { set_error("adamw: tensor %d: null pointer", i); return THCB200_ERR_ARG; }
  }
  if (master && dtype != THCB200_F16) { set_error("adamw: masters go with half parameters"); return THCB200_ERR_ARG; }
  if (master)
    for (int i = 0; i < n; ++i)
      if (!tensors[i].master && tensors[i].numel > 0) { set_error("adamw: tensor %d has no master, others have", i); return THCB200_ERR_ARG; }
  try {
    const int rc = check_list(tensors, n, dtype_size(dtype), bits == 8 ? kStep8 : kStep32, master, "adamw");
    if (rc) return rc;
  } catch (const std::bad_alloc &) {
    set_error("adamw: out of host memory");
    return THCB200_ERR_NOMEM;
  }
  cudaStream_t st = (cudaStream_t)stream;
  set_plan_name(bits == 8 ? "adamw8" : "adamw32");
  switch (dtype) {
    case THCB200_F16: return run_step_typed<__half>(tensors, n, bits, master, a, st);
    case THCB200_F32: return run_step_typed<float>(tensors, n, bits, master, a, st);
    default: return run_step_typed<double>(tensors, n, bits, master, a, st);
  }
}

int thcb200_adamw_values(thcb200_ctx *ctx, const thcb200_adamw_tensor *tensors, int n, void *stream) {
  if (!ctx || n < 0 || (n > 0 && !tensors)) { set_error("adamw_values: null argument"); return THCB200_ERR_ARG; }
  for (int i = 0; i < n; ++i) {
    const thcb200_adamw_tensor &t = tensors[i];
    if (t.numel < 0) { set_error("adamw_values: tensor %d has a negative size", i); return THCB200_ERR_SIZE; }
    if (t.numel > 0 && (!t.param || !t.master || !t.m || !t.v || !t.m_unit || !t.v_unit)) {
      set_error("adamw_values: tensor %d: null pointer", i);
      return THCB200_ERR_ARG;
    }
  }
  try {
    const int rc = check_list(tensors, n, 4, kStepValues, true, "adamw_values");
    if (rc) return rc;
  } catch (const std::bad_alloc &) {
    set_error("adamw_values: out of host memory");
    return THCB200_ERR_NOMEM;
  }
  cudaStream_t st = (cudaStream_t)stream;
  set_plan_name("adamw_values");
  if (n <= kFewTensors)
    return launch_table<kFewTensors>(tensors, n, 4, kStepValues, [&](const StepTable<kFewTensors> &table, unsigned tiles) {
      launch_pdl(adamw_values_kernel<kFewTensors>, tiles, kStepThreads, 0, st, table);
    });
  return launch_table<kManyTensors>(tensors, n, 4, kStepValues, [&](const StepTable<kManyTensors> &table, unsigned tiles) {
    launch_pdl(adamw_values_kernel<kManyTensors>, tiles, kStepThreads, 0, st, table);
  });
}

}  // extern "C"
