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
// Moments and codes take one IEEE operation after the other (the library is compiled without contraction), so they do not
// depend on the compiler's choice of fused operations; the 8-bit form's parameter takes the approximate root and reciprocal.
//
// Both are bound by HBM in principle.  200 M float elements in 290 tensors, B200: 32-bit moments 800 us, 5.6 GB, 7000 GB/s (the
// box's copy: 6558).  8-bit moments, 3.2 GB: 795 us, 4.0 TB/s, bound by instruction issue (about 90 per element): 1310 us with
// scalar instructions, IEEE roots and byte conversions, 925 us packed, 890 us with 1024 threads per SM, 860 us with the next tile
// prefetched into the L2, 840 us with the rare exact codes apart, 795 us with CTAs of 128 threads (a loop of 1500; 695 us before the
// power limit holds the clocks back).  Half parameters issue as many: 806 us for 2.0 GB, with masters 850 us for 3.2 GB.
#include <cuda_fp16.h>
#include <float.h>
#include <math.h>

#include <algorithm>
#include <new>
#include <type_traits>
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
constexpr int kCodeThreads = 128, kCodeTile = kCodeThreads * kStepItems;   // the 8-bit step's: smaller CTAs fall into step less (69 -> 67 us, 20 M elements)
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
constexpr int kFewTensors = 16, kSomeTensors = 80, kManyTensors = 320;   // 1, 6 and 22.5 KiB of arguments: a launch with the last takes 2 us longer

template <typename A> struct StepScalars { A beta1, one_minus_beta1, beta2, one_minus_beta2, keep, size, root, eps, grad_scale; uint32_t dither; };
constexpr size_t kArgumentBytes = 32764;                                 // of a kernel launch

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
template <int TILE> __device__ __forceinline__ Place place_of(const StepEntry &e, uint32_t tile) {
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t block = (int64_t)(tile - e.first_tile) * TILE + (int64_t)warp * kUnitItems;
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
  const Place q = place_of<kStepTile>(e, blockIdx.x);
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
// Codes are handled as floats: c * |c| and (c c)(c c) are the products the definition names, and bytes become floats and
// back by their place in the significand of 2^23 + c (an exact addition) instead of conversion instructions.  Neighbouring
// elements share the packed float instructions (two IEEE operations each).
using F2 = unsigned long long;
__device__ __forceinline__ F2 pair(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__host__ __device__ __forceinline__ F2 both(float a) {
#ifdef __CUDA_ARCH__
  return pair(a, a);
#else
  uint32_t b;
  memcpy(&b, &a, 4);
  return (F2)b << 32 | b;
#endif
}
__device__ __forceinline__ float lo_of(F2 x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float hi_of(F2 x) { return __uint_as_float((uint32_t)(x >> 32)); }
__device__ __forceinline__ F2 add2(F2 a, F2 b) { F2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
// The two products, as a * b + z with z = -0 from the kernel's arguments: the assembler contracts a packed product and the
// packed sum behind it into one operation (a last bit of a moment differed), whatever it is told; a value it does not know to be
// zero stops it.
__device__ __forceinline__ F2 mul2(F2 a, F2 b, F2 z) { F2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(z)); return r; }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) { F2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
// The step's scalars, as pairs.
struct StepPairs {
  F2 grad_scale, beta1, one_minus_beta1, beta2, one_minus_beta2, keep, minus_size, root, eps;
  F2 minus_zero;
  uint32_t dither;
};
static_assert(sizeof(StepTable<kManyTensors>) + std::max(sizeof(StepPairs), sizeof(StepScalars<double>)) + alignof(StepPairs) <= kArgumentBytes);
__device__ __forceinline__ F2 sub2(F2 a, F2 b) { return fma2(b, both(-1.0f), a); }   // no instruction for the sign
__device__ __forceinline__ F2 fma2_down(F2 a, F2 b, F2 c) { F2 r; asm("fma.rm.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }

// Byte k of a word as 2^23 + byte.
__device__ __forceinline__ float byte_magic(uint32_t word, int k) { return __uint_as_float(__byte_perm(word, 0x4b000000u, 0x7440 | k)); }
// Half k of a word as 2^7 + half / 65536.
__device__ __forceinline__ float half_magic(uint32_t word, int k) { return __uint_as_float(__byte_perm(word, 0x43000000u, k ? 0x7432 : 0x7410)); }
constexpr float kMagic = 8388608.0f, kByteMagic = 12582912.0f;      // 1.5 * 2^23: -128..255 end up in the low byte
__device__ __forceinline__ float first_value(float c) { return c * fabsf(c); }
__device__ __forceinline__ float second_value(float c) { const float f = c * c; return f * f; }
constexpr uint32_t kDitherPlace = 0x9E3779B9u;         // 2^32 over the golden ratio; the step's hash is added to place * this
__device__ __forceinline__ uint32_t dither_of(uint32_t h) {
  h = (h ^ h >> 16) * kDitherPlace;
  h = (h ^ h >> 15) * kDitherPlace;
  return h ^ h >> 16;
}
__device__ __forceinline__ float root_near(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float inverse_near(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float max_or_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max_of(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float one_if_below(float a, float b) {
  float r;
  asm("set.lt.f32.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The last code of 0..TOP whose value is at most x, or by the dither (0..65535 of 65536) the next.
template <int TOP, bool FOURTH>
__device__ __forceinline__ float code_exact(float x, float root, float dither) {
  auto value = [](float k) { return FOURTH ? second_value(k) : k * k; };
  float k = fminf(floorf(root), (float)TOP);
  if (value(k) > x) k -= 1.0f;
  if (k < (float)TOP && value(k + 1.0f) <= x) k += 1.0f;
  if (k < (float)TOP && dither * 0x1p-16f * (value(k + 1.0f) - value(k)) < x - value(k)) k += 1.0f;
  return k;
}
// The same for two elements without the corrections.  `root` is within 2^-21 of the code as a real number, so the integer
// part k of root (1 - 2^-20) is the code or, next to a border, the one before (and below the top code even for the block's
// largest).  If x has reached k + 1, the dither picks k + 1, which is right unless the dither is so small that k + 2
// is due: the distance x - value(k + 1) is below 2^-10 of a step there.  `rare` becomes positive for a superset of those.
template <bool FOURTH>
__device__ __forceinline__ F2 codes_near(F2 x, F2 root, F2 dither, float &rare, const StepPairs &c) {
  const F2 k = add2(fma2_down(root, both(1.0f - 0x1p-20f), both(kMagic)), both(-kMagic)), next = add2(k, both(1.0f));
  F2 low = mul2(k, k, c.minus_zero), high = mul2(next, next, c.minus_zero);
  if constexpr (FOURTH) { low = mul2(low, low, c.minus_zero); high = mul2(high, high, c.minus_zero); }
  const F2 step = sub2(high, low), above = sub2(x, low), bar = mul2(dither, step, c.minus_zero);
  const F2 over = fma2(step, both(-(1.0f - 0x1p-9f)), sub2(above, bar));
  rare = max_of(rare, lo_of(over), hi_of(over));
  return add2(k, pair(one_if_below(lo_of(bar), lo_of(above)), one_if_below(hi_of(bar), hi_of(above))));
}

constexpr float kFirstTop = (float)(1.0 / 16129.0), kSecondTop = (float)(1.0 / (255.0 * 255.0 * 255.0 * 255.0));
// Blocks whose largest value is below these (where a unit would leave the normal floats) are stored as zero.
constexpr float kFirstLeast = 1e-30f, kSecondLeast = 1e-28f;
// A block whose largest value is not finite has no unit: NaN, and with it the whole block (an infinite one would leave its element
// an infinity of either sign, as the codes of NaN fall, beside NaN for the code 0).
__device__ __forceinline__ float unit_of(float most, float least, float top) { return most < least ? 0.0f : most <= FLT_MAX ? most * top : NAN; }

// The thread's eight codes, as two words.
template <typename T>
__device__ __forceinline__ void load_codes(uint32_t (&w)[2], const T *p, const Place &q) {
  Eight<T> x;
  load_eight(x, p, q);
  memcpy(w, &x, 8);
}
template <typename T>
__device__ __forceinline__ void store_codes(T *p, const uint32_t (&w)[2], const Place &q) {
  Eight<T> x;
  memcpy(&x, w, 8);
  store_eight(p, x, q);
}

// m and v of elements j and j + 1 from their codes.
__device__ __forceinline__ F2 first_pair(const uint32_t (&c)[2], int j, F2 unit, const StepPairs &p) {
  const F2 k = add2(pair(byte_magic(c[j / 4], j % 4), byte_magic(c[j / 4], j % 4 + 1)), both(-(kMagic + 128.0f)));
  return mul2(pair(first_value(lo_of(k)), first_value(hi_of(k))), unit, p.minus_zero);
}
__device__ __forceinline__ F2 second_pair(const uint32_t (&c)[2], int j, F2 unit, const StepPairs &p) {
  const F2 k = add2(pair(byte_magic(c[j / 4], j % 4), byte_magic(c[j / 4], j % 4 + 1)), both(-kMagic)), f = mul2(k, k, p.minus_zero);
  return mul2(mul2(f, f, p.minus_zero), unit, p.minus_zero);
}

// Asks for the tile that this CTA's successor on the SM will work on: the loads of a short-lived CTA with many instructions
// between them otherwise leave the memory idle while its warps compute.
constexpr uint32_t kTilesAhead = 8 * kNumSM_B200;
template <int TILE> __device__ __forceinline__ void prefetch_ahead(const void *base, uint32_t esz, const StepEntry &e, uint32_t tile) {
  const int64_t at = (int64_t)(tile - e.first_tile + kTilesAhead) * TILE;
  const char *p = (const char *)base + at * esz;
  if (at + TILE <= e.n && ((uintptr_t)p & 15) == 0)
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" :: "l"(p), "r"(TILE * esz) : "memory");
}

__device__ __forceinline__ float pick(const F2 (&x)[kStepItems / 2], int j) {      // element j, without an indexed register
  float r = 0;
#pragma unroll
  for (int i = 0; i < kStepItems; ++i) r = i == j ? (i & 1 ? hi_of(x[i / 2]) : lo_of(x[i / 2])) : r;
  return r;
}

template <typename T, bool MASTER, int N>
__global__ void __launch_bounds__(kCodeThreads, 8)
adamw8_kernel(const __grid_constant__ StepTable<N> table, const __grid_constant__ StepPairs c) {
  pdl_prologue();
  const StepEntry &e = entry_of(table, blockIdx.x);
  const Place q = place_of<kCodeTile>(e, blockIdx.x);
  const int64_t block = (int64_t)(blockIdx.x - e.first_tile) * (kCodeThreads / 32) + (threadIdx.x >> 5);
  if (block * kUnitItems >= e.n) return;      // whole warps
  Eight<float> p;
  Eight<T> g;
  uint32_t cm[2], cv[2];
  load_param<T, MASTER>(p, e, q);
  load_eight(g, (const T *)e.grad, q);
  load_codes(cm, (const int8_t *)e.m, q);
  load_codes(cv, (const uint8_t *)e.v, q);
  if (threadIdx.x < 4) {
    const void *base = threadIdx.x == 0 ? (MASTER ? e.master : e.param) : threadIdx.x == 1 ? e.grad : threadIdx.x == 2 ? e.m : e.v;
    prefetch_ahead<kCodeTile>(base, threadIdx.x == 0 ? (MASTER ? 4u : (uint32_t)sizeof(T)) : threadIdx.x == 1 ? (uint32_t)sizeof(T) : 1u, e, blockIdx.x);
  }
  const F2 mu = both(e.m_unit[block]), vu = both(e.v_unit[block]);
  cm[0] ^= 0x80808080u;                       // signed codes as 128 + c
  cm[1] ^= 0x80808080u;
  F2 m[kStepItems / 2], v[kStepItems / 2];
#pragma unroll
  for (int i = 0; i < kStepItems / 2; ++i) {
    const F2 gi = mul2(pair(to_math(g.e[2 * i]), to_math(g.e[2 * i + 1])), c.grad_scale, c.minus_zero);
    m[i] = add2(mul2(first_pair(cm, 2 * i, mu, c), c.beta1, c.minus_zero), mul2(gi, c.one_minus_beta1, c.minus_zero));
    v[i] = add2(mul2(second_pair(cv, 2 * i, vu, c), c.beta2, c.minus_zero), mul2(mul2(gi, c.one_minus_beta2, c.minus_zero), gi, c.minus_zero));
    // the approximate root flushes what is below the normal floats: 2^-126 is nothing beside any other v
    const F2 vr = add2(v[i], both(0x1p-126f));
    const F2 den = fma2(pair(root_near(lo_of(vr)), root_near(hi_of(vr))), c.root, c.eps);
    const F2 ratio = mul2(m[i], pair(inverse_near(lo_of(den)), inverse_near(hi_of(den))), c.minus_zero);
    const F2 pi = fma2(c.minus_size, ratio, mul2(pair(p.e[2 * i], p.e[2 * i + 1]), c.keep, c.minus_zero));
    p.e[2 * i] = lo_of(pi);
    p.e[2 * i + 1] = hi_of(pi);
  }
  store_param<T, MASTER>(p, e, q);
  if (!q.wide) {
#pragma unroll
    for (int i = 0; i < kStepItems / 2; ++i) {
      if (q.at(2 * i) >= q.n) m[i] = v[i] = 0;
      else if (q.at(2 * i + 1) >= q.n) { m[i] = pair(lo_of(m[i]), 0.0f); v[i] = pair(lo_of(v[i]), 0.0f); }
    }
  }
  float mmost = 0, vmost = 0;
#pragma unroll
  for (int i = 0; i < kStepItems / 2; ++i) {
    mmost = max_or_nan(mmost, fabsf(lo_of(m[i])), fabsf(hi_of(m[i])));
    vmost = max_or_nan(vmost, lo_of(v[i]), hi_of(v[i]));
  }
  // over the warp by the bits: a NaN's are above infinity's and win
  mmost = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(mmost)));
  vmost = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(vmost)));
  const float nmu = unit_of(mmost, kFirstLeast, kFirstTop), nvu = unit_of(vmost, kSecondLeast, kSecondTop);
  const float mi = nmu > 0 ? 1.0f / nmu : 0.0f, vi = nvu > 0 ? 1.0f / nvu : 0.0f;
  const uint32_t h = (uint32_t)q.at(0) * kDitherPlace + c.dither, hstep = q.wide ? kDitherPlace : 32u * kDitherPlace;
  F2 km[kStepItems / 2], kv[kStepItems / 2];
  float rare = 0;
#pragma unroll
  for (int i = 0; i < kStepItems / 2; ++i) {
    const uint32_t d0 = dither_of(h + 2 * i * hstep), d1 = dither_of(h + (2 * i + 1) * hstep);
    const F2 xm = pair(fabsf(lo_of(m[i])) * mi, fabsf(hi_of(m[i])) * mi), xv = mul2(v[i], both(vi), c.minus_zero);
    km[i] = codes_near<false>(xm, pair(root_near(lo_of(xm)), root_near(hi_of(xm))),
                              add2(pair(half_magic(d0, 1), half_magic(d1, 1)), both(-128.0f)), rare, c);
    kv[i] = codes_near<true>(xv, pair(root_near(root_near(lo_of(xv))), root_near(root_near(hi_of(xv)))),
                             add2(pair(half_magic(d0, 0), half_magic(d1, 0)), both(-128.0f)), rare, c);
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    uint32_t bm[4], bv[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int j = 2 * w + i;
      const F2 sm = add2(pair(copysignf(lo_of(km[j]), lo_of(m[j])), copysignf(hi_of(km[j]), hi_of(m[j]))), both(kByteMagic));
      // at least 1 where v is above zero: v 2^200, cut at 1, is 0 or 1
      const F2 sv = add2(pair(fmaxf(lo_of(kv[j]), __saturatef(lo_of(v[j]) * 0x1p100f * 0x1p100f)),
                              fmaxf(hi_of(kv[j]), __saturatef(hi_of(v[j]) * 0x1p100f * 0x1p100f))), both(kByteMagic));
      bm[2 * i] = (uint32_t)sm;
      bm[2 * i + 1] = (uint32_t)(sm >> 32);
      bv[2 * i] = (uint32_t)sv;
      bv[2 * i + 1] = (uint32_t)(sv >> 32);
    }
    cm[w] = __byte_perm(__byte_perm(bm[0], bm[1], 0x0040), __byte_perm(bm[2], bm[3], 0x0040), 0x5410);
    cv[w] = __byte_perm(__byte_perm(bv[0], bv[1], 0x0040), __byte_perm(bv[2], bv[3], 0x0040), 0x5410);
  }
  store_codes((int8_t *)e.m, cm, q);
  store_codes((uint8_t *)e.v, cv, q);
  if (rare > 0) {      // apart from the codes above, so that nothing of it costs the others a register
#pragma unroll 1
    for (int j = 0; j < kStepItems; ++j) {
      const float mj = pick(m, j), vj = pick(v, j);
      const uint32_t d = dither_of(h + j * hstep);
      const float xm = fabsf(mj) * mi, xv = vj * vi;
      const float a = code_exact<127, false>(xm, root_near(xm), (float)(d >> 16)), b = code_exact<255, true>(xv, root_near(root_near(xv)), (float)(d & 0xffffu));
      if (q.at(j) >= q.n) break;
      ((int8_t *)e.m)[q.at(j)] = (int8_t)(int)copysignf(a, mj);
      ((uint8_t *)e.v)[q.at(j)] = (uint8_t)(int)(vj > 0 ? fmaxf(b, 1.0f) : b);
    }
  }
  if ((threadIdx.x & 31) == 0) {
    e.m_unit[block] = nmu;
    e.v_unit[block] = nvu;
  }
}

// What the codes stand for: param and master of the entry are the float results for the first and second moment.  200 M elements,
// 2 GB: 307 us, the copy rate; 362 us without the prefetch, 341 and 387 us with two and four blocks a warp.
template <int N>
__global__ void __launch_bounds__(kStepThreads)
adamw_values_kernel(const __grid_constant__ StepTable<N> table, const __grid_constant__ StepPairs c) {
  pdl_prologue();
  const StepEntry &e = entry_of(table, blockIdx.x);
  const Place q = place_of<kStepTile>(e, blockIdx.x);
  const int64_t block = (int64_t)(blockIdx.x - e.first_tile) * (kStepThreads / 32) + (threadIdx.x >> 5);
  if (block * kUnitItems >= e.n) return;
  uint32_t cm[2], cv[2];
  Eight<float> m, v;
  if (threadIdx.x < 2) prefetch_ahead<kStepTile>(threadIdx.x ? e.v : e.m, 1, e, blockIdx.x);
  load_codes(cm, (const int8_t *)e.m, q);
  load_codes(cv, (const uint8_t *)e.v, q);
  const F2 mu = both(e.m_unit[block]), vu = both(e.v_unit[block]);
  cm[0] ^= 0x80808080u;
  cm[1] ^= 0x80808080u;
#pragma unroll
  for (int j = 0; j < kStepItems; j += 2) {
    const F2 a = first_pair(cm, j, mu, c), b = second_pair(cv, j, vu, c);
    m.e[j] = lo_of(a);
    m.e[j + 1] = hi_of(a);
    v.e[j] = lo_of(b);
    v.e[j + 1] = hi_of(b);
  }
  store_eight((float *)e.param, m, q);
  store_eight((float *)e.master, v, q);
}

// ---- host --------------------------------------------------------------------------------------
bool on_grid(const void *p, size_t esz) {          // element sizes are powers of two
  const size_t bytes = esz * kStepItems > 32 ? 32 : esz * kStepItems;
  return ((uintptr_t)p & (bytes - 1)) == 0;
}

// Two arrays that share memory, one of them written, would make the step depend on the order of threads.  The arrays of one
// kind mostly are pieces of one buffer in address order: each kind's are sorted if need be, and the kinds then merged,
// which is only walked through where their spans meet.
struct Range { uintptr_t lo, hi; };
struct Ranges {
  static constexpr int kKinds = 7;
  std::vector<Range> r;
  size_t first[kKinds + 1] = {};
  bool written[kKinds] = {};
  int kinds = 0;
  void add(const void *p, size_t bytes) { r.push_back(Range{(uintptr_t)p, (uintptr_t)p + bytes}); }
  void close_kind(bool is_written) {
    if (r.size() == first[kinds]) return;
    written[kinds] = is_written;
    first[++kinds] = r.size();
  }
  bool overlap() {
    const auto before = [](const Range &a, const Range &b) { return a.lo < b.lo; };
    Range span[kKinds];
    for (int k = 0; k < kinds; ++k) {
      const auto b = r.begin() + (ptrdiff_t)first[k], e = r.begin() + (ptrdiff_t)first[k + 1];
      if (!std::is_sorted(b, e, before)) std::sort(b, e, before);
      span[k] = *b;
      for (auto i = b + 1; i < e; ++i) {
        if (written[k] && i->lo < (i - 1)->hi) return true;
        span[k].hi = std::max(span[k].hi, i->hi);
      }
    }
    std::sort(span, span + kinds, before);
    bool apart = true;
    for (int k = 1; k < kinds; ++k) apart = apart && span[k].lo >= span[k - 1].hi;
    if (apart) return false;
    size_t at[kKinds];
    for (int k = 0; k < kinds; ++k) at[k] = first[k];
    uintptr_t reach = 0, reach_written = 0;   // ends of the arrays met so far
    for (size_t n = 0; n < r.size(); ++n) {
      int least = -1;
      for (int k = 0; k < kinds; ++k)
        if (at[k] < first[k + 1] && (least < 0 || r[at[k]].lo < r[at[least]].lo)) least = k;
      const Range &x = r[at[least]++];
      if (x.lo < (written[least] ? reach : reach_written)) return true;
      reach = std::max(reach, x.hi);
      if (written[least]) reach_written = std::max(reach_written, x.hi);
    }
    return false;
  }
};

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
      const uint64_t n = (uint64_t)t[i].numel, need = kind == kStep8 ? (n + kCodeTile - 1) / kCodeTile : (n + kStepTile - 1) / kStepTile;
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

// launch_pdl without a copy of the table on the way.
template <typename K, int N, typename S>
void launch_step(K kernel, unsigned tiles, unsigned threads, cudaStream_t st, const StepTable<N> &table, const S &scalars) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = tiles;
  cfg.blockDim = threads;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  void *args[] = {const_cast<StepTable<N> *>(&table), const_cast<S *>(&scalars)};
  (void)cudaLaunchKernelExC(&cfg, (const void *)kernel, args);      // its error is the caller's cudaGetLastError
}

// `f` with the size of the smallest table that takes the list, or the largest there is.
template <typename F> int with_table(int count, F f) {
  if (count <= kFewTensors) return f(std::integral_constant<int, kFewTensors>());
  if (count <= kSomeTensors) return f(std::integral_constant<int, kSomeTensors>());
  return f(std::integral_constant<int, kManyTensors>());
}

StepPairs step_pairs(const StepScalars<float> &s) {
  StepPairs c;
  c.grad_scale = both(s.grad_scale);
  c.beta1 = both(s.beta1);
  c.one_minus_beta1 = both(s.one_minus_beta1);
  c.beta2 = both(s.beta2);
  c.one_minus_beta2 = both(s.one_minus_beta2);
  c.keep = both(s.keep);
  c.minus_size = both(-s.size);
  c.root = both(s.root);
  c.eps = both(s.eps);
  c.minus_zero = both(-0.0f);
  c.dither = s.dither;
  return c;
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
      launch_step(adamw_kernel<T, MASTER, N>, tiles, kStepThreads, st, table, s);
    });
  if constexpr (sizeof(T) < 8)
    return launch_table<N>(t, count, sizeof(T), kStep8, [&, pairs = step_pairs(s)](const StepTable<N> &table, unsigned tiles) {
      launch_step(adamw8_kernel<T, MASTER, N>, tiles, kCodeThreads, st, table, pairs);
    });
  return THCB200_ERR_UNSUPPORTED;
}

template <typename T>
int run_step_typed(const thcb200_adamw_tensor *t, int count, int bits, bool master, const thcb200_adamw_args &a, cudaStream_t st) {
  return with_table(count, [&](auto size) {
    if constexpr (sizeof(T) == 2) {
      if (master) return run_step<T, true, size()>(t, count, bits, a, st);
    }
    return run_step<T, false, size()>(t, count, bits, a, st);
  });
}

// Kinds: param, m, v, grad, master, m_unit, v_unit.  The usual list, each kind in address order and apart from the others, is seen in
// one walk (110 tensors 2.8 -> 0.9 us of host time); false for any other, whatever it is.
bool plainly_apart(const thcb200_adamw_tensor *t, int n, const size_t (&size)[Ranges::kKinds]) {
  Range span[Ranges::kKinds] = {};
  for (int i = 0; i < n; ++i) {
    const size_t k = (size_t)t[i].numel, blocks = (k + kUnitItems - 1) / kUnitItems;
    if (k == 0) continue;
    const void *const p[Ranges::kKinds] = {t[i].param, t[i].m, t[i].v, t[i].grad, t[i].master, t[i].m_unit, t[i].v_unit};
#pragma GCC unroll 8
    for (int what = 0; what < Ranges::kKinds; ++what) {
      if (size[what] == 0) continue;
      const uintptr_t lo = (uintptr_t)p[what];
      if (lo < span[what].hi) return false;
      if (span[what].hi == 0) span[what].lo = lo;
      span[what].hi = lo + (what < 5 ? k : blocks) * size[what];
    }
  }
  for (int a = 0; a < Ranges::kKinds; ++a)
    for (int b = 0; b < a; ++b)
      if (span[a].lo < span[b].hi && span[b].lo < span[a].hi) return false;
  return true;
}

int check_list(const thcb200_adamw_tensor *t, int n, size_t esz, StepKind kind, bool master, const char *name) {
  const size_t wsz = esz == 8 ? 8 : 4, msz = kind == kStep32 ? wsz : 1;
  const bool values = kind == kStepValues;
  size_t size[Ranges::kKinds];
  for (int what = 0; what < Ranges::kKinds; ++what) {
    const bool there = what < 3 || (what == 3 && !values) || (what == 4 && (master || values)) || (what > 4 && kind != kStep32);
    const size_t each[Ranges::kKinds] = {values ? 4 : esz, msz, msz, esz, values ? 4 : wsz, 4, 4};
    size[what] = there ? each[what] : 0;
  }
  if (plainly_apart(t, n, size)) return 0;
  Ranges ranges;
  ranges.r.reserve((size_t)n * Ranges::kKinds + 1);
  for (int what = 0; what < Ranges::kKinds; ++what) {
    for (int i = 0; size[what] && i < n; ++i) {
      const size_t k = (size_t)t[i].numel, blocks = (k + kUnitItems - 1) / kUnitItems;
      if (k == 0) continue;
      const void *const p[Ranges::kKinds] = {t[i].param, t[i].m, t[i].v, t[i].grad, t[i].master, t[i].m_unit, t[i].v_unit};
      ranges.add(p[what], (what < 5 ? k : blocks) * size[what]);
    }
    ranges.close_kind(values ? what == 0 || what == 4 : what != 3);
  }
  if (ranges.overlap()) { set_error("%s: a tensor that is written shares memory with another (each may be listed once)", name); return THCB200_ERR_ARG; }
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
  const StepPairs pairs = step_pairs(StepScalars<float>());
  return with_table(n, [&](auto size) {
    constexpr int N = decltype(size)::value;
    return launch_table<N>(tensors, n, 4, kStepValues, [&](const StepTable<N> &table, unsigned tiles) {
      launch_step(adamw_values_kernel<N>, tiles, kStepThreads, st, table, pairs);
    });
  });
}

}  // extern "C"
