// Rows of an embedding table, scaled on the way out, and the table's gradient.
//
//   forward    result[t, :] = scale * weight[index[t], :]
//   gradient   grad_weight[r, :] (+)= scale * sum over the tokens t with index[t] = r of grad_output[t, :]
//
// The gradient adds the tokens of a row in token order, in double (float for half, as the reductions of this library):
// the tokens are sorted by row (keysort.cu), a CTA walks a fixed chunk of the sorted list, and a row whose tokens cross
// chunks is joined from the chunks' partial sums in chunk order.  No atomics on data: results repeat bit for bit, where
// indexAdd adds in any order and, for half, rounds every addend to 11 bits.
#include <cuda_fp16.h>

#include <algorithm>

#include "context.h"
#include "core.cuh"
#include "keysort.h"
#include "plan.h"
#include "rows.cuh"

namespace thcb {
namespace {

constexpr int kLookThreads = 256;
constexpr int kLookUnroll = 4;

// Row of token i, or the row count where it has none.
__device__ __forceinline__ uint32_t row_key(const SortInput &in, int64_t i, bool count) {
  const int64_t raw = in.index[i * in.stride], k = raw - 1;   // positions are 1-based (TH_INDEX_BASE)
  const bool row = (uint64_t)k < (uint64_t)in.limit, skip = in.skip != 0 && raw == in.skip;
  if (!row && !skip && count) atomicAdd(in.errors, 1u);
  return row && !skip ? (uint32_t)k : (uint32_t)in.limit;
}

// One vector of V elements per item, kLookUnroll items per thread: the positions come first, then all row loads are in
// flight together.
template <typename T, int V>
__global__ void __launch_bounds__(kLookThreads)
embedding_kernel(T *out, const T *weight, const int64_t *index, FastDiv32 vecs32, uint64_t vecs, uint64_t items,
                 int64_t index_stride, int64_t rows, int64_t row_stride, int64_t out_stride, typename TypeTraits<T>::Math scale, unsigned int *errors) {
  pdl_prologue();
  const uint64_t base = (uint64_t)blockIdx.x * (kLookThreads * kLookUnroll) + threadIdx.x;
  uint64_t tok[kLookUnroll], col[kLookUnroll];
  int64_t row[kLookUnroll];
#pragma unroll
  for (int u = 0; u < kLookUnroll; ++u) {
    const uint64_t i = base + (uint64_t)u * kLookThreads;
    row[u] = -1;
    if (i >= items) continue;
    if (items <= 0xffffffffull) {
      uint32_t q, r;
      vecs32.divmod((uint32_t)i, q, r);
      tok[u] = q;
      col[u] = r;
    } else {
      tok[u] = i / vecs;
      col[u] = i - tok[u] * vecs;
    }
    row[u] = index[(int64_t)tok[u] * index_stride] - 1;            // positions are 1-based (TH_INDEX_BASE)
  }
  Pack<T, V> x[kLookUnroll];
  unsigned int bad = 0;
#pragma unroll
  for (int u = 0; u < kLookUnroll; ++u) {
    if (base + (uint64_t)u * kLookThreads >= items || (uint64_t)row[u] < (uint64_t)rows) continue;
    bad += col[u] == 0 ? 1u : 0u;
    row[u] = -1;
  }
#pragma unroll
  for (int u = 0; u < kLookUnroll; ++u)
    if (row[u] >= 0) x[u] = load_pack<T, V>(weight + row[u] * row_stride + (int64_t)(col[u] * V));
#pragma unroll
  for (int u = 0; u < kLookUnroll; ++u) {
    if (row[u] < 0) continue;
#pragma unroll
    for (int e = 0; e < V; ++e) x[u].e[e] = from_math<T>(to_math(x[u].e[e]) * scale);
    store_pack<T, V>(out + (int64_t)tok[u] * out_stride + (int64_t)(col[u] * V), x[u]);
  }
  if (bad) atomicAdd(errors, bad);
}

// Rows of single elements: a warp, or a team of 4, 8 or 16 lanes for narrow rows, takes kLookItems elements per lane, a team's width
// apart, of a token's row, and reads its position once: 20000 tokens of 2047 halves 34 us, 5003 of 1001 floats 5.3 us, where elements
// taken one by one took 103 and 13.4.  It is bound by instructions (79 % of the issue slots before addresses were constants apart, 55 us).
template <typename T> constexpr int kLookItems = sizeof(T) == 8 ? 4 : 8;
// PLAIN: whole warps and neighbouring columns, so that a lane's addresses are one and constants.
template <typename T, bool PLAIN>
__global__ void __launch_bounds__(kLookThreads)
embedding_single_kernel(T *out, const T *weight, const int64_t *index, FastDiv32 per32, uint64_t per, uint64_t items, uint32_t bits, int64_t width,
                        int64_t index_stride, int64_t rows, int64_t row_stride, int64_t col_stride, int64_t out_stride, typename TypeTraits<T>::Math scale,
                        unsigned int *errors) {
  constexpr int G = kLookItems<T>;
  pdl_prologue();
  const uint32_t team_bits = PLAIN ? 5 : bits;
  const uint64_t unit = ((uint64_t)blockIdx.x * kLookThreads + threadIdx.x) >> team_bits;
  if (unit >= items) return;
  uint64_t token, stretch;
  if (items <= 0xffffffffull) {
    uint32_t q, r;
    per32.divmod((uint32_t)unit, q, r);
    token = q;
    stretch = r;
  } else {
    token = unit / per;
    stretch = unit - token * per;
  }
  const uint32_t team = 1u << team_bits, lane = threadIdx.x & (team - 1);
  const int64_t col0 = (int64_t)(stretch * G << team_bits) + lane, row = index[(int64_t)token * index_stride] - 1;   // positions are 1-based
  if ((uint64_t)row >= (uint64_t)rows) {
    if (col0 == 0) atomicAdd(errors, 1u);
    return;
  }
  const T *p = weight + row * row_stride + (PLAIN ? col0 : col0 * col_stride);
  T *q = out + (int64_t)token * out_stride + col0;
  const int64_t step = PLAIN ? 32 : team * col_stride;
  if (width <= col0) return;
  const uint32_t left = (uint32_t)min(width - col0, (int64_t)(G * 32));       // columns from the lane's first on
  T x[G];
#pragma unroll
  for (int g = 0; g < G; ++g)
    if (g * team < left) x[g] = p[g * step];
#pragma unroll
  for (int g = 0; g < G; ++g)
    if (g * team < left) q[g * team] = from_math<T>(to_math(x[g]) * scale);
}

// ---- gradient ----------------------------------------------------------------------------------
constexpr int kGradThreads = 256;
// Rows on their way while others are added, kGradBatch at a time: vectors by asynchronous copies into shared memory,
// kGradStages batches of them; single elements, whose copies cost more instructions than they save, by loads.  A thread takes
// kGradCols single elements of a row: 9979 tokens of 545 halves, 5003 of 1001 floats and 6000 of 2047 halves take 29.9, 27.5 and 42.3 us
// by one (8 rows in a batch), 26.7, 24.6 and 36.8 by two, 27.6, 24.8 and 33.1 by four (of 2 rows).
constexpr int kGradStages = 3;
constexpr int kGradBatch = 4;
template <typename T, int V> constexpr bool kGradCopies = V > 1;
template <typename T, int V> constexpr int kGradCols = V > 1 ? 1 : 2;
template <typename T, int V> constexpr size_t kGradRing = kGradCopies<T, V> ? kGradStages * kGradBatch * kGradThreads * sizeof(T) * V : 0;
constexpr int kGradMaxChunk = 64;    // sorted tokens per CTA
constexpr int kGradKeys = 1024;      // sorted tokens per CTA where rows are narrow and it takes several chunks
constexpr uint32_t kJoinChunks = 64; // partial sums that one CTA joins
constexpr uint32_t kGradMinChunk = 8, kGradMinGroup = 4;
// Words a CTA's groups hold their tokens' keys and places in, and at most: kGradKeys tokens, or the shortest chunk for every group.
constexpr uint32_t grad_words(uint32_t groups, uint32_t chunk) { return groups * (4 * chunk + 2); }
constexpr uint32_t kGradMaxWords = 4 * kGradKeys + 2 * kGradThreads / kGradMinGroup;
static_assert(kGradMinChunk * kGradThreads / kGradMinGroup <= kGradKeys && kGradMaxWords >= kGradThreads, "also the flags of the rows a CTA clears");

template <typename T> struct GradArgs {
  T *table;
  const T *grad;
  const uint32_t *key, *pos;
  SortInput index;                           // the positions themselves, for few tokens
  typename TypeTraits<T>::Acc *partial;      // [chunk][head, tail][width]
  uint32_t *start_count;                     // rows that lie across more than two chunks
  uint4 *starts;                             // for each, or each section: the chunk it begins in, the chunks behind that, its key, the section
  int64_t tokens, width, rows;
  int64_t grad_stride, grad_col, table_stride;
  uint32_t chunk, chunks;
  uint32_t group_bits;                       // 2^group_bits threads take a chunk together: 256 for wide rows
  uint32_t sum_ctas, zero_rows;              // CTAs that sum; table rows that one of the others checks and clears
  typename TypeTraits<T>::Acc scale;
};

// A row's sum, rounded once: over what is there or, `old` holding it, added to it.
template <typename T, int V, bool ADD>
__device__ __forceinline__ void write_row(const GradArgs<T> &a, uint32_t key, int64_t col, const typename TypeTraits<T>::Acc (&acc)[V], const Pack<T, V> &old) {
  using Acc = typename TypeTraits<T>::Acc;
  Pack<T, V> out;
#pragma unroll
  for (int e = 0; e < V; ++e) out.e[e] = ADD ? round_from<T>((Acc)to_math(old.e[e]) + acc[e] * a.scale) : round_from<T>(acc[e] * a.scale);
  store_pack<T, V>(a.table + (int64_t)key * a.table_stride + col, out);
}

// Partial sums lie in rows of `width` accumulators, on 16-byte boundaries where the rows' elements are taken in vectors.
template <typename T, int V>
__device__ __forceinline__ void add_partial(typename TypeTraits<T>::Acc (&acc)[V], const typename TypeTraits<T>::Acc *p) {   // past L1
  using Acc = typename TypeTraits<T>::Acc;
  constexpr int W = V > 1 ? 16 / sizeof(Acc) : 1;
#pragma unroll
  for (int e = 0; e < V; e += W) {
    if constexpr (V > 1) {
      const int4 raw = __ldcg(reinterpret_cast<const int4 *>(p + e));
      const Pack<Acc, W> x = *reinterpret_cast<const Pack<Acc, W> *>(&raw);
#pragma unroll
      for (int k = 0; k < W; ++k) acc[e + k] += x.e[k];
    } else {
      acc[e] += __ldcg(p + e);
    }
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_sums(typename TypeTraits<T>::Acc *p, const typename TypeTraits<T>::Acc (&acc)[V]) {
  using Acc = typename TypeTraits<T>::Acc;
  constexpr int W = V > 1 ? 16 / sizeof(Acc) : 1;
#pragma unroll
  for (int e = 0; e < V; e += W) {
    Pack<Acc, W> x;
#pragma unroll
    for (int k = 0; k < W; ++k) x.e[k] = acc[e + k];
    *reinterpret_cast<Pack<Acc, W> *>(p + e) = x;
  }
}

// CTAs 0 .. chunks-1 sum the rows named in their chunk of the sorted tokens; the ones behind clear the rows no token
// names (accumulate = 0).
// FEW: every CTA puts all tokens (at most kFewTokens) in order itself, and a row is summed by the chunk it begins in however
// long it is: no sort before and no join behind.  One launch for three saves 1.2 to 2.4 us on rows that hardly repeat (64
// tokens of 1024 halves 6.7 -> 5.4, of 1001 floats 6.5 -> 4.1), but a row's tokens are then added one after another, 0.28 us
// each: all 64 the same 8.1 -> 18.8 us, all 128 9.9 -> 36.4.  64 bounds what that can cost.
constexpr int kFewTokens = 64;

template <typename T, int V, bool ADD, bool FEW>
__global__ void __launch_bounds__(kGradThreads, 4)
embedding_grad_kernel(GradArgs<T> a) {
  using Acc = typename TypeTraits<T>::Acc;
  constexpr int B = kGradBatch;
  pdl_prologue();
  const uint32_t group = 1u << a.group_bits, groups = kGradThreads >> a.group_bits, mine = threadIdx.x >> a.group_bits, member = threadIdx.x & (group - 1);
  constexpr int G = kGradCols<T, V>;
  const int64_t col = ((int64_t)blockIdx.y * (G * group) + member) * V, apart = group * V;      // column g of the thread: col + g * apart
  extern __shared__ Bytes16 grad_dynamic[];
  Pack<T, V> *grad_ring = reinterpret_cast<Pack<T, V> *>(grad_dynamic);
  uint32_t *grad_smem = reinterpret_cast<uint32_t *>(reinterpret_cast<char *>(grad_dynamic) + kGradRing<T, V>);
  __shared__ uint32_t few_raw[FEW ? kFewTokens : 1], few_key[FEW ? kFewTokens + 2 : 1], few_pos[FEW ? kFewTokens : 1];
  if constexpr (FEW) {
    const uint32_t i = threadIdx.x, n = (uint32_t)a.tokens;
    if (i < n) few_raw[i] = row_key(a.index, i, blockIdx.x == 0 && blockIdx.y == 0);
    __syncthreads();
    if (i < n) {
      const uint32_t k = few_raw[i];
      uint32_t place = 0;
      for (uint32_t j = 0; j < n; ++j) place += few_raw[j] < k || (few_raw[j] == k && j < i) ? 1u : 0u;
      few_key[place + 1] = k;
      few_pos[place] = i;
    }
    if (i == 0) {
      few_key[0] = 0xfffffffeu;
      few_key[n + 1] = 0xffffffffu;
    }
    __syncthreads();
  }
  const uint32_t *sorted = FEW ? few_key + 1 : a.key;
  if (blockIdx.x >= a.sum_ctas) {
    const int64_t row0 = (int64_t)(blockIdx.x - a.sum_ctas) * a.zero_rows;
    if (threadIdx.x < a.zero_rows) {
      const int64_t row = row0 + threadIdx.x;
      // first sorted key that is not below the row
      int64_t lo = 0, hi = a.tokens;
      while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if ((int64_t)sorted[mid] < row) lo = mid + 1; else hi = mid;
      }
      grad_smem[threadIdx.x] = row >= a.rows || (lo < a.tokens && (int64_t)sorted[lo] == row);
    }
    __syncthreads();
    if (col >= a.width) return;
    Pack<T, V> zero;
#pragma unroll
    for (int e = 0; e < V; ++e) zero.e[e] = round_from<T>((Acc)0);
    for (uint32_t r = mine; r < a.zero_rows; r += groups)
      if (!grad_smem[r]) {
#pragma unroll
        for (int g = 0; g < G; ++g)
          if (g == 0 || col + g * apart < a.width) store_pack<T, V>(a.table + (row0 + r) * a.table_stride + col + g * apart, zero);
      }
    return;
  }
  const uint32_t index = blockIdx.x * groups + mine;            // the group's chunk
  const int64_t begin = (int64_t)index * a.chunk;
  uint32_t *skey = FEW ? few_key + min(begin, a.tokens) : grad_smem + mine * (2 * a.chunk + 2);
  uint32_t *spos = FEW ? few_pos + min(begin, a.tokens) : grad_smem + groups * (2 * a.chunk + 2) + mine * 2 * a.chunk;
  const uint32_t own = index < a.chunks ? (uint32_t)min((int64_t)a.chunk, a.tokens - begin) : 0;
  const uint32_t seen = index < a.chunks ? (uint32_t)min(FEW ? a.tokens : (int64_t)2 * a.chunk, a.tokens - begin) : 0;
  // skey[0]: the key in front of the chunk; then the chunk's, the next chunk's, and the one behind (a sentinel ends the list)
  if (!FEW && own > 0) {
    for (uint32_t i = member; i < seen + 2; i += group) {
      const int64_t p = begin + (int64_t)i - 1;
      skey[i] = p < 0 ? 0xfffffffeu : a.key[p];
      if (i >= 1 && i <= seen) spos[i - 1] = a.pos[p];
    }
  }
  const uint32_t none = (uint32_t)a.rows;
  // the row that is under way at the chunk's start, and the one at its end
  const bool wide_open = !FEW && own > 0 && begin > a.chunk && a.key[begin - a.chunk - 1] == a.key[begin];   // began before the last chunk
  __syncthreads();
  if (col >= a.width || own == 0) return;
  const uint32_t first = skey[1], last = skey[own];
  const bool head = skey[0] == first;
  const bool goes_on = skey[own + 1] == last, far = !FEW && seen == 2 * a.chunk && skey[2 * a.chunk + 1] == last;
  // A row that began in the last chunk and ends in this one was that chunk's; one that lies across more chunks leaves its
  // sum over this one for the join.
  const bool head_long = !FEW && head && (wide_open || (goes_on && first == last));
  const bool tail_long = goes_on && far;               // a row that began here: it does not end in the next chunk either
  uint32_t from = 0, to = own;
  if (head && !head_long)
    while (from < own && skey[from + 1] == first) ++from;
  if (goes_on && !tail_long && !(head && first == last))
    while (to < seen && skey[to + 1] == last) ++to;
  if (last == none)                                    // items without a row come last
    for (to = from; to < own && skey[to + 1] != none;) ++to;
  Acc acc[G][V];
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int e = 0; e < V; ++e) acc[g][e] = 0;
  const auto there = [&](int g) { return g == 0 || col + g * apart < a.width; };
  const auto row_ends = [&](uint32_t i) { return i + 1 >= to || skey[i + 2] != skey[i + 1]; };
  // Adds token i; the sum of a row that ends there goes to the table, over `old` or not, or to the partial sums.
  const auto add = [&](const Pack<T, V> *x, uint32_t i, const Pack<T, V> *old) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int e = 0; e < V; ++e) acc[g][e] += (Acc)to_math(x[g].e[e]);
    if (!row_ends(i)) return;
    const uint32_t key = skey[i + 1];
    const bool in_head = head_long && key == first, in_tail = tail_long && key == last;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (there(g)) {
        if (in_head || in_tail) store_sums<T, V>(a.partial + ((int64_t)index * 2 + (in_head ? 0 : 1)) * a.width + col + g * apart, acc[g]);
        else write_row<T, V, ADD>(a, key, col + g * apart, acc[g], old[g]);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) acc[g][e] = 0;
    }
  };
  Pack<T, V> old[ADD ? B : 1][G];
  // what the sum of a row that ends at token i is added to comes with the token's batch
  const auto read_old = [&](Pack<T, V> (&o)[ADD ? B : 1][G], uint32_t i, int u) {
    if (!ADD || !row_ends(i)) return;
#pragma unroll
    for (int g = 0; g < G; ++g)
      if (there(g)) o[ADD ? u : 0][g] = load_pack<T, V>(a.table + (int64_t)skey[i + 1] * a.table_stride + col + g * apart);
  };
  if constexpr (kGradCopies<T, V>) {
    // every thread copies what it will add itself, so that no barrier is needed: two batches on their way while one is added
    const auto copy = [&](uint32_t i0, int stage) {
#pragma unroll
      for (int u = 0; u < B; ++u)
        if (i0 + u < to)
          copy_async<T, V>(&grad_ring[(stage * B + u) * kGradThreads + threadIdx.x], a.grad + (int64_t)spos[i0 + u] * a.grad_stride + col * a.grad_col);
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    copy(from, 0);
    copy(from + B, 1);
    int stage = 0;
    for (uint32_t i = from; i < to; i += B) {
      copy(i + 2 * B, stage == 0 ? 2 : stage - 1);
#pragma unroll
      for (int u = 0; u < B; ++u)
        if (i + u < to) read_old(old, i + u, u);
      asm volatile("cp.async.wait_group 2;" ::: "memory");
#pragma unroll
      for (int u = 0; u < B; ++u) {
        if (i + u >= to) break;
        add(&grad_ring[(stage * B + u) * kGradThreads + threadIdx.x], i + u, old[ADD ? u : 0]);
      }
      stage = stage == 2 ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  } else {
    for (uint32_t i = from; i < to; i += B) {
      Pack<T, V> x[B][G];
#pragma unroll
      for (int u = 0; u < B; ++u) {
        if (i + u >= to) continue;
#pragma unroll
        for (int g = 0; g < G; ++g)
          if (there(g)) x[u][g] = load_pack<T, V>(a.grad + (int64_t)spos[i + u] * a.grad_stride + (col + g * apart) * a.grad_col);
        read_old(old, i + u, u);
      }
#pragma unroll
      for (int u = 0; u < B; ++u) {
        if (i + u >= to) break;
        add(x[u], i + u, old[ADD ? u : 0]);
      }
    }
  }
  // A row across more than two chunks is joined later: its chunks whose first token is the row's, the next two at least.
  if (!FEW && blockIdx.y == 0 && member == 0 && tail_long && last != none && !(head && first == last)) {
    int64_t lo = (int64_t)index + 3, hi = a.chunks, reach = 2;
    while (lo + reach < hi && a.key[(lo + reach) * a.chunk] == last) { lo += reach + 1; reach *= 2; }
    hi = min(hi, lo + reach);
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (a.key[mid * a.chunk] == last) lo = mid + 1; else hi = mid;
    }
    const uint32_t count = (uint32_t)(lo - 1 - (int64_t)index), sections = (count + kJoinChunks - 1) / kJoinChunks;
    if (sections > 1) {
      // the next chunk is this row's throughout and leaves its second place free: it counts the sections that are done
      uint32_t *done = reinterpret_cast<uint32_t *>(a.partial + ((int64_t)index * 2 + 3) * a.width);
      for (int64_t p = 0; p < (a.width + 32 * V - 1) / (32 * V); ++p) done[p] = 0;
    }
    const uint32_t at = atomicAdd(a.start_count, sections);
    for (uint32_t s = 0; s < sections; ++s) a.starts[at + s] = make_uint4(index, count, last, s);
  }
}

// Joins the rows whose tokens cross chunks.  `starts` lists the chunks in which such a row begins (in the order their CTAs came
// by, which no result depends on); a CTA takes a row and a piece of its columns, its warps take runs of the row's chunks, and
// the warps' sums are added in chunk order.  A row of more than kJoinChunks chunks is listed once for each section of that
// many; the CTA that ends last adds the sections' sums, in their order.  (One row for all tokens, by one CTA and by sections:
// 65536 of 64 halves 165 -> 34 us, 200000 of 2048 halves 300 -> 201.)
constexpr int kJoinWarps = kGradThreads / 32;

template <typename T, int V, bool ADD>
__global__ void __launch_bounds__(kGradThreads)
embedding_grad_join_kernel(GradArgs<T> a) {
  using Acc = typename TypeTraits<T>::Acc;
  pdl_prologue();
  __shared__ Acc part[kJoinWarps][32 * V];
  __shared__ uint32_t ended;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t entries = *a.start_count, pieces = (uint32_t)((a.width + 32 * V - 1) / (32 * V));
  for (uint64_t job = blockIdx.x; job < (uint64_t)entries * pieces; job += gridDim.x) {
    const uint4 row = a.starts[job / pieces];
    const uint32_t piece = (uint32_t)(job % pieces), sections = (row.y + kJoinChunks - 1) / kJoinChunks;
    const int64_t col = ((int64_t)piece * 32 + lane) * V, stride = 2 * a.width;
    Acc acc[V];
    // the sum of the n partial sums from p on, `step` apart, and of `more`: complete in the first warp
    const auto join = [&](const Acc *p, int64_t step, uint32_t n, const Acc *more) {
      const uint32_t per = (n + kJoinWarps - 1) / kJoinWarps, from = min(warp * per, n), to = min(from + per, n);
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] = 0;
      if (col < a.width) {
        if (more && warp == 0) add_partial<T, V>(acc, more);
#pragma unroll 8
        for (uint32_t c = from; c < to; ++c) add_partial<T, V>(acc, p + c * step);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) part[warp][lane * V + e] = acc[e];
      __syncthreads();
      if (warp == 0 && col < a.width) {
#pragma unroll
        for (int w = 1; w < kJoinWarps; ++w)
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] += part[w][lane * V + e];
      }
    };
    Pack<T, V> old;
    if (ADD && warp == 0 && col < a.width) old = load_pack<T, V>(a.table + (int64_t)row.z * a.table_stride + col);
    Acc *const behind = a.partial + ((int64_t)row.x + 1) * stride + col;      // the first chunk after the one it begins in
    const uint32_t first = row.w * kJoinChunks;
    join(behind + first * stride, stride, min(row.y - first, kJoinChunks), row.w == 0 ? behind - a.width : nullptr);
    if (sections > 1) {
      if (warp == 0) {
        if (col < a.width) store_sums<T, V>(behind + first * stride, acc);
        __threadfence();
        __syncwarp();
        if (lane == 0) ended = atomicAdd(reinterpret_cast<uint32_t *>(a.partial + ((int64_t)row.x * 2 + 3) * a.width) + piece, 1u) + 1;
      }
      __syncthreads();
      const bool all = ended == sections;
      if (all) {
        __threadfence();
        join(behind, kJoinChunks * stride, sections, nullptr);
      } else {
        __syncthreads();           // `ended` is read before the next job
        continue;
      }
    }
    if (warp == 0 && col < a.width) write_row<T, V, ADD>(a, row.z, col, acc, old);
    __syncthreads();
  }
}

// ---- host --------------------------------------------------------------------------------------
template <typename T>
int run_embedding(thcb200_ctx *ctx, const MatView &out, const MatView &w, const int64_t *index, int64_t index_stride, double scale,
                  cudaStream_t st) {
  using Math = typename TypeTraits<T>::Math;
  unsigned int *errors = index_errors(ctx);
  const int bytes = mat_vec(out, sizeof(T), 32) && mat_vec(w, sizeof(T), 32) ? 32 : mat_vec(out, sizeof(T), 16) && mat_vec(w, sizeof(T), 16) ? 16 : sizeof(T);
  if (bytes == (int)sizeof(T)) {
    constexpr int G = kLookItems<T>;
    uint32_t team_bits = 5;
    while (team_bits > 2 && (int64_t)(G << (team_bits - 1)) >= out.cols) --team_bits;
    const uint64_t per = ((uint64_t)out.cols + (G << team_bits) - 1) / (G << team_bits), items = per * (uint64_t)out.rows;
    const uint64_t per_cta = kLookThreads >> team_bits, blocks = (items + per_cta - 1) / per_cta;
    if (blocks >= (1ull << 31) || per >= (1ull << 31)) { set_error("embedding: tensor too large"); return THCB200_ERR_LIMIT; }
    launch_pdl(team_bits == 5 && w.col_stride == 1 ? embedding_single_kernel<T, true> : embedding_single_kernel<T, false>, (unsigned)blocks, kLookThreads, 0,
               st, (T *)out.data, (const T *)w.data, index, FastDiv32((uint32_t)per), per, items, team_bits, out.cols, index_stride, w.rows, w.row_stride,
               w.col_stride, out.row_stride, (Math)scale, errors);
    count_launch();
    THCB_CUDA_TRY(cudaGetLastError());
    return 0;
  }
  const uint64_t vecs = (uint64_t)out.cols * sizeof(T) / bytes;
  const uint64_t items = vecs * (uint64_t)out.rows;
  const uint64_t blocks = (items + kLookThreads * kLookUnroll - 1) / (kLookThreads * kLookUnroll);
  if (blocks >= (1ull << 31) || vecs >= (1ull << 31)) { set_error("embedding: tensor too large"); return THCB200_ERR_LIMIT; }
  const FastDiv32 div((uint32_t)vecs);
  auto launch = [&](auto kernel) {
    launch_pdl(kernel, (unsigned)blocks, kLookThreads, 0, st, (T *)out.data, (const T *)w.data, index, div, vecs, items, index_stride, w.rows,
               w.row_stride, out.row_stride, (Math)scale, errors);
  };
  if (bytes == 32) launch(embedding_kernel<T, 32 / sizeof(T)>);
  else launch(embedding_kernel<T, 16 / sizeof(T)>);
  count_launch();
  THCB_CUDA_TRY(cudaGetLastError());
  return 0;
}

uint32_t grad_chunk(int64_t tokens, uint32_t groups, int64_t slabs) {
  // long chunks leave fewer partial sums, short ones give every SM several CTAs (8, 6, 4 and 2 of them: 65536 tokens of 2048
  // halves 156.5, 152.6, 152.7, 152.7 us, 5003 of 1001 floats 29.1, 29.1, 31.1, 38.5, 10562 of 2368 42.3, 38.7, 38.7, 41.2)
  uint32_t c = kGradMaxChunk;
  while (c > kGradMinChunk && (c * groups > kGradKeys || tokens / (c * groups) * slabs < 6 * kNumSM_B200)) c >>= 1;
  return c;
}

template <typename T>
int run_embedding_grad(thcb200_ctx *ctx, const MatView &table, const MatView &grad, const SortInput &in, double scale, int accumulate,
                       cudaStream_t st) {
  using Acc = typename TypeTraits<T>::Acc;
  constexpr int VB = 16 / sizeof(T);
  const bool vec = mat_vec(table, sizeof(T), 16) && mat_vec(grad, sizeof(T), 16);
  const int64_t vecs = vec ? table.cols / VB : table.cols;
  uint32_t group_bits = 8;
  const int cols = vec ? kGradCols<T, VB> : kGradCols<T, 1>;
  while ((1u << group_bits) > kGradMinGroup && (cols << (group_bits - 1)) >= vecs) --group_bits;
  const uint32_t group = 1u << group_bits, groups = kGradThreads >> group_bits, zero_rows = groups >= 8 ? kGradThreads : 32;
  const int64_t slabs = (vecs + cols * group - 1) / (cols * group);
  const uint32_t chunk = grad_chunk(in.n, groups, slabs);
  const int64_t chunks = (in.n + chunk - 1) / chunk, sum_ctas = (chunks + groups - 1) / groups;
  const int64_t zero = accumulate ? 0 : (table.rows + zero_rows - 1) / zero_rows;
  if (chunks + zero >= (1ll << 31) || slabs > 65535) { set_error("embeddingAccGrad: tensor too large"); return THCB200_ERR_LIMIT; }
  const size_t nk = ((size_t)(in.n + 1) * 4 + 255) & ~(size_t)255, np = ((size_t)in.n * 4 + 255) & ~(size_t)255;
  const size_t pb = ((size_t)chunks * 2 * (size_t)table.cols * sizeof(Acc) + 255) & ~(size_t)255, sb = ((size_t)(chunks + 1) * sizeof(uint4) + 255) & ~(size_t)255;
  const bool few = in.n <= kFewTokens;
  Workspace ws(ctx, few ? 0 : nk + np + pb + sb + sort_by_key_bytes(in.n, in.limit), st);
  if (!ws.ok) return THCB200_ERR_NOMEM;
  GradArgs<T> a;
  a.index = in;
  a.key = (uint32_t *)ws.data;
  a.pos = (uint32_t *)(ws.data + nk);
  a.partial = (Acc *)(ws.data + nk + np);
  a.start_count = (uint32_t *)(ws.data + nk + np + pb);
  a.starts = (uint4 *)a.start_count + 1;
  if (!few) {
    const int rc = sort_by_key(in, (uint32_t *)a.key, (uint32_t *)a.pos, a.start_count, ws.data + nk + np + pb + sb, st);
    if (rc) return rc;
  }
  a.table = (T *)table.data;
  a.grad = (const T *)grad.data;
  a.tokens = in.n;
  a.width = table.cols;
  a.rows = table.rows;
  a.grad_stride = grad.row_stride;
  a.grad_col = vec ? 1 : grad.col_stride;
  a.table_stride = table.row_stride;
  a.chunk = chunk;
  a.chunks = (uint32_t)chunks;
  a.group_bits = group_bits;
  a.sum_ctas = (uint32_t)sum_ctas;
  a.zero_rows = zero_rows;
  a.scale = (Acc)scale;
  const dim3 grid((unsigned)(sum_ctas + zero), (unsigned)slabs);
  const size_t ring = vec ? kGradRing<T, VB> : kGradRing<T, 1>, smem = ring + std::max(grad_words(groups, chunk), zero_rows) * sizeof(uint32_t);
  const size_t most = ring + kGradMaxWords * sizeof(uint32_t);             // 64.5 KiB
  const int64_t piece = vec ? 32 * VB : 32, pieces = (table.cols + piece - 1) / piece;
  const unsigned join = (unsigned)(chunks * pieces < 8 * kNumSM_B200 ? chunks * pieces : 8 * kNumSM_B200);
  const bool joined = !few && chunks > 2;      // a row across more than two chunks needs three
  auto sum = [&](auto kernel) -> int {
    // the limit is the kernel's, not the call's: what one call needs would be below what another thread's is about to launch with
    if (most + 2048 > 48 * 1024) THCB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
    launch_pdl(kernel, grid, kGradThreads, smem, st, a);
    return 0;
  };
  int rc = 0;
#define THCB_GRAD(V, ADD) \
  do { \
    rc = few ? sum(embedding_grad_kernel<T, V, ADD, true>) : sum(embedding_grad_kernel<T, V, ADD, false>); \
    if (!rc && joined) launch_pdl(embedding_grad_join_kernel<T, V, ADD>, join, kGradThreads, 0, st, a); \
  } while (0)
  if (vec && accumulate) THCB_GRAD(VB, true);
  else if (vec) THCB_GRAD(VB, false);
  else if (accumulate) THCB_GRAD(1, true);
  else THCB_GRAD(1, false);
#undef THCB_GRAD
  if (rc) return rc;
  count_launch(joined ? 2 : 1);
  THCB_CUDA_TRY(cudaGetLastError());
  return 0;
}

}  // namespace
}  // namespace thcb

using namespace thcb;

extern "C" {

int thcb200_embedding(thcb200_ctx *ctx, const thcb200_tensor *result, const thcb200_tensor *weight, const thcb200_tensor *index, double scale,
                      void *stream) {
  if (!ctx) { set_error("embedding: null context"); return THCB200_ERR_ARG; }
  MatView out, w;
  HostView vi;
  int rc = to_mat_view(result, &out, "embedding result");
  if (!rc) rc = to_mat_view(weight, &w, "embedding weight");
  if (!rc) rc = to_host_view(index, &vi, "embedding index");
  if (rc) return rc;
  if (!floating(w.dtype) || out.dtype != w.dtype) { set_error("embedding: weight and result must be of one floating-point type"); return THCB200_ERR_ARG; }
  if (vi.dtype != THCB200_I64 || vi.ndim != 1) { set_error("embedding: the index must be a vector of I64"); return THCB200_ERR_ARG; }
  if (out.cols != w.cols || out.rows != vi.sizes[0]) { set_error("embedding: sizes do not match"); return THCB200_ERR_SIZE; }
  if (!dense_rows(out)) { set_error("embedding: the result must have dense rows that do not overlap"); return THCB200_ERR_ARG; }
  if (out.rows == 0 || out.cols == 0) return THCB200_OK;
  cudaStream_t st = (cudaStream_t)stream;
  set_plan_name("embedding");
  switch (w.dtype) {
    case THCB200_F16: return run_embedding<__half>(ctx, out, w, (const int64_t *)vi.data, vi.strides[0], scale, st);
    case THCB200_F32: return run_embedding<float>(ctx, out, w, (const int64_t *)vi.data, vi.strides[0], scale, st);
    default: return run_embedding<double>(ctx, out, w, (const int64_t *)vi.data, vi.strides[0], scale, st);
  }
}

int thcb200_embedding_grad(thcb200_ctx *ctx, const thcb200_tensor *grad_weight, const thcb200_tensor *grad_output, const thcb200_tensor *index,
                           double scale, int64_t padding_index, int accumulate, void *stream) {
  if (!ctx) { set_error("embedding_grad: null context"); return THCB200_ERR_ARG; }
  MatView table, grad;
  HostView vi;
  int rc = to_mat_view(grad_weight, &table, "embedding_grad gradient");
  if (!rc) rc = to_mat_view(grad_output, &grad, "embedding_grad output gradient");
  if (!rc) rc = to_host_view(index, &vi, "embedding_grad index");
  if (rc) return rc;
  if (!floating(table.dtype) || grad.dtype != table.dtype) { set_error("embedding_grad: both gradients must be of one floating-point type"); return THCB200_ERR_ARG; }
  if (vi.dtype != THCB200_I64 || vi.ndim != 1) { set_error("embedding_grad: the index must be a vector of I64"); return THCB200_ERR_ARG; }
  if (grad.cols != table.cols || grad.rows != vi.sizes[0]) { set_error("embedding_grad: sizes do not match"); return THCB200_ERR_SIZE; }
  if (padding_index < 0 || padding_index > table.rows) { set_error("embedding_grad: padding index out of range"); return THCB200_ERR_ARG; }
  if (!dense_rows(table)) { set_error("embedding_grad: the table's gradient must have dense rows that do not overlap"); return THCB200_ERR_ARG; }
  if (table.rows == 0 || table.cols == 0 || (grad.rows == 0 && accumulate)) return THCB200_OK;
  if (table.rows > kSortMaxKeys || grad.rows > kSortMaxItems) { set_error("embedding_grad: more than 2^31 rows or tokens"); return THCB200_ERR_LIMIT; }
  THCB_CTX_LOCK(ctx);
  SortInput in;
  in.index = (const int64_t *)vi.data;
  in.stride = vi.strides[0];
  in.n = grad.rows;
  in.limit = table.rows;
  in.skip = padding_index;
  in.zero_is_none = 0;
  in.errors = index_errors(ctx);
  cudaStream_t st = (cudaStream_t)stream;
  set_plan_name("embedding_grad");
  switch (table.dtype) {
    case THCB200_F16: return run_embedding_grad<__half>(ctx, table, grad, in, scale, accumulate, st);
    case THCB200_F32: return run_embedding_grad<float>(ctx, table, grad, in, scale, accumulate, st);
    default: return run_embedding_grad<double>(ctx, table, grad, in, scale, accumulate, st);
  }
}

}  // extern "C"
