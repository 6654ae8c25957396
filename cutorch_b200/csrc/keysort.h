// Stable sort of row numbers: the order in which the embedding gradient adds its tokens and in which the
// expert calls lay out theirs.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "context.h"

namespace thcb {

constexpr int64_t kSortMaxItems = (1ll << 31) - (1ll << 16);   // positions and tile arithmetic stay below 2^31
constexpr int64_t kSortMaxKeys = (1ll << 31) - 2;
constexpr int kSortMaxBins = 2048;                             // keys of one counting pass

// keys[i] = index[i * stride] - 1 when that lies in [0, limit) and index[i] != skip; `limit` otherwise, so that the
// items without a row come last.  An item that is neither 0-with-zero_is_none, nor skip, nor a row is counted in *errors.
struct SortInput {
  const int64_t *index;
  int64_t stride;
  int64_t n;
  int64_t limit;
  int64_t skip;         // 0: none
  int zero_is_none;     // position 0 is not an error
  unsigned int *errors;
};

// Workspace of sort_by_key for this many items.
size_t sort_by_key_bytes(int64_t n, int64_t limit);
// out_key[p], out_pos[p]: key and item number of the p-th item in (key, item number) order; both hold n entries
// followed by one sentinel key (0xffffffff) in out_key.  *zero becomes 0 on the way.
int sort_by_key(const SortInput &in, uint32_t *out_key, uint32_t *out_pos, uint32_t *zero, void *ws, cudaStream_t st);

// One counting pass over at most kSortMaxBins - 1 keys: slot[i] = 1-based place of item i (0 for an item without a
// key), order[p] = 1-based item at place p (0 behind the last), offsets[e] = items with a key below e, e = 0 .. limit.
size_t sort_to_slots_bytes(int64_t n, int64_t limit);
int sort_to_slots(const SortInput &in, int64_t *slot, int64_t *order, int64_t *offsets, void *ws, cudaStream_t st);

}  // namespace thcb
