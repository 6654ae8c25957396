// What the calls that move whole rows share (embedding.cu, expert.cu): matrices with any row stride, vectors of
// elements, and the workspace of a call.
#pragma once

#include <cuda_fp16.h>

#include "context.h"
#include "core.cuh"
#include "plan.h"

namespace thcb {

// V neighbouring elements moved by one access.
template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T e[V]; };

template <typename T, int V> __device__ __forceinline__ Pack<T, V> load_pack(const T *p) {
  Pack<T, V> x;
  if constexpr (sizeof(T) * V == 16) {
    const Bytes16 b = ld16_stream(p);
    memcpy(&x, &b, 16);
  } else if constexpr (sizeof(T) * V == 32) {
    const Bytes32 b = ld32_stream(p);
    memcpy(&x, &b, 32);
  } else {
    x = *reinterpret_cast<const Pack<T, V> *>(p);
  }
  return x;
}
// The same for rows that other warps of the CTA read as well: through the L1.
template <typename T, int V> __device__ __forceinline__ Pack<T, V> load_kept(const T *p) {
  Pack<T, V> x;
  if constexpr (sizeof(T) * V == 32) {
    Bytes32 b;
    asm volatile("ld.global.v8.u32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(b.w[0]), "=r"(b.w[1]), "=r"(b.w[2]), "=r"(b.w[3]), "=r"(b.w[4]), "=r"(b.w[5]), "=r"(b.w[6]), "=r"(b.w[7]) : "l"(p));
    memcpy(&x, &b, 32);
  } else {
    x = *reinterpret_cast<const Pack<T, V> *>(p);
  }
  return x;
}
template <typename T, int V> __device__ __forceinline__ void store_pack(T *p, const Pack<T, V> &x) {
  if constexpr (sizeof(T) * V == 16) {
    Bytes16 b;
    memcpy(&b, &x, 16);
    st16(p, b);
  } else if constexpr (sizeof(T) * V == 32) {
    Bytes32 b;
    memcpy(&b, &x, 32);
    st32(p, b);
  } else {
    *reinterpret_cast<Pack<T, V> *>(p) = x;
  }
}

// Asynchronous copy of a 16-byte vector into shared memory.
template <typename T, int V> __device__ __forceinline__ void copy_async(void *shared, const T *p) {
  static_assert(sizeof(T) * V == 16, "a vector");
  const uint32_t s = (uint32_t)__cvta_generic_to_shared(shared);
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(s), "l"(p) : "memory");
}

// An accumulator rounded once to the element type.
template <typename T> __device__ __forceinline__ T round_from(typename TypeTraits<T>::Acc v) { return (T)v; }
template <> __device__ __forceinline__ __half round_from<__half>(float v) { return __float2half_rn(v); }

struct MatView {
  char *data;
  int dtype;
  int64_t rows, cols, row_stride, col_stride;
};

inline bool floating(int dtype) { return dtype == THCB200_F16 || dtype == THCB200_F32 || dtype == THCB200_F64; }

inline int to_mat_view(const thcb200_tensor *t, MatView *m, const char *what) {
  HostView v;
  const int rc = to_host_view(t, &v, what);
  if (rc) return rc;
  if (v.ndim != 2) { set_error("%s: expected a matrix", what); return THCB200_ERR_ARG; }
  m->data = v.data;
  m->dtype = v.dtype;
  m->rows = v.sizes[0];
  m->cols = v.sizes[1];
  m->row_stride = v.strides[0];
  m->col_stride = v.strides[1];
  return 0;
}

// Rows made of whole vectors of `bytes`, each on its own boundary.
inline bool mat_vec(const MatView &m, size_t esz, size_t bytes) {
  return m.col_stride == 1 && (size_t)m.cols * esz % bytes == 0 && (m.rows <= 1 || (uint64_t)m.row_stride * esz % bytes == 0) &&
         (uintptr_t)m.data % bytes == 0;
}

// A matrix that can be written row by row: dense rows, none on top of another.
inline bool dense_rows(const MatView &m) {
  return (m.col_stride == 1 || m.cols <= 1) && (m.rows <= 1 || m.row_stride >= m.cols);
}

// The context's count of positions out of range (thcb200_take_index_errors reads it).
inline unsigned int *index_errors(thcb200_ctx *ctx) { return reinterpret_cast<unsigned int *>(ctx->status) + 1; }

// Scratch of one call: the context's workspace for rows, or, while the stream is being captured into a graph, an allocation that
// becomes part of that graph: a graph that outlives the call must not hold the address of a buffer that later calls share
// and may replace.  The caller holds the context's lock.
struct Workspace {
  char *data;
  bool ok;
  Workspace(thcb200_ctx *ctx, size_t bytes, cudaStream_t st) : data(nullptr), ok(true), owned_(nullptr), st_(st) {
    if (bytes == 0) return;
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(st, &status) != cudaSuccess) {
      set_error("workspace: the stream's capture status is unknown: %s", cudaGetErrorString(cudaGetLastError()));
      ok = false;
      return;
    }
    if (status == cudaStreamCaptureStatusNone) {
      data = (char *)ctx_rows_workspace(ctx, bytes);
    } else if (device_alloc_async(&owned_, bytes, st) == cudaSuccess) {
      data = (char *)owned_;
    } else {
      cudaGetLastError();
      set_error("workspace: cannot allocate %zu bytes in the captured stream", bytes);
    }
    ok = data != nullptr;
  }
  ~Workspace() { if (owned_) cudaFreeAsync(owned_, st_); }
  Workspace(const Workspace &) = delete;
  Workspace &operator=(const Workspace &) = delete;

 private:
  void *owned_;
  cudaStream_t st_;
};

}  // namespace thcb
