// Host-side helpers shared by the C-ABI entry points: error reporting,
// argument checks, device queries and TMA descriptor creation.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/iris_b200.h"

namespace iris {

// Records the message returned by iris_last_error() (thread-local).
int set_error(int code, const char* fmt, ...);

int num_sms();

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// Rows whose strides can all be used: that of a dimension with one entry says nothing and becomes 0.
inline iris_head_rows used_strides(iris_head_rows r, int64_t batch, int64_t heads, int64_t tokens) {
  if (batch <= 1) r.stride_b = 0;
  if (heads <= 1) r.stride_h = 0;
  if (tokens <= 1) r.stride_n = 0;
  return r;
}

inline bool aligned_n(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; }

// 2-D bf16 tensor map (inner dim first) with 128-byte swizzle and the given box.
int make_tmap_2d_bf16(CUtensorMap* map, const void* base, int64_t inner, int64_t outer, int64_t row_stride_elems,
                      int box_inner, int box_outer);

// 3-D bf16 tensor map (inner, mid, outer) with 128-byte swizzle.
int make_tmap_3d_bf16(CUtensorMap* map, const void* base, int64_t d0, int64_t d1, int64_t d2, int64_t stride1_elems,
                      int64_t stride2_elems, int box0, int box1, int box2);

// 2-D map of bytes with 128-byte swizzle (row_bytes a multiple of 16).
int make_tmap_2d_bytes(CUtensorMap* map, const void* base, int64_t inner, int64_t outer, int64_t row_bytes,
                       int box_inner, int box_outer);

// 4-D map (head columns, tokens, heads, batch) of 2-byte elements (dtype
// IRIS_BF16 or IRIS_F16) with 128-byte swizzle and boxes of 64 columns x box_rows
// tokens; element strides. A stride of 0 (heads, batch) maps one entry: its
// coordinate must be 0.
int make_tmap_heads(CUtensorMap* map, const void* base, int dtype, int64_t head_dim, int64_t tokens, int64_t heads,
                    int64_t batch, int64_t stride_n, int64_t stride_h, int64_t stride_b, int box_rows);

// Launch a kernel that may start before its predecessor in the stream has ended (it
// begins with grid_wait, common.cuh); cluster: CTAs per cluster along x.
template <typename... Params, typename... Args>
cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, unsigned threads, size_t smem, cudaStream_t stream,
                         unsigned cluster, const Args&... args) {
  cudaLaunchAttribute attrs[2] = {};
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = cluster;
  attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = attrs;
  config.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&config, kernel, args...);
}

}  // namespace iris

#define IRIS_REQUIRE(cond, msg)                           \
  do {                                                    \
    if (!(cond)) return ::iris::set_error(IRIS_EINVAL, "%s", msg); \
  } while (0)

#define IRIS_CUDA(expr)                                                                                   \
  do {                                                                                                    \
    cudaError_t _e = (expr);                                                                              \
    if (_e != cudaSuccess) return ::iris::set_error(IRIS_ECUDA, "%s: %s", #expr, cudaGetErrorString(_e)); \
  } while (0)

#define IRIS_CHECK_STATUS(expr)   \
  do {                            \
    int _s = (expr);              \
    if (_s != IRIS_OK) return _s; \
  } while (0)
