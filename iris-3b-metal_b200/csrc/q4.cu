// Small-M linear over 4-bit weights (the form of iris_gemv with fewer bits):
// w[n, k] = scale[n, k / G] (q[n, k] - zero[n, k / G]), zero 8 where none is given;
// out[m, n] = act_out(sum_k act_in(x[m, k]) w[n, k] + bias[n]).
#include "common.cuh"
#include "iris_abi_internal.h"

namespace iris {
namespace q4 {

constexpr int THREADS = 256;
constexpr int ROWS = 16;  // rows of x per pass over the weights

IRIS_DEVICE float silu(float v) { return v / (1.f + __expf(-v)); }

__global__ void __launch_bounds__(THREADS) gemv_q4_kernel(const void* __restrict__ x, int x_dtype, int M, int K,
                                                          int64_t ldx, const uint8_t* __restrict__ packed,
                                                          const __nv_bfloat16* __restrict__ scale,
                                                          const uint8_t* __restrict__ zero, int group,
                                                          const float* __restrict__ bias, void* __restrict__ out,
                                                          int out_dtype, int N, int silu_in, int silu_out) {
  const int lane = threadIdx.x & 31;
  const int n = blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
  if (n >= N) return;
  const int groups = K / group;
  for (int m0 = 0; m0 < M; m0 += ROWS) {
    float acc[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) acc[j] = 0.f;
    for (int k = lane * 8; k < K; k += 256) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(packed + (static_cast<int64_t>(n) * K + k) / 2);
      const int64_t g = static_cast<int64_t>(n) * groups + k / group;
      const float s = __bfloat162float(scale[g]);
      const float z = zero ? static_cast<float>(zero[g]) : 8.f;
#pragma unroll
      for (int j = 0; j < ROWS; ++j) {
        if (m0 + j < M) {
          float part = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float v = load_elem(x, (m0 + j) * ldx + k + e, x_dtype);
            if (silu_in) v = silu(v);
            part += v * (static_cast<float>((w >> (4 * e)) & 15u) - z);
          }
          acc[j] += s * part;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      if (m0 + j < M) {
        const float sum = warp_sum(acc[j]) + (bias ? bias[n] : 0.f);
        if (lane == 0) store_elem(out, static_cast<int64_t>(m0 + j) * N + n, out_dtype, silu_out ? silu(sum) : sum);
      }
    }
  }
}

}  // namespace q4
}  // namespace iris

using namespace iris;

extern "C" int iris_gemv_q4(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, const void* packed,
                            const void* scale, const void* zero, int64_t group, const float* bias, void* out,
                            int out_dtype, int64_t N, int silu_in, int silu_out, void* stream) {
  using namespace iris::q4;
  IRIS_REQUIRE(x && packed && scale && out, "gemv_q4: null pointer");
  IRIS_REQUIRE(group == 32 || group == 64 || group == 128, "gemv_q4: groups of 32, 64 or 128 weights");
  IRIS_REQUIRE(M > 0 && M <= 64 && N > 0 && K > 0 && K % group == 0, "gemv_q4: 1 to 64 rows; K must be a multiple of the group");
  IRIS_REQUIRE(N < (1ll << 31) && K < (1ll << 28) && ldx >= K, "gemv_q4: size");
  IRIS_REQUIRE(x_dtype >= IRIS_F32 && x_dtype <= IRIS_F16 && out_dtype >= IRIS_F32 && out_dtype <= IRIS_F16, "gemv_q4: bad dtype");
  IRIS_REQUIRE(aligned16(x) && aligned16(packed) && aligned_n(scale, 2) && ldx % 8 == 0,
               "gemv_q4: x rows and weights must be 16-byte aligned");
  const int64_t blocks = (N + THREADS / 32 - 1) / (THREADS / 32);
  gemv_q4_kernel<<<static_cast<unsigned>(blocks), THREADS, 0, static_cast<cudaStream_t>(stream)>>>(
      x, x_dtype, static_cast<int>(M), static_cast<int>(K), ldx, static_cast<const uint8_t*>(packed),
      static_cast<const __nv_bfloat16*>(scale), static_cast<const uint8_t*>(zero), static_cast<int>(group), bias, out,
      out_dtype, static_cast<int>(N), silu_in, silu_out);
  IRIS_CUDA(cudaGetLastError());
  return IRIS_OK;
}
