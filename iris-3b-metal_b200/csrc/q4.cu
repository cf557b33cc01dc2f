// Small-M linear over 4-bit weights (the form of iris_gemv with fewer bits):
// w[n, k] = scale[n, k / G] (q[n, k] - zero[n, k / G]), zero 8 where none is given;
// out[m, n] = act_out(sum_k act_in(x[m, k]) w[n, k] + bias[n]).
//
// HBM-bound on N K / 2 bytes of weights, as long as few instructions are spent per
// weight: the products run on mma.sync m16n8k16 with the weights as the 16-row
// operand and x's rows as its 8 columns, so that a weight costs its unpacking alone
// (and / or, subtract, half an instruction each) whatever M is.
//  - q - zero is exact in the operand type: q is put into the mantissa of 128 (bf16)
//    or 1024 (f16) and 128 + zero or 1024 + zero subtracted. Scales are applied in
//    fp32 to each group's fp32 sum, so weights are never rounded.
//  - a 32-bit word holds 8 neighbouring k; one mask takes nibbles i and i + 4. The sum
//    over k has no order, so x is laid out in shared memory in the order in which the
//    words come apart, one 16-byte vector per lane and word; the four lanes of a
//    weight row split a group's words, so that every product of an mma has one scale.
//  - x in 16 bits goes in as it is. FP32 (and act_in's results) go in as three bf16
//    columns, 8 bits each of the 24, cut off rather than rounded: their sum is x, and
//    the columns are free up to 8 of them.
// A CTA owns 32 weight rows and, in a cluster, one part of K; its warps take 128-wide
// pieces of K in turn, each through its own ring of cp.async copies, which is filled
// before x is laid out. Sums are joined in shared memory (over the cluster's CTAs
// through distributed shared memory) in a fixed order.
#include "common.cuh"
#include "iris_abi_internal.h"

namespace iris {
namespace q4 {

constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int STAGES = 4;
constexpr int TILES = 2, ROWS = 16 * TILES;  // weight rows of a CTA
constexpr int STEP = 128;                    // k of one ring slot: 64 bytes of each row
constexpr int SLOT = ROWS * STEP / 2;        // bytes
constexpr int ROUND = STEP * WARPS;          // k of one round of the warps

struct Params {
  const void* x;
  int x_dtype;
  int M, K;
  int64_t ldx;
  const uint8_t* packed;
  const __nv_bfloat16* scale;
  const uint8_t* zero;
  const float* bias;
  void* out;
  int out_dtype;
  int N;
  int silu_in, silu_out;
  int parts;     // CTAs of a cluster: parts of K
  int part_k;    // k of a part, a multiple of ROUND
  int chunk_k;   // k of x in shared memory at a time, a multiple of ROUND
  int pass_rows;  // rows of x per blockIdx.y
};

IRIS_DEVICE float silu(float v) { return v / (1.f + __expf(-v)); }

template <typename T>
struct Magic;
template <>
struct Magic<__nv_bfloat16> {
  static constexpr uint32_t kOne = 0x43004300u;  // 128, 128
  IRIS_DEVICE static uint32_t sub(uint32_t a, uint32_t b) {
    __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<uint32_t*>(&r);
  }
  IRIS_DEVICE static void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct Magic<__half> {
  static constexpr uint32_t kOne = 0x64006400u;  // 1024, 1024
  IRIS_DEVICE static uint32_t sub(uint32_t a, uint32_t b) {
    __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<uint32_t*>(&r);
  }
  IRIS_DEVICE static void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// x as three bf16 values whose sum it is: the top 8 bits of its mantissa, the next 8,
// the rest. Infinities and NaN go into the first alone.
IRIS_DEVICE void split3(float v, uint16_t (&t)[3]) {
  const bool finite = isfinite(v);
  const uint32_t top = __float_as_uint(v) & 0xffff0000u;
  t[0] = isnan(v) ? 0x7fc0u : static_cast<uint16_t>(top >> 16);
  const float rest = finite ? v - __uint_as_float(top) : 0.f;
  const uint32_t mid = __float_as_uint(rest) & 0xffff0000u;
  t[1] = static_cast<uint16_t>(mid >> 16);
  t[2] = static_cast<uint16_t>(__float_as_uint(rest - __uint_as_float(mid)) >> 16);
}

// Where 16-byte piece `piece` of row `row` lies in a slot's 64-byte row: rows two apart
// take turned pieces, so that 4-, 8- and 16-byte reads of 8 rows meet no bank twice.
IRIS_DEVICE int swizzle(int row, int piece) { return piece ^ ((row >> 2 & 1) | (row & 2)); }

// COLS8: groups of 8 columns of the mma (rows of x times TERMS); G: weights per scale.
template <typename T, int TERMS, int COLS8, int G>
__global__ void __launch_bounds__(THREADS) gemv_q4_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, quad = lane & 3;
  const int n0 = static_cast<int>(blockIdx.x / p.parts) * ROWS;
  const int part = static_cast<int>(blockIdx.x % p.parts);
  const int m0 = static_cast<int>(blockIdx.y) * p.pass_rows;
  const int rows = min(p.pass_rows, p.M - m0), cols = rows * TERMS;
  const int k0 = part * p.part_k, k1 = min(k0 + p.part_k, p.K);
  const int groups = p.K / G;
  const int rounds = k1 > k0 ? (k1 - k0 + ROUND - 1) / ROUND : 0;
  constexpr int PER = STEP / G;  // groups per step
  constexpr int WORDS = G / 32;  // words of a group per lane of a row

  const uint32_t ring = smem_addr(smem_raw) + warp * (STAGES * SLOT);
  uint8_t* ring_ptr = smem_raw + warp * (STAGES * SLOT);
  uint8_t* xs = smem_raw + WARPS * STAGES * SLOT;  // [chunk_k / 32][cols][32] in the order of use

  // this lane's share of a step's scales and zeros: group `quad` of rows g, g + 8, g + 16, g + 24
  uint32_t sz[STAGES][2 * TILES];
  auto load = [&](int t, int u) {  // round t into slot u
    const int k = k0 + t * ROUND + warp * STEP;
    if (t < rounds && k < k1) {
#pragma unroll
      for (int e = 0; e < ROWS * 4 / 32; ++e) {
        const int row = e * 8 + g, n = n0 + row;
        const bool real = n < p.N && k + quad * 32 < p.K;
        const uint8_t* src = p.packed + (real ? (static_cast<int64_t>(n) * p.K + k) / 2 + quad * 16 : 0);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ring + u * SLOT + row * 64 +
                                                                           swizzle(row, quad) * 16),
                     "l"(src), "r"(real ? 16 : 0)
                     : "memory");
      }
#pragma unroll
      for (int r = 0; r < 2 * TILES; ++r) {
        const int n = n0 + g + 8 * r, grp = k / G + quad;
        uint32_t v = 0;
        if (quad < PER && n < p.N && grp < groups) {
          const int64_t at = static_cast<int64_t>(n) * groups + grp;
          v = static_cast<uint32_t>(__bfloat16_as_ushort(__ldg(p.scale + at))) << 16;
          v |= p.zero ? __ldg(p.zero + at) : 8u;
        }
        sz[u][r] = v;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int u = 0; u < STAGES; ++u) load(u, u);

  // x for k in [from, from + chunk_k) of this part: zeros behind K
  auto lay_out = [&](int from) {
    const int words = min(p.chunk_k, (k1 - from + ROUND - 1) / ROUND * ROUND) / 8;  // 8 k each
    for (int e = threadIdx.x; e < words * rows; e += THREADS) {
      const int m = e / words, w = e - m * words;
      const int k = from + w * 8;
      float v[8];
      if (k < p.K) {
        const int64_t at = static_cast<int64_t>(m0 + m) * p.ldx + k;
        if (p.x_dtype == IRIS_F32) {
          const float4 a = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.x) + at));
          const float4 b = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.x) + at) + 1);
          v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
          const uint4 a = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.x) + at));
          const uint32_t h[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = p.x_dtype == IRIS_BF16 ? unpack_bf16x2(h[i])
                                                    : __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
          }
        }
        if (p.silu_in) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = silu(v[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
      }
      // word w is word j of lane q's share of its group
      const int grp = w / (G / 8), in = w % (G / 8), q = in / WORDS, j = in % WORDS;
      uint16_t h[TERMS][8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (TERMS == 3) {
          uint16_t t[3];
          split3(v[i], t);
          h[0][i] = t[0], h[1][i] = t[1], h[2][i] = t[2];
        } else {
          h[0][i] = sizeof(T) == 2 && Magic<T>::kOne == Magic<__half>::kOne ? __half_as_ushort(__float2half_rn(v[i]))
                                                                            : __bfloat16_as_ushort(__float2bfloat16_rn(v[i]));
        }
      }
#pragma unroll
      for (int t = 0; t < TERMS; ++t) {
        uint32_t* dst = reinterpret_cast<uint32_t*>(xs + ((grp * WORDS + j) * cols + m * TERMS + t) * 64 + q * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) dst[i] = h[t][i] | static_cast<uint32_t>(h[t][i + 4]) << 16;
      }
    }
  };

  float total[TILES][COLS8][4];
#pragma unroll
  for (int r = 0; r < TILES; ++r)
#pragma unroll
    for (int c = 0; c < COLS8; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) total[r][c][e] = 0.f;

  const int chunk_rounds = p.chunk_k / ROUND;
  int chunk_t = 0;  // round within the chunk
  for (int t0 = 0; t0 < rounds; t0 += STAGES) {
#pragma unroll
    for (int u = 0; u < STAGES; ++u) {
      const int t = t0 + u;
      if (t < rounds) {  // uniform over the CTA
        if (chunk_t == 0) {
          if (t > 0) __syncthreads();  // the chunk before is read
          lay_out(k0 + t * ROUND);
          __syncthreads();
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        __syncwarp();
        const int k = k0 + t * ROUND + warp * STEP;
        if (k < k1) {
          const uint8_t* slot = ring_ptr + u * SLOT;
          const uint8_t* xk = xs + (chunk_t * WARPS + warp) * 4 * cols * 64 + g * 64 + quad * 16;
#pragma unroll
          for (int grp = 0; grp < PER; ++grp) {
            float acc[TILES][COLS8][4];
#pragma unroll
            for (int r = 0; r < TILES; ++r)
#pragma unroll
              for (int c = 0; c < COLS8; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[r][c][e] = 0.f;
            uint32_t meta[2 * TILES], less[2 * TILES], w[2 * TILES][WORDS];
#pragma unroll
            for (int r = 0; r < 2 * TILES; ++r) {
              meta[r] = __shfl_sync(0xffffffffu, sz[u][r], (lane & ~3) + grp);
              less[r] = (meta[r] & 0xffu) * 0x00010001u | Magic<T>::kOne;
              const int row = g + 8 * r;
              const int byte = grp * (G / 2) + quad * (G / 8);  // of the row's 64
              const uint8_t* src = slot + row * 64 + swizzle(row, byte >> 4) * 16 + (byte & 15);
              if constexpr (WORDS == 4) {
                const uint4 v = *reinterpret_cast<const uint4*>(src);
                w[r][0] = v.x, w[r][1] = v.y, w[r][2] = v.z, w[r][3] = v.w;
              } else if constexpr (WORDS == 2) {
                const uint2 v = *reinterpret_cast<const uint2*>(src);
                w[r][0] = v.x, w[r][1] = v.y;
              } else {
                w[r][0] = *reinterpret_cast<const uint32_t*>(src);
              }
            }
#pragma unroll
            for (int j = 0; j < WORDS; ++j) {
              uint4 xb[COLS8];
#pragma unroll
              for (int c = 0; c < COLS8; ++c)
                xb[c] = c * 8 + g < cols ? *reinterpret_cast<const uint4*>(xk + (grp * WORDS + j) * cols * 64 + c * 512)
                                         : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
              for (int s = 0; s < 2; ++s) {  // nibbles 0, 4 and 1, 5, then 2, 6 and 3, 7
#pragma unroll
                for (int r = 0; r < TILES; ++r) {
                  uint32_t a[4];
#pragma unroll
                  for (int h = 0; h < 4; ++h) {  // rows g, g + 8; then the second pair of nibbles
                    const int row = 2 * r + (h & 1);
                    const uint32_t v = w[row][j] >> (8 * s + 4 * (h >> 1));
                    a[h] = Magic<T>::sub((v & 0x000f000fu) | Magic<T>::kOne, less[row]);
                  }
#pragma unroll
                  for (int c = 0; c < COLS8; ++c)
                    Magic<T>::mma(acc[r][c], a, s == 0 ? xb[c].x : xb[c].z, s == 0 ? xb[c].y : xb[c].w);
                }
              }
            }
#pragma unroll
            for (int r = 0; r < TILES; ++r) {
              const float s0 = __uint_as_float(meta[2 * r] & 0xffff0000u), s1 = __uint_as_float(meta[2 * r + 1] & 0xffff0000u);
#pragma unroll
              for (int c = 0; c < COLS8; ++c) {
                total[r][c][0] = fmaf(s0, acc[r][c][0], total[r][c][0]);
                total[r][c][1] = fmaf(s0, acc[r][c][1], total[r][c][1]);
                total[r][c][2] = fmaf(s1, acc[r][c][2], total[r][c][2]);
                total[r][c][3] = fmaf(s1, acc[r][c][3], total[r][c][3]);
              }
            }
          }
        }
        __syncwarp();  // the slot is read
        load(t + STAGES, u);
        if (++chunk_t == chunk_rounds) chunk_t = 0;
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();  // rings and x are done with
  // [warp][row][COLS8 * 8] sums; then one thread per (row of x, weight row)
  float* sums = reinterpret_cast<float*>(smem_raw);
  constexpr int WIDTH = COLS8 * 8;
#pragma unroll
  for (int r = 0; r < TILES; ++r)
#pragma unroll
    for (int c = 0; c < COLS8; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<float2*>(sums + (warp * ROWS + 16 * r + 8 * h + g) * WIDTH + c * 8 + 2 * quad) =
            make_float2(total[r][c][2 * h], total[r][c][2 * h + 1]);
  if (p.parts > 1) cluster_sync();
  else __syncthreads();
  if (part == 0) {
    for (int e = threadIdx.x; e < rows * ROWS; e += THREADS) {
      const int m = e / ROWS, row = e % ROWS;
      float v = 0.f;
      for (int q = 0; q < p.parts; ++q) {
        const uint32_t base = p.parts > 1 ? map_to_cta(sums, static_cast<uint32_t>(q)) : smem_addr(sums);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          float x[TERMS];
#pragma unroll
          for (int t = 0; t < TERMS; ++t)
            asm volatile("ld.shared::cluster.f32 %0, [%1];"
                         : "=f"(x[t])
                         : "r"(base + 4 * ((w * ROWS + row) * WIDTH + m * TERMS + t))
                         : "memory");
#pragma unroll
          for (int t = TERMS - 1; t >= 0; --t) v += x[t];
        }
      }
      const int n = n0 + row;
      if (n < p.N) {
        if (p.bias) v += __ldg(p.bias + n);
        store_elem(p.out, static_cast<int64_t>(m0 + m) * p.N + n, p.out_dtype, p.silu_out ? silu(v) : v);
      }
    }
  }
  if (p.parts > 1) cluster_sync();  // no CTA leaves while its sums are read
}

constexpr int X_BYTES = 64 * 1024;  // x in shared memory at a time, at most

template <typename T, int TERMS, int COLS8, int G>
int launch_g(Params& p, int passes, cudaStream_t st) {
  auto kernel = gemv_q4_kernel<T, TERMS, COLS8, G>;
  const int cols = p.pass_rows * TERMS;
  const int64_t tiles = (p.N + ROWS - 1) / ROWS;
  // parts of K over a cluster's CTAs: as many as give every SM two CTAs, or as keep a part of x in shared memory
  int parts = 1;
  const int64_t wanted = 2 * num_sms();
  while (parts < 8 && p.K > 2 * parts * ROUND &&
         (tiles * passes * parts < wanted || static_cast<int64_t>(p.K) * cols * 2 / parts > X_BYTES))
    parts *= 2;
  p.parts = parts;
  p.part_k = ((p.K + parts - 1) / parts + ROUND - 1) / ROUND * ROUND;
  const int most = X_BYTES / (cols * 2) / ROUND * ROUND;
  p.chunk_k = p.part_k < most ? p.part_k : most;
  const int used = WARPS * STAGES * SLOT + p.chunk_k * cols * 2;
  const int sums = WARPS * ROWS * COLS8 * 8 * 4;
  const int smem = used > sums ? used : sums;
  static int configured[64] = {0};
  int dev = 0;
  IRIS_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || configured[dev] == 0) {
    IRIS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, WARPS * STAGES * SLOT + X_BYTES));
    if (dev < 64) configured[dev] = 1;
  }
  cudaLaunchAttribute cluster = {};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = static_cast<unsigned>(parts);
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(tiles * parts), static_cast<unsigned>(passes));
  config.blockDim = dim3(THREADS);
  config.dynamicSmemBytes = static_cast<size_t>(smem);
  config.stream = st;
  config.attrs = &cluster;
  config.numAttrs = 1;
  IRIS_CUDA(cudaLaunchKernelEx(&config, kernel, p));
  return IRIS_OK;
}

template <typename T, int TERMS, int COLS8>
int launch(Params& p, int64_t group, cudaStream_t st) {
  const int most = COLS8 * 8 / TERMS;
  const int passes = (p.M + most - 1) / most;
  p.pass_rows = (p.M + passes - 1) / passes;
  if (group == 32) return launch_g<T, TERMS, COLS8, 32>(p, passes, st);
  if (group == 64) return launch_g<T, TERMS, COLS8, 64>(p, passes, st);
  return launch_g<T, TERMS, COLS8, 128>(p, passes, st);
}

// Columns for the rows at hand: one mma per weight operand up to 8 of them, more
// mmas on the same unpacked weights above.
template <typename T>
int launch_rows(Params& p, int64_t group, cudaStream_t st) {
  if (p.M <= 8) return launch<T, 1, 1>(p, group, st);
  if (p.M <= 16) return launch<T, 1, 2>(p, group, st);
  return launch<T, 1, 4>(p, group, st);
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
  IRIS_REQUIRE(N < (1ll << 28) && K < (1ll << 28) && ldx >= K, "gemv_q4: size");
  IRIS_REQUIRE(x_dtype >= IRIS_F32 && x_dtype <= IRIS_F16 && out_dtype >= IRIS_F32 && out_dtype <= IRIS_F16, "gemv_q4: bad dtype");
  IRIS_REQUIRE(aligned16(x) && aligned16(packed) && aligned_n(scale, 2) && ldx % 8 == 0,
               "gemv_q4: x rows and weights must be 16-byte aligned");
  Params p = {};
  p.x = x, p.x_dtype = x_dtype, p.M = static_cast<int>(M), p.K = static_cast<int>(K), p.ldx = ldx;
  p.packed = static_cast<const uint8_t*>(packed), p.scale = static_cast<const __nv_bfloat16*>(scale);
  p.zero = static_cast<const uint8_t*>(zero), p.bias = bias, p.out = out, p.out_dtype = out_dtype;
  p.N = static_cast<int>(N), p.silu_in = silu_in, p.silu_out = silu_out;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (x_dtype == IRIS_F32 || silu_in) {  // fp32 values: three columns a row
    if (M <= 2) return launch<__nv_bfloat16, 3, 1>(p, group, st);
    if (M <= 5) return launch<__nv_bfloat16, 3, 2>(p, group, st);
    if (M <= 8) return launch<__nv_bfloat16, 3, 3>(p, group, st);
    return launch<__nv_bfloat16, 3, 6>(p, group, st);
  }
  if (x_dtype == IRIS_F16) return launch_rows<__half>(p, group, st);
  return launch_rows<__nv_bfloat16>(p, group, st);
}
