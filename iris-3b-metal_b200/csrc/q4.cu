// Small-M linear over 4-bit weights (the form of iris_gemv with fewer bits):
// w[n, k] = scale[n, k / G] (q[n, k] - zero[n, k / G]), zero 8 where none is given;
// out[m, n] = act_out(sum_k act_in(x[m, k]) w[n, k] + bias[n]).
//
// HBM-bound on N K / 2 bytes of weights, as long as few instructions are spent per
// weight: the products run on mma.sync m16n8k16 with the weights as the 16-row
// operand and x's rows as its 8 columns, so that a weight costs its unpacking alone
// (and / or, subtract, half an instruction each), once for up to 32 rows of 16 bits or 16
// of fp32. More rows are passes of those, and each reads and unpacks every weight again.
//  - q - zero is exact in the operand type: q is put into the mantissa of 128 (bf16)
//    or 1024 (f16) and 128 + zero or 1024 + zero subtracted. Scales are applied in
//    fp32 to each group's fp32 sum, so weights are never rounded.
//  - a 32-bit word holds 8 neighbouring k; one mask takes nibbles i and i + 4. The sum
//    over k has no order, so x is laid out in shared memory in the order in which the
//    words come apart, one 16-byte vector per lane and word; the four lanes of a
//    weight row split a group's words, so that every product of an mma has one scale.
//  - x in 16 bits goes in as it is. FP32 (and act_in's results) go in as three bf16
//    columns, 8 bits each of the 24, cut off rather than rounded: their sum is x, and
//    the columns are free up to 8 of them. (To 2^-133, bf16's last bit: rows that lie
//    below 1e-33 throughout keep fewer than 24 bits.)
// A CTA owns 128 weight rows, 32 a warp, and, in a cluster, one part of K, whose x it
// lays out once for all of them; a warp streams 256-wide pieces of its rows through
// its own ring of TMA copies (one instruction for 32 rows; filled before x is laid
// out). Each part's sums are stored into the shared memory of the CTA that owns the
// row (no CTA waits on another's memory: reading the sums from there instead took 2 to
// 4 us of a call's 12 to 21), which adds them in a fixed order.
//
// Measured: 8192 -> 32768, groups of 128, one bf16 row 41 us (3.4 TB/s, 0.52 of a plain
// copy), 8 rows 61, 16 rows 87, 32 rows 139, 64 rows (two passes) 278. The unpacking (7 and / shift operations a word at half rate, 3 more per mma)
// alone takes about 19 us, the copies alone 25, the start (launch, cluster, first
// copies, x) 5; they overlap in part. 2560 -> 15360, groups of 64, one fp32 row 12.7 us
// (1.7 TB/s), 8 rows 21, 16 rows 42, 64 rows (four passes) 149; 6848 -> 2561, groups of
// 32 with zeros, 16 f16 rows 16.1 us: an SM has four warps or eight, each a chain of shared memory -> unpacking -> mma -> scale. Deeper rings,
// scales prefetched into L2, two accumulators a sum: no gain; eight warps of 16 rows in place
// of four 15.0 us there, but 7.6 instead of 6.8 for 2560 -> 2560, one row; three CTAs an
// SM for one row instead of four 47.7 us; twice the parts 43.9 us, 18.5 the 2560 -> 15360.
#include <algorithm>

#include "common.cuh"
#include "iris_abi_internal.h"

namespace iris {
namespace q4 {

constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int MOST_STAGES = 4;               // ring slots of a warp: two to four (see launch_g)
constexpr int TILES = 2, ROWS = 16 * TILES;  // weight rows of a warp
constexpr int STEP = 256;                    // k of one ring slot: 128 bytes of each row
constexpr int SLOT = ROWS * STEP / 2;        // bytes
constexpr int MOST_PARTS = 8;                // CTAs of a cluster

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
  int part_k;    // k of a part, a multiple of STEP
  int chunk_k;   // k of x in shared memory at a time, a multiple of STEP
  int pass_rows;  // rows of x per blockIdx.y
  int stages;     // ring slots of a warp
};

// With the fast exponential, as iris_gemv has it: its relative error is |v| 2^-24 for
// negative v, 2^-18 at -64 where silu is -1e-26.
IRIS_DEVICE float silu(float v) { return v / (1.f + __expf(-v)); }

// (v & mask) | bits in one instruction
IRIS_DEVICE uint32_t put(uint32_t v, uint32_t mask, uint32_t bits) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(v), "r"(mask), "r"(bits));
  return d;
}

// Weights of two nibbles as the operand type, and the products. unpack<I>: nibbles I
// and I + 4 of word w, less their zero, as a pair; less(z): what a group's zero is kept as.
template <typename T>
struct Operand;
template <>
struct Operand<__nv_bfloat16> {
  static constexpr uint32_t kOne = 0x43004300u;  // 128: the mantissa's last bit is 1
  using Less = uint32_t;
  IRIS_DEVICE static Less less(uint32_t z) { return __byte_perm(z, 0x43u, 0x4040); }  // z in byte 0
  template <int I>
  IRIS_DEVICE static uint32_t unpack(uint32_t w, Less z) {
    uint32_t a = put(w >> (4 * I), 0x000f000fu, kOne);
    __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&z));
    return *reinterpret_cast<uint32_t*>(&r);
  }
  IRIS_DEVICE static void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  IRIS_DEVICE static void mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  }
};
template <>
struct Operand<__half> {
  static constexpr uint32_t kOne = 0x64006400u;  // 1024
  struct Less {
    uint32_t low, high;  // 1024 + z; -(64 + z)
  };
  IRIS_DEVICE static Less less(uint32_t z) {  // z in byte 0, 16 z in byte 1
    return Less{__byte_perm(z, 0x64u, 0x4040), __byte_perm(z, 0xd4u, 0x4141)};
  }
  template <int I>
  IRIS_DEVICE static uint32_t unpack(uint32_t w, Less z) {
    __half2 r;
    if constexpr (I % 2 == 0) {
      uint32_t a = put(w >> (4 * I), 0x000f000fu, kOne);
      r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&z.low));
    } else {  // four bits up: 1024 + 16 q, a sixteenth of it less 64 + z (both exact), without a shift of its own
      uint32_t a = put(w >> (4 * (I - 1)), 0x00f000f0u, kOne);
      const uint32_t sixteenth = 0x2c002c00u;
      r = __hfma2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<const __half2*>(&sixteenth), *reinterpret_cast<__half2*>(&z.high));
    }
    return *reinterpret_cast<uint32_t*>(&r);
  }
  IRIS_DEVICE static void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  IRIS_DEVICE static void mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  }
};

// x as three bf16 values whose sum it is: the top 8 bits of its mantissa, the next 8,
// the rest. Infinities and NaN go into the first alone.
IRIS_DEVICE void split3(float v, uint32_t (&t)[3]) {
  const bool finite = isfinite(v);
  const uint32_t top = __float_as_uint(v) & 0xffff0000u;
  t[0] = isnan(v) ? 0x7fc0u : top >> 16;
  const float rest = finite ? v - __uint_as_float(top) : 0.f;
  const uint32_t mid = __float_as_uint(rest) & 0xffff0000u;
  t[1] = mid >> 16;
  t[2] = __float_as_uint(rest - __uint_as_float(mid)) >> 16;
}

// One result from the definition, its weights scaled before the sum: for results that are
// not finite, since a group's unscaled sum of x (q - zero) leaves fp32 where a scaled one
// need not (|x| from 2e35 on). By one thread; NaN and infinities in x come here too.
__device__ __noinline__ float sum_scaled(const Params& p, int group, int m, int n) {
  const int groups = p.K / group;
  const uint32_t* words = reinterpret_cast<const uint32_t*>(p.packed + static_cast<int64_t>(n) * (p.K / 2));
  float total = 0.f;
  for (int g = 0; g < groups; ++g) {
    const int64_t at = static_cast<int64_t>(n) * groups + g;
    const uint32_t zero = p.zero ? p.zero[at] : 8u;
    const float s = zero < 16u ? __bfloat162float(p.scale[at]) : __int_as_float(0x7fc00000), z = static_cast<float>(zero);
    float part[8] = {};
    for (int w = g * (group / 8); w < (g + 1) * (group / 8); ++w) {
      const uint32_t q = words[w];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = load_elem(p.x, m * p.ldx + w * 8 + j, p.x_dtype);
        part[j] = fmaf(p.silu_in ? silu(v) : v, s * (static_cast<float>(q >> (4 * j) & 15u) - z), part[j]);
      }
    }
    total += ((part[0] + part[1]) + (part[2] + part[3])) + ((part[4] + part[5]) + (part[6] + part[7]));
    if (isnan(total)) break;
  }
  return total;
}

// The weight row that a lane's row index g of the mma stands for: with the copy's
// 128-byte swizzle (16-byte piece x of row r at x ^ (r % 8)) the 4-, 8- or 16-byte reads
// of lanes that read together then meet no bank twice.
IRIS_DEVICE int weight_row(int g) { return (g & 1) << 2 | (g & 2) | g >> 2; }

// CTAs of an SM: as many as leave the columns' sums in registers.
constexpr int ctas_per_sm(int cols8) { return cols8 == 1 ? 4 : cols8 == 2 ? 3 : 2; }

// COLS8: groups of 8 columns of the mma (rows of x times TERMS); G: weights per scale.
template <typename T, int TERMS, int COLS8, int G>
__global__ void __launch_bounds__(THREADS, ctas_per_sm(COLS8)) gemv_q4_kernel(const __grid_constant__ CUtensorMap tw,
                                                          const __grid_constant__ Params p) {
  extern __shared__ __align__(1024) uint8_t smem_unaligned[];
  __shared__ uint64_t full[WARPS][MOST_STAGES];
  __shared__ int abort_flag;
  uint8_t* smem_raw = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_unaligned) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, quad = lane & 3;
  const int n0 = (static_cast<int>(blockIdx.x / p.parts) * WARPS + warp) * ROWS;  // this warp's first weight row
  const int part = static_cast<int>(blockIdx.x % p.parts);
  const int m0 = static_cast<int>(blockIdx.y) * p.pass_rows;
  const int rows = min(p.pass_rows, p.M - m0), cols = rows * TERMS;
  const int k0 = part * p.part_k, k1 = min(k0 + p.part_k, p.K);
  const int groups = p.K / G;
  const int steps = k1 > k0 ? (k1 - k0 + STEP - 1) / STEP : 0;
  constexpr int PER = STEP / G;                // groups per step
  constexpr int WORDS = G / 32;                // words of a group per lane of a row
  constexpr int HELD = (PER + 3) / 4;          // scales and zeros that a lane holds for each of its rows:
  constexpr int SPAN = PER < 4 ? 4 / PER : 1;  // of so many steps

  uint8_t* ring = smem_raw + warp * (p.stages * SLOT);
  float* sums = reinterpret_cast<float*>(smem_raw + WARPS * p.stages * SLOT);  // other CTAs store here: a place of its own
  uint8_t* xs = smem_raw + WARPS * p.stages * SLOT + WARPS * ROWS * COLS8 * 8 * 4;  // [chunk_k / 32][cols][32] in the order of use
  volatile int* abort = &abort_flag;
  __shared__ __align__(16) uint8_t zeros[16];
  if (threadIdx.x < 4) reinterpret_cast<uint32_t*>(zeros)[threadIdx.x] = 0u;
  if (threadIdx.x == 0) {
    for (int w = 0; w < WARPS; ++w)
      for (int u = 0; u < p.stages; ++u) mbar_init(&full[w][u], 1);
    abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  if (p.parts > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  grid_wait();
  grid_trigger();

  // x for k in [from, from + chunk_k) of this part: zeros behind K. Word w (8 k) of a
  // row is word j of lane q's share of its group. A thread takes BATCH words at once,
  // grabbed (their loads overlap) and then put in place.
  constexpr int BATCH = TERMS == 1 ? 8 : 4;
  uint4 raw[BATCH][TERMS == 1 ? 1 : 2];  // fp32: two pieces a word
  auto grab = [&](int from, int words, int e0) {
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int e = e0 + i * THREADS, m = e / words, k = from + (e - m * words) * 8;
      const bool real = m < rows && k < p.K;
      const int64_t at = static_cast<int64_t>(m0 + m) * p.ldx + k;
#pragma unroll
      for (int h = 0; h < (TERMS == 1 ? 1 : 2); ++h) raw[i][h] = make_uint4(0u, 0u, 0u, 0u);
      if (!real) continue;
      if (TERMS == 1 || p.x_dtype != IRIS_F32) {
        raw[i][0] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.x) + at);
      } else {
#pragma unroll
        for (int h = 0; h < (TERMS == 1 ? 1 : 2); ++h)
          raw[i][h] = reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(p.x) + at)[h];
      }
    }
  };
  auto put = [&](int words, int e0) {
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int e = e0 + i * THREADS, m = e / words, w = e - m * words;
      if (m >= rows) continue;
      const int grp = w / (G / 8), in = w % (G / 8), q = in / WORDS, j = in % WORDS;
      uint8_t* to = xs + ((grp * WORDS + j) * cols + m * TERMS) * 64 + q * 16;
      const uint4 a = raw[i][0];
      if constexpr (TERMS == 1) {  // in 16 bits as it is: only the order changes
        *reinterpret_cast<uint4*>(to) = make_uint4(__byte_perm(a.x, a.z, 0x5410), __byte_perm(a.x, a.z, 0x7632),
                                                   __byte_perm(a.y, a.w, 0x5410), __byte_perm(a.y, a.w, 0x7632));
      } else {
        float v[8];
        if (p.x_dtype == IRIS_F32) {
          const uint4 b = raw[i][TERMS == 1 ? 0 : 1];
          const uint32_t f[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
          for (int h = 0; h < 8; ++h) v[h] = __uint_as_float(f[h]);
        } else {
          const uint32_t f[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const float2 d = p.x_dtype == IRIS_BF16 ? unpack_bf16x2(f[h])
                                                    : __half22float2(*reinterpret_cast<const __half2*>(&f[h]));
            v[2 * h] = d.x, v[2 * h + 1] = d.y;
          }
        }
        uint32_t t[8][3];
#pragma unroll
        for (int h = 0; h < 8; ++h) split3(p.silu_in ? silu(v[h]) : v[h], t[h]);
#pragma unroll
        for (int c = 0; c < 3; ++c)
          *reinterpret_cast<uint4*>(to + c * 64) = make_uint4(t[0][c] | t[4][c] << 16, t[1][c] | t[5][c] << 16,
                                                              t[2][c] | t[6][c] << 16, t[3][c] | t[7][c] << 16);
      }
    }
  };
  auto words_of = [&](int from) { return min(p.chunk_k, (k1 - from + STEP - 1) / STEP * STEP) / 8; };  // of a row
  if (steps > 0) grab(k0, words_of(k0), threadIdx.x);  // ahead of the weights, not behind them in the queue

  auto load = [&](int t, int slot) {  // step t into its slot
    if (lane == 0 && t < steps && n0 < p.N) {
      mbar_arrive_expect_tx(&full[warp][slot], SLOT);
      // rows from N on and k from K on: zeros
      tma_load_2d(&tw, &full[warp][slot], ring + slot * SLOT, (k0 + t * STEP) / 2, n0);
    }
  };
  for (int t = 0; t < p.stages; ++t) load(t, t);

  // lane (g, quad) holds groups quad, quad + 4 of SPAN steps, of rows weight_row(g) + 0, 8, 16, 24, fetched ahead
  const int row_g = weight_row(g);
  uint16_t sz_scale[2 * TILES][HELD];
  uint32_t sz_zero[2 * TILES][HELD];
  const int64_t meta0 = static_cast<int64_t>(n0 + row_g) * groups + k0 / G + quad;
  const uint16_t* scale_at = reinterpret_cast<const uint16_t*>(p.scale) + meta0;
  const uint8_t* zero_at = p.zero ? p.zero + meta0 : nullptr;
  const int real_rows = min(2 * TILES, max(0, (p.N - n0 - row_g + 7) / 8));  // of this lane's that exist
  int grps_left = k1 / G - k0 / G - quad;                                    // groups of this lane's from here on
  auto fetch = [&]() {
#pragma unroll
    for (int r = 0; r < 2 * TILES; ++r) {
#pragma unroll
      for (int h = 0; h < HELD; ++h) {
        uint16_t scale = 0;
        uint32_t zero = 8;
        if (r < real_rows && 4 * h < grps_left && quad + 4 * h < PER * SPAN) {
          // volatile: where they stand, a span ahead of their use
          const int64_t at = static_cast<int64_t>(8 * r) * groups + 4 * h;
          asm volatile("ld.global.u16 %0, [%1];" : "=h"(scale) : "l"(scale_at + at));
          if (zero_at) asm volatile("ld.global.u8 %0, [%1];" : "=r"(zero) : "l"(zero_at + at));
        }
        sz_scale[r][h] = scale;
        sz_zero[r][h] = zero;
      }
    }
    scale_at += SPAN * STEP / G;
    if (zero_at) zero_at += SPAN * STEP / G;
    grps_left -= SPAN * STEP / G;
  };
  fetch();

  float total[TILES][COLS8][4];
#pragma unroll
  for (int r = 0; r < TILES; ++r)
#pragma unroll
    for (int c = 0; c < COLS8; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) total[r][c][e] = 0.f;

  auto lay_out = [&](int from, int first) {
    const int words = words_of(from);
    for (int e0 = first; e0 < words * rows; e0 += BATCH * THREADS) {
      grab(from, words, e0);
      put(words, e0);
    }
  };
  if (steps > 0) {
    put(words_of(k0), threadIdx.x);
    lay_out(k0, threadIdx.x + BATCH * THREADS);
    __syncthreads();
  }
  bool ok = true;
  const int chunk_steps = p.chunk_k / STEP;
  int chunk_t = 0;  // step within the chunk
  int at_slot = 0;  // the step's slot and its phase
  uint32_t phase = 0;
  uint32_t now[2 * TILES][HELD];
  uint32_t zeros_seen = 0;
#pragma unroll 1
  for (int t = 0; t < steps; ++t) {
    if (chunk_t == chunk_steps) {  // uniform over the CTA
      chunk_t = 0;
      __syncthreads();  // the chunk before is read
      lay_out(k0 + t * STEP, threadIdx.x);
      __syncthreads();
    }
    if (t % SPAN == 0) {
#pragma unroll
      for (int r = 0; r < 2 * TILES; ++r)
#pragma unroll
        for (int h = 0; h < HELD; ++h) {  // scale, 16 zero, zero
          now[r][h] = static_cast<uint32_t>(sz_scale[r][h]) << 16 | sz_zero[r][h] * 0x1001u;
          zeros_seen |= sz_zero[r][h];
        }
      fetch();
    }
    if (n0 < p.N && ok) {
      ok = mbar_wait(&full[warp][at_slot], phase, abort);
      const uint8_t* slot = ring + at_slot * SLOT + row_g * 128;
      const int held_by = (lane & ~3) + t % SPAN * PER;  // the lane with the step's first group
      // this lane's column of each 8, or zeros
      const uint8_t* xk[COLS8];
      int xstep[COLS8];
#pragma unroll
      for (int c = 0; c < COLS8; ++c) {
        const bool real = c * 8 + g < cols;
        xk[c] = real ? xs + (chunk_t * (STEP / 32) * cols + c * 8 + g) * 64 + quad * 16 : zeros;
        xstep[c] = real ? cols * 64 : 0;
      }
#pragma unroll
      for (int grp = 0; grp < PER; ++grp) {
        float acc[TILES][COLS8][4];
        uint32_t meta[2 * TILES], w[2 * TILES][WORDS];
        typename Operand<T>::Less less[2 * TILES];
#pragma unroll
        for (int r = 0; r < 2 * TILES; ++r) {
          meta[r] = __shfl_sync(0xffffffffu, now[r][grp / 4], held_by + grp % 4);
          less[r] = Operand<T>::less(meta[r]);
          const int byte = grp * (G / 2) + quad * (G / 8);  // of the row's 128
          const uint8_t* src = slot + r * 1024 + (((byte >> 4) ^ row_g) * 16 | (byte & 15));
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
          for (int c = 0; c < COLS8; ++c) {
            xb[c] = *reinterpret_cast<const uint4*>(xk[c]);
            xk[c] += xstep[c];
          }
#pragma unroll
          for (int half = 0; half < 2; ++half)  // neighbouring mmas add to different sums: none waits for the one before
#pragma unroll
            for (int r = 0; r < TILES; ++r) {
              const uint32_t u0 = w[2 * r][j], u1 = w[2 * r + 1][j];
              const auto z0 = less[2 * r], z1 = less[2 * r + 1];
              uint32_t a[4];
              if (half == 0) {
                a[0] = Operand<T>::template unpack<0>(u0, z0), a[1] = Operand<T>::template unpack<0>(u1, z1);
                a[2] = Operand<T>::template unpack<1>(u0, z0), a[3] = Operand<T>::template unpack<1>(u1, z1);
              } else {
                a[0] = Operand<T>::template unpack<2>(u0, z0), a[1] = Operand<T>::template unpack<2>(u1, z1);
                a[2] = Operand<T>::template unpack<3>(u0, z0), a[3] = Operand<T>::template unpack<3>(u1, z1);
              }
#pragma unroll
              for (int c = 0; c < COLS8; ++c) {
                if (half == 1) Operand<T>::mma(acc[r][c], a, xb[c].z, xb[c].w);
                else if (j == 0) Operand<T>::mma_first(acc[r][c], a, xb[c].x, xb[c].y);
                else Operand<T>::mma(acc[r][c], a, xb[c].x, xb[c].y);
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
    ok = __all_sync(0xffffffffu, ok);  // and the slot is read by every lane
    if (ok) load(t + p.stages, at_slot);
    if (++at_slot == p.stages) at_slot = 0, phase ^= 1u;
    ++chunk_t;
  }
  if (!ok) {  // a wait gave up (device error word): no copy may land after the CTA is gone; NaN rather than wrong sums
    int dummy = 0;
    for (int t = 0; t < steps && n0 < p.N; ++t)
      mbar_wait(&full[warp][t % p.stages], static_cast<uint32_t>((t / p.stages) & 1), &dummy);
#pragma unroll
    for (int r = 0; r < TILES; ++r)
#pragma unroll
      for (int c = 0; c < COLS8; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) total[r][c][e] = __int_as_float(0x7fc00000);
  }
  if (__any_sync(0xffffffffu, zeros_seen > 15u)) {  // a zero point of more than 4 bits: its weight row is NaN
    const int from = k0 / G, groups_here = k1 / G - from;
#pragma unroll
    for (int r = 0; r < 2 * TILES; ++r) {
      bool bad = false;
      for (int i = quad; r < real_rows && i < groups_here; i += 4)
        bad = bad || p.zero[static_cast<int64_t>(n0 + row_g + 8 * r) * groups + from + i] > 15;
      const unsigned row_bad = __ballot_sync(0xffffffffu, bad) >> (lane & ~3) & 0xfu;  // the row's four lanes
      if (row_bad == 0u) continue;
      if (quad == 0) atomicOr(&g_device_error, kErrBadArgument);
#pragma unroll
      for (int c = 0; c < COLS8; ++c) total[r / 2][c][r % 2 * 2] = total[r / 2][c][r % 2 * 2 + 1] = __int_as_float(0x7fc00000);
    }
  }
  if (p.parts > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // the cluster's CTAs have begun
  // sums [part][row][COLS8 * 8] of the rows that a CTA owns, 128 / parts of them
  constexpr int WIDTH = COLS8 * 8, CTA_ROWS = WARPS * ROWS;
  const int owned = CTA_ROWS / p.parts;
#pragma unroll
  for (int r = 0; r < TILES; ++r)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = warp * ROWS + 16 * r + 8 * h + row_g, owner = row / owned;
      float* at = sums + (part * owned + row - owner * owned) * WIDTH + 2 * quad;
      const uint32_t to = p.parts > 1 ? map_to_cta(at, static_cast<uint32_t>(owner)) : 0u;
#pragma unroll
      for (int c = 0; c < COLS8; ++c) {
        const float x = total[r][c][2 * h], y = total[r][c][2 * h + 1];
        if (p.parts > 1)
          asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to + c * 32), "f"(x), "f"(y) : "memory");
        else
          *reinterpret_cast<float2*>(at + c * 8) = make_float2(x, y);
      }
    }
  if (p.parts > 1) cluster_sync();
  else __syncthreads();
  const int first_row = static_cast<int>(blockIdx.x / p.parts) * CTA_ROWS + part * owned;
  for (int e = threadIdx.x; e < owned * rows; e += THREADS) {
    const int m = e / owned, row = e - m * owned, n = first_row + row;
    if (n >= p.N) continue;
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < MOST_PARTS; ++q)
      if (q < p.parts)
#pragma unroll
        for (int c = TERMS - 1; c >= 0; --c) v += sums[(q * owned + row) * WIDTH + m * TERMS + c];
    if (!isfinite(v)) v = sum_scaled(p, G, m0 + m, n);
    if (p.bias) v += p.bias[n];
    store_elem(p.out, static_cast<int64_t>(m0 + m) * p.N + n, p.out_dtype, p.silu_out ? silu(v) : v);
  }
}

constexpr int SM_BYTES = 228 * 1024, CTA_BYTES = 2048 + 512;  // shared memory of an SM; of a CTA beside its rings and x
constexpr int X_BYTES = 48 * 1024;  // x in shared memory at a time, at most
static_assert(X_BYTES / (48 * 2) >= STEP, "a step of x in 48 columns, the most that a pass has");

template <typename T, int TERMS, int COLS8, int G>
int launch_g(Params& p, int passes, cudaStream_t st) {
  auto kernel = gemv_q4_kernel<T, TERMS, COLS8, G>;
  const int cols = p.pass_rows * TERMS;
  const int64_t tiles = (p.N + WARPS * ROWS - 1) / (WARPS * ROWS);
  // parts of K over a cluster's CTAs: as many as still run at once
  int parts = 1;
  while (parts < MOST_PARTS && p.K > parts * STEP && tiles * passes * parts * 2 <= ctas_per_sm(COLS8) * num_sms()) parts *= 2;
  p.parts = parts;
  p.part_k = ((p.K + parts - 1) / parts + STEP - 1) / STEP * STEP;
  const int most = X_BYTES / (cols * 2) / STEP * STEP;
  p.chunk_k = p.part_k < most ? p.part_k : most;
  // ring slots: what shared memory leaves once the CTAs that each SM gets (at most ctas_per_sm) and their x have a place
  const int64_t per_sm = std::min<int64_t>(ctas_per_sm(COLS8), (tiles * passes * parts + num_sms() - 1) / num_sms());
  const int beside = WARPS * ROWS * COLS8 * 8 * 4 + p.chunk_k * cols * 2;  // the sums and x
  const int64_t left = SM_BYTES / per_sm - CTA_BYTES - beside;
  const int64_t fit = std::min<int64_t>(left / (WARPS * SLOT), (p.part_k + STEP - 1) / STEP);
  p.stages = static_cast<int>(std::max<int64_t>(2, std::min<int64_t>(MOST_STAGES, fit)));
  const int smem = 1024 + WARPS * p.stages * SLOT + beside;
  static int configured[64] = {0};
  int dev = 0;
  IRIS_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || configured[dev] == 0) {
    IRIS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 1024 + WARPS * MOST_STAGES * SLOT + WARPS * ROWS * COLS8 * 8 * 4 + X_BYTES));
    if (dev < 64) configured[dev] = 1;
  }
  CUtensorMap tw;
  IRIS_CHECK_STATUS(make_tmap_2d_bytes(&tw, p.packed, p.K / 2, p.N, p.K / 2, STEP / 2, ROWS));
  IRIS_CUDA(launch_early(kernel, dim3(static_cast<unsigned>(tiles * parts), static_cast<unsigned>(passes)), THREADS, smem, st,
                         static_cast<unsigned>(parts), tw, p));
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

extern "C" int iris_gemv_q4(const iris_q4_problem* q, void* stream) {
  using namespace iris::q4;
  IRIS_REQUIRE(q != nullptr && q->x && q->packed && q->scale && q->out, "gemv_q4: null pointer");
  IRIS_REQUIRE(q->group == 32 || q->group == 64 || q->group == 128, "gemv_q4: groups of 32, 64 or 128 weights");
  IRIS_REQUIRE(q->M > 0 && q->M <= 64 && q->N > 0 && q->K > 0 && q->K % q->group == 0,
               "gemv_q4: 1 to 64 rows; K must be a multiple of the group");
  IRIS_REQUIRE(q->N < (1ll << 28) && q->K < (1ll << 28) && q->ldx >= q->K, "gemv_q4: size");
  IRIS_REQUIRE(q->x_dtype >= IRIS_F32 && q->x_dtype <= IRIS_F16 && q->out_dtype >= IRIS_F32 && q->out_dtype <= IRIS_F16,
               "gemv_q4: bad dtype");
  IRIS_REQUIRE(aligned16(q->x) && aligned16(q->packed) && aligned_n(q->scale, 2) && q->ldx % 8 == 0,
               "gemv_q4: x rows and weights must be 16-byte aligned");
  Params p = {};
  p.x = q->x, p.x_dtype = static_cast<int>(q->x_dtype), p.M = static_cast<int>(q->M), p.K = static_cast<int>(q->K);
  p.ldx = q->ldx, p.packed = static_cast<const uint8_t*>(q->packed);
  p.scale = static_cast<const __nv_bfloat16*>(q->scale), p.zero = static_cast<const uint8_t*>(q->zero);
  p.bias = q->bias, p.out = q->out, p.out_dtype = static_cast<int>(q->out_dtype), p.N = static_cast<int>(q->N);
  p.silu_in = q->silu_in != 0, p.silu_out = q->silu_out != 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p.x_dtype == IRIS_F32 || p.silu_in) {  // fp32 values: three columns a row
    if (p.M <= 2) return launch<__nv_bfloat16, 3, 1>(p, q->group, st);
    if (p.M <= 5) return launch<__nv_bfloat16, 3, 2>(p, q->group, st);
    if (p.M <= 8) return launch<__nv_bfloat16, 3, 3>(p, q->group, st);
    return launch<__nv_bfloat16, 3, 6>(p, q->group, st);
  }
  if (p.x_dtype == IRIS_F16) return launch_rows<__half>(p, q->group, st);
  return launch_rows<__nv_bfloat16>(p, q->group, st);
}
