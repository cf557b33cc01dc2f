// Linear over 8-bit weights with a scale for each token and channel:
//   x_scale[m] = max_k |x[m, k]| / 127,   q[m, k] = the whole number nearest 127 x[m, k] / max_k |x[m, k]|
//   out[m, n] = x_scale[m] w_scale[n] sum_k q[m, k] w[n, k] + bias[n]
// The sum is of whole numbers and exact in int32 (K <= 131071: 128 * 128 * K < 2^31),
// so how K is split changes nothing.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "iris_abi_internal.h"

namespace iris {
namespace i8 {

// ------------------------------------------------------------------ rows to 8 bits
// HBM-bound: one read of x, one byte written per value. A team of warps takes a row and
// keeps it in registers between the maximum and the rounding (what does not fit is read again).
//
// q is the correctly rounded quotient y = 127 x / max, halves to even, so that the 8-bit
// values are the formula's, whatever order or unit computes them.
//  - Rows of 16 bits meet halves often (a quarter of a warp's vectors hold one). With 127 / max =
//    hi + lo to 48 bits, fma(x, hi, x lo) is y rounded to fp32: a half comes out as
//    itself, and any other y, a ratio of short numbers, stays on its side: it is at least 2^-19 of
//    itself away (254 m - h M 2^j is a whole number, m and M below 2^11), fp32 rounds by 2^-24.
//  - FP32 rows: x hi is off by at most 127 (2^-24 + 2^-24) < 2^-16, so its nearest whole number
//    is y's unless it lies within 2^-15 of a half h; then 254 x is compared with 2 h max,
//    both exact in 64 bits.
//
// Measured, bf16: 16384 rows of 8192 92 to 94 us (4.4 TB/s; 110 without the next row's loads under this
// one's rounding, 170 with halves looked at again), 2400 of 2560 5.2, 8 of 2560 1.8.
struct QuantizeParams {
  const void* x;
  int8_t* q;
  float* scale;
  int64_t ldx, ldq;
  int M, K;
};

template <typename T>
struct Vec {  // values of a 16-byte vector
  static constexpr int N = 16 / sizeof(T);
};

template <typename T>
IRIS_DEVICE float value_of(const uint4& v, int e);
template <>
IRIS_DEVICE float value_of<float>(const uint4& v, int e) {
  return __uint_as_float(e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w);
}
template <>
IRIS_DEVICE float value_of<__nv_bfloat16>(const uint4& v, int e) {
  const uint32_t w = e < 2 ? v.x : e < 4 ? v.y : e < 6 ? v.z : v.w;
  return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
}
template <>
IRIS_DEVICE float value_of<__half>(const uint4& v, int e) {
  const uint32_t w = e < 2 ? v.x : e < 4 ? v.y : e < 6 ? v.z : v.w;
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return e & 1 ? f.y : f.x;
}

// Largest magnitude of a vector as the bits of its type: they order like magnitudes,
// infinities and NaN above all others.
template <typename T>
IRIS_DEVICE uint32_t top_of(const uint4& v, uint32_t top) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    top = sizeof(T) == 4 ? max(top, w[i] & 0x7fffffffu) : __vmaxu2(top, w[i] & 0x7fff7fffu);
  return top;
}

template <typename T, bool ALIGNED>
IRIS_DEVICE uint4 load_vec(const T* row, int v, int K) {
  constexpr int N = Vec<T>::N;
  if (ALIGNED && (v + 1) * N <= K) return *reinterpret_cast<const uint4*>(row + v * N);
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const int k = v * N + e;
    if (k >= K) continue;
    if (sizeof(T) == 4) w[e % 4] = reinterpret_cast<const uint32_t*>(row)[k];
    else w[e / 2 % 4] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(row)[k]) << (16 * (e & 1));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// What a row's values are multiplied by.
struct Factors {
  float hi, lo;  // 127 / (top up)
  float top, up; // the largest magnitude, scaled by a power of two where it is extreme (extreme: up is not 1)
};

// A vector's 8-bit values from 64-bit comparisons: values next to halves, and rows of
// extreme values, whose factors alone would leave fp32.
template <typename T>
__device__ __noinline__ uint2 round_exactly(uint4 v, float hi, float top, float up) {
  uint32_t packed[2] = {0u, 0u};
#pragma unroll 1
  for (int e = 0; e < Vec<T>::N; ++e) {
    const float x = value_of<T>(v, e) * up;
    const float low = floorf(x * hi);
    const double off = fma(254.0, static_cast<double>(x), -(2.0 * low + 1.0) * top);
    const int lo = static_cast<int>(low), q = off > 0 || (off == 0 && (lo & 1)) ? lo + 1 : lo;
    packed[e >> 2] |= (static_cast<uint32_t>(q) & 0xffu) << (8 * (e & 3));
  }
  return make_uint2(packed[0], packed[1]);
}

template <typename T>
IRIS_DEVICE uint2 round_vec(const uint4& v, const Factors& f) {
  constexpr int N = Vec<T>::N;
  uint32_t packed[2] = {0u, 0u};
  bool again = f.up != 1.f;
  constexpr float kWhole = 12582912.f;  // 1.5 * 2^23: the sum's last bit is 1
  const float2 hi = make_float2(f.hi, f.hi), lo = make_float2(f.lo, f.lo), whole = make_float2(kWhole, kWhole);
#pragma unroll
  for (int g = 0; g < N / 4; ++g) {
    uint32_t b[4];
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      const float2 x = make_float2(value_of<T>(v, 4 * g + e), value_of<T>(v, 4 * g + e + 1));
      float2 t;
      if (sizeof(T) == 2) {
        t = __fadd2_rn(__ffma2_rn(x, hi, __fmul2_rn(x, lo)), whole);
      } else {
        t = __ffma2_rn(x, hi, whole);
        const float2 r = __ffma2_rn(x, hi, __ffma2_rn(t, make_float2(-1.f, -1.f), whole));  // minus the whole number
        again = again || fmaxf(fabsf(r.x), fabsf(r.y)) > 0.5f - 1.f / 32768;
      }
      b[e] = __float_as_uint(t.x), b[e + 1] = __float_as_uint(t.y);
    }
    packed[g] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  }
  return again ? round_exactly<T>(v, f.hi, f.top, f.up) : make_uint2(packed[0], packed[1]);
}

template <typename T>
IRIS_DEVICE void store_vec(int8_t* out, const uint4& v, int at, int K, const Factors& f) {
  constexpr int N = Vec<T>::N;
  const uint2 w = round_vec<T>(v, f);
  if ((at + 1) * N <= K) {
    if (N == 8) *reinterpret_cast<uint2*>(out + at * N) = w;
    else *reinterpret_cast<uint32_t*>(out + at * N) = w.x;
  } else {
    const uint32_t packed[2] = {w.x, w.y};
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (at * N + e < K) out[at * N + e] = static_cast<int8_t>(packed[e >> 2] >> (8 * (e & 3)) & 0xffu);
  }
}

// From the bits of a row's largest magnitude. Extreme rows are scaled to where the factors are
// normal numbers, exactly but for values that round to 0; a row that is not finite gives
// zeros (its values are to be taken as such).
template <typename T>
IRIS_DEVICE Factors factors_of(uint32_t top, float* scale) {
  const float size = value_of<T>(make_uint4(top, 0u, 0u, 0u), 0);
  const bool finite = size < INFINITY;  // not so for NaN
  *scale = finite ? __fdiv_rn(size, 127.f) : NAN;
  Factors f;
  f.up = !finite ? 0.f : size < 0x1p-100f ? 0x1p100f : size > 0x1p60f ? 0x1p-100f : 1.f;
  f.top = finite ? size * f.up : 0.f;
  f.hi = f.top > 0.f ? __fdiv_rn(127.f, f.top) : 0.f;
  f.lo = f.top > 0.f ? __fdiv_rn(fmaf(-f.hi, f.top, 127.f), f.top) : 0.f;
  return f;
}

constexpr int KEPT = 4;  // vectors of a row that a thread keeps

template <typename T, int WARPS, bool ALIGNED>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : WARPS * 32, WARPS == 8 ? 4 : 8) quantize_kernel(const QuantizeParams p) {
  constexpr int TEAM = WARPS * 32, N = Vec<T>::N;
  __shared__ uint32_t tops[2][WARPS];
  // in this order: the product behind this kernel copies weights before its own wait (Params::early),
  // which are there because every CTA here has waited for what may have written them
  grid_wait();
  grid_trigger();
  const int t = WARPS == 1 ? threadIdx.x & 31 : threadIdx.x;
  const int vecs = (p.K + N - 1) / N;
  const int step = WARPS == 1 ? gridDim.x * 4 : gridDim.x;
  const T* x = reinterpret_cast<const T*>(p.x);
  uint4 kept[KEPT];
  auto load = [&](int64_t m) {
#pragma unroll
    for (int i = 0; i < KEPT; ++i) {
      const int v = t + i * TEAM;
      kept[i] = m < p.M && v < vecs ? load_vec<T, ALIGNED>(x + m * p.ldx, v, p.K) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  int64_t m = WARPS == 1 ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
  load(m);
  for (int turn = 0; m < p.M; m += step, turn ^= 1) {
    const T* row = x + m * p.ldx;
    uint4 now[KEPT];
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < KEPT; ++i) {
      now[i] = kept[i];
      top = top_of<T>(now[i], top);
    }
    load(m + step);  // the next row's values are on their way while this one's are rounded
    for (int v = t + KEPT * TEAM; v < vecs; v += TEAM) top = top_of<T>(load_vec<T, ALIGNED>(row, v, p.K), top);
    if (sizeof(T) == 2) top = max(top & 0xffffu, top >> 16);
    top = __reduce_max_sync(0xffffffffu, top);
    if (WARPS > 1) {
      if ((threadIdx.x & 31) == 0) tops[turn][threadIdx.x >> 5] = top;
      __syncthreads();  // and no warp is a row ahead of another's reading
#pragma unroll
      for (int w = 0; w < WARPS; ++w) top = max(top, tops[turn][w]);
    }
    float scale;
    const Factors f = factors_of<T>(top, &scale);
    const bool finite = f.up != 0.f;
    if (t == 0) p.scale[m] = scale;
    int8_t* out = p.q + m * p.ldq;
    auto store = [&](const uint4& v, int at) { store_vec<T>(out, finite ? v : make_uint4(0u, 0u, 0u, 0u), at, p.K, f); };
#pragma unroll
    for (int i = 0; i < KEPT; ++i)
      if (t + i * TEAM < vecs) store(now[i], t + i * TEAM);
    for (int v = t + KEPT * TEAM; v < vecs; v += TEAM) store(load_vec<T, ALIGNED>(row, v, p.K), v);
  }
}

template <typename T, bool ALIGNED>
int launch_quantize(const QuantizeParams& p, cudaStream_t st) {
  const int vecs = (p.K + Vec<T>::N - 1) / Vec<T>::N;
  // the smallest team that keeps a row; no more CTAs than the SMs hold at once
  const int64_t rows = p.M, sms = num_sms();
  if (vecs <= KEPT * 32)
    IRIS_CUDA(launch_early(quantize_kernel<T, 1, ALIGNED>, dim3(static_cast<unsigned>(std::min((rows + 3) / 4, 8 * sms))), 128, 0, st, 1, p));
  else if (vecs <= KEPT * 128)
    IRIS_CUDA(launch_early(quantize_kernel<T, 4, ALIGNED>, dim3(static_cast<unsigned>(std::min(rows, 8 * sms))), 128, 0, st, 1, p));
  else
    IRIS_CUDA(launch_early(quantize_kernel<T, 8, ALIGNED>, dim3(static_cast<unsigned>(std::min(rows, 4 * sms))), 256, 0, st, 1, p));
  return IRIS_OK;
}

template <typename T>
int quantize(const QuantizeParams& p, cudaStream_t st) {
  const bool aligned = aligned16(p.x) && p.ldx * static_cast<int64_t>(sizeof(T)) % 16 == 0;
  return aligned ? launch_quantize<T, true>(p, st) : launch_quantize<T, false>(p, st);
}

// ------------------------------------------------------------------- the product
// A tile is 128 weight rows (TMEM lanes) by T tokens (columns): the weights are the
// tensor cores' first operand, whatever the number of tokens, so that few tokens waste
// none of it and the lanes of a warp write neighbouring channels of out, at any N.
//
// Measured in graph replays, us, rows in bf16 and their rounding included (tokens, K -> N): 1, 2560 ->
// 2560 5.5 (the product alone 4.5; x is read twice, a barrier between, then the cluster's exchange);
// 64, 8192 -> 32768 51.5 (5.3 TB/s of weights, 0.81 of a plain copy; 53 among other work); 2400, 2560 ->
// 6848 42 (2.0 POP/s: 270 tiles are 3.65 waves of 74 pairs, and 6 us start and end them); 4096, 8192 ->
// 8192 193, 174 of them the product (tensor pipe 82% busy); 16384, 8192 -> 8192 770 to 780 in short
// runs, the product 680 to 725 (2.9 to 3.2 POP/s), 843 in long ones under the power cap.
constexpr int BN = 128, SLAB = 128;  // weight rows of a CTA, k of a ring slot (bytes)
constexpr int EPILOGUE = 8;  // warps: two for each quarter of the TMEM lanes, half of the tokens each
constexpr int THREADS = 64 + 32 * EPILOGUE;

struct Params {
  const float* x_scale;
  const float* w_scale;
  const float* bias;
  void* out;
  int M, N, K, out_dtype;
  int splits;         // parts of K, the CTAs of a cluster
  int token_tiles;
  int early;          // the predecessor is this call's quantize_kernel: the weights are there before it ends
};

__host__ __device__ constexpr uint32_t idesc_i8(int m, int n) {
  return (2u << 4)                                // D format: S32
         | (1u << 7)                              // A format: signed 8-bit
         | (1u << 10)                             // B format: signed 8-bit
         | (static_cast<uint32_t>(n >> 3) << 17)  // N / 8
         | (static_cast<uint32_t>(m >> 4) << 24); // M / 16
}
IRIS_DEVICE void umma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// sum * x_scale * w_scale: the smaller scale first, so that no step leaves fp32 where
// the product does not. A NaN scale stays.
IRIS_DEVICE float scaled(int sum, float xs, float ws, float bias) {
  const bool less = fabsf(xs) < fabsf(ws);
  return fmaf(static_cast<float>(sum) * (less ? xs : ws), less ? ws : xs, bias);
}
IRIS_DEVICE void store_out(const Params& p, int64_t at, float y) { store_elem(p.out, at, p.out_dtype, y); }

template <typename O>
IRIS_DEVICE O rounded(float y);
template <>
IRIS_DEVICE float rounded<float>(float y) { return y; }
template <>
IRIS_DEVICE __nv_bfloat16 rounded<__nv_bfloat16>(float y) { return __float2bfloat16_rn(y); }
template <>
IRIS_DEVICE __half rounded<__half>(float y) { return __float2half_rn(y); }

// A warp's 32 channels (lane: channel n) of tokens [m0, m0 + count) from TMEM columns [at, at + count).
template <typename O>
IRIS_DEVICE void store_columns_as(const Params& p, uint32_t at, int m0, int count, int n, bool ok) {
  const int lane = threadIdx.x & 31;
  const bool real = n < p.N;
  const float ws = real ? p.w_scale[n] : 0.f, bias = real && p.bias ? p.bias[n] : 0.f;
  O* out = reinterpret_cast<O*>(p.out) + static_cast<int64_t>(m0) * p.N + n;
#pragma unroll 1
  for (int c = 0; c < count; c += 16) {
    const int most = real ? p.M - m0 - c : 0;
    if (m0 + c >= p.M) break;
    uint32_t r[16];
    tmem_ld16(at + c, r);
    const float mine = m0 + c + (lane & 15) < p.M ? p.x_scale[m0 + c + (lane & 15)] : 0.f;
    tmem_wait_ld();
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float xs = __shfl_sync(0xffffffffu, mine, e);
      const float y = ok ? scaled(static_cast<int>(r[e]), xs, ws, bias) : NAN;
      if (e < most) *out = rounded<O>(y);
      out += p.N;
    }
  }
}
IRIS_DEVICE void store_columns(const Params& p, uint32_t at, int m0, int count, int n, bool ok) {
  if (p.out_dtype == IRIS_F32) store_columns_as<float>(p, at, m0, count, n, ok);
  else if (p.out_dtype == IRIS_BF16) store_columns_as<__nv_bfloat16>(p, at, m0, count, n, ok);
  else store_columns_as<__half>(p, at, m0, count, n, ok);
}

// Few tokens, or few weight rows: a CTA of T tokens, two CTAs to an SM or (DEEP) one with
// twice the ring, filled and committed two slabs at a time.
template <int T, bool DEEP>
struct Rows {
  static constexpr int SLABS = DEEP ? 2 : 1;  // of a stage
  static constexpr int X_BYTES = T * SLAB, W_BYTES = BN * SLAB, STAGE = SLABS * (X_BYTES + W_BYTES);
  static constexpr int STAGES = T <= 32 ? 5 : T == 64 ? 4 : 3;
  static constexpr int COLS = T < 32 ? 32 : T;
  static constexpr int RING = STAGES * STAGE;
  // the parts' sums: few tokens' have a place of their own, many tokens' lie in the ring
  static constexpr bool APART = T <= 16;
  static constexpr int PARTS = T * BN * 4;
  static constexpr int SMEM = 1024 + RING + (APART ? PARTS : 0) + 256;
  static_assert(PARTS <= RING && SMEM <= 232448, "the parts of a tile lie in the ring");
};

template <int T, bool DEEP>
struct RowsSmem {
  uint64_t full[Rows<T, DEEP>::STAGES], empty[Rows<T, DEEP>::STAGES], done;
  uint32_t tmem_base;
  int abort, bad[8];
};

template <int T, bool DEEP>
__global__ void __launch_bounds__(THREADS, DEEP ? 1 : 2)
    rows_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tx,
                const __grid_constant__ Params p) {
  using R = Rows<T, DEEP>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  auto* s = reinterpret_cast<RowsSmem<T, DEEP>*>(ring + R::RING + (R::APART ? R::PARTS : 0));
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const int part = static_cast<int>(blockIdx.x % p.splits), unit = static_cast<int>(blockIdx.x / p.splits);
  const int m0 = unit % p.token_tiles * T, n0 = unit / p.token_tiles * BN;
  const int slabs = (p.K + SLAB - 1) / SLAB;
  const int first = static_cast<int>(static_cast<int64_t>(slabs) * part / p.splits);
  const int count = static_cast<int>(static_cast<int64_t>(slabs) * (part + 1) / p.splits) - first;
  const int steps = (count + R::SLABS - 1) / R::SLABS;

  if (threadIdx.x == 0) {
    for (int i = 0; i < R::STAGES; ++i) {
      mbar_init(&s->full[i], 1);
      mbar_init(&s->empty[i], 1);
    }
    mbar_init(&s->done, 1);
    s->abort = 0;
    for (int i = 0; i < 8; ++i) s->bad[i] = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tw);
    tma_prefetch_desc(&tx);
  }
  auto load_w = [&](int i) {
    const int st = i % R::STAGES, n = min(R::SLABS, count - i * R::SLABS);
    mbar_arrive_expect_tx(&s->full[st], n * (R::W_BYTES + R::X_BYTES));
    for (int j = 0; j < n; ++j)
      tma_load_2d(&tw, &s->full[st], ring + st * R::STAGE + j * R::W_BYTES, (first + i * R::SLABS + j) * SLAB, n0);
  };
  const int ahead = p.early ? min(steps, R::STAGES) : 0;
  if (threadIdx.x == 0)
    for (int i = 0; i < ahead; ++i) load_w(i);
  __syncthreads();
  if (p.splits > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  volatile int* abort = &s->abort;
  grid_wait();

  if (warp == 0) {
    // ----------------------------------------------------------------- TMA
    if (lane == 0) {
      auto load_x = [&](int i) {
        const int st = i % R::STAGES, n = min(R::SLABS, count - i * R::SLABS);
        for (int j = 0; j < n; ++j)
          tma_load_2d(&tx, &s->full[st], ring + st * R::STAGE + R::SLABS * R::W_BYTES + j * R::X_BYTES,
                      (first + i * R::SLABS + j) * SLAB, m0);
      };
      for (int i = 0; i < ahead; ++i) load_x(i);
      bool ok = true;
      int issued = ahead;
      for (; issued < steps; ++issued) {
        ok = mbar_wait(&s->empty[issued % R::STAGES], static_cast<uint32_t>((issued / R::STAGES) & 1) ^ 1u, abort);
        if (!ok) break;
        load_w(issued);
        load_x(issued);
      }
      if (!ok) {  // no copy may land after the CTA is gone
        int dummy = 0;
        for (int i = max(0, issued - R::STAGES); i < issued; ++i)
          mbar_wait(&s->full[i % R::STAGES], static_cast<uint32_t>((i / R::STAGES) & 1), &dummy);
      }
    }
  } else if (warp == 1) {
    // ----------------------------------------------------------------- MMA
    // TMEM only after the wait (a CTA that held some while it waits could keep its predecessor's,
    // which still have to allocate theirs, from ever ending), and the successor only after TMEM
    tmem_alloc(&s->tmem_base, R::COLS);
    grid_trigger();
    tc_fence_before();
    __syncwarp();
    barrier_tell<1, 32 + 32 * EPILOGUE>();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&s->tmem_base);
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_i8(BN, T);
      for (int i = 0; i < steps; ++i) {
        const int st = i % R::STAGES, n = min(R::SLABS, count - i * R::SLABS);
        if (!mbar_wait(&s->full[st], static_cast<uint32_t>((i / R::STAGES) & 1), abort)) break;
        tc_fence_after();
        for (int j = 0; j < n; ++j) {
          const uint32_t w_addr = smem_addr(ring + st * R::STAGE + j * R::W_BYTES);
          const uint32_t x_addr = smem_addr(ring + st * R::STAGE + R::SLABS * R::W_BYTES + j * R::X_BYTES);
#pragma unroll
          for (int k = 0; k < SLAB / 32; ++k)
            umma_i8(tmem, umma_desc(w_addr + k * 32, 16, 1024, kLayoutSw128), umma_desc(x_addr + k * 32, 16, 1024, kLayoutSw128),
                    idesc, (i | j | k) != 0 ? 1u : 0u);
        }
        umma_commit(&s->empty[st]);
      }
      umma_commit(&s->done);  // also after a wait that gave up: all that was issued ends before TMEM is freed
      int dummy = 0;
      mbar_wait(&s->done, 0, &dummy);
    }
  }
  __syncwarp();
  // ------------------------------------------------------------- epilogue
  bool ok = true;
  float my_scale = 0.f, my_bias = 0.f;
  uint32_t tmem = 0;
  if (warp >= 2) {
    if (n0 + (warp & 3) * 32 + lane < p.N) {
      my_scale = p.w_scale[n0 + (warp & 3) * 32 + lane];
      if (p.bias) my_bias = p.bias[n0 + (warp & 3) * 32 + lane];
    }
    barrier_wait<1, 32 + 32 * EPILOGUE>();
    tmem = s->tmem_base;
    ok = __all_sync(0xffffffffu, mbar_wait(&s->done, 0, abort));
    ok = ok && *abort == 0;
    tc_fence_after();
  }
  const int quarter = warp & 3, half = warp >= 6;
  const int n = n0 + quarter * 32 + lane;
  const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  const bool real = n < p.N;
  constexpr int SHARE = T >= 32 ? T / 2 : T;  // a warp's tokens; fewer than 32 are one warp's
  const int c_first = half * SHARE, c_end = min(T, c_first + SHARE);
  if (p.splits == 1) {
    if (warp >= 2 && c_first < T) store_columns(p, lanes + c_first, m0 + c_first, SHARE, n, ok);
  } else {
    // each part's sums go to the CTA that owns the columns: as soon as it has begun, or, where
    // they lie in its ring, when no copy and no MMA of that CTA uses it any more
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (!R::APART) cluster_sync();
    const int own = T / p.splits, log_own = __ffs(own) - 1;  // columns of a CTA: a power of two, 2 at least
    // a lane's sums in neighbouring words: 128 bytes a store (four columns of a lane as one
    // 16-byte store each took a third longer: 64 rows 2560 -> 2560 8.8 -> 11.7 us)
    int* parts = reinterpret_cast<int*>(ring + (R::APART ? R::RING : 0));  // [part][column][128]
    if (warp >= 2) {
#pragma unroll 1
      for (int c = c_first; c < c_end; c += 16) {
        uint32_t r[16];
        tmem_ld16(lanes + c, r);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int col = c + e;
          const uint32_t to = map_to_cta(parts + (part * own + (col & (own - 1))) * BN + quarter * 32 + lane,
                                         static_cast<uint32_t>(col >> log_own));
          asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(r[e]) : "memory");
        }
      }
      if (!ok && lane < p.splits) {
        const uint32_t to = map_to_cta(&s->bad[part], static_cast<uint32_t>(lane));
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(1) : "memory");
      }
    }
    cluster_sync();
    if (warp >= 2) {
      bool bad = false;
      for (int i = 0; i < p.splits; ++i) bad = bad || s->bad[i] != 0;
      const int* from = parts + quarter * 32 + lane;
#pragma unroll 1
      for (int c = 4 * half; c < own; c += 8) {
        const int m = m0 + part * own + c;
        if (m >= p.M) break;
        int sum[4] = {0, 0, 0, 0};
#pragma unroll 2
        for (int i = 0; i < p.splits; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (e < 2 || own >= 4) sum[e] += from[(i * own + c + e) * BN];
        const int most = real ? min(min(own, 4), p.M - m) : 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < most) store_out(p, static_cast<int64_t>(m + e) * p.N + n, bad ? NAN : scaled(sum[e], p.x_scale[m + e], my_scale, my_bias));
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(s->tmem_base, R::COLS);
}

template <int T, bool DEEP>
int launch_rows(const CUtensorMap& tw, const CUtensorMap& tx, Params p, int splits, cudaStream_t st) {
  auto kernel = rows_kernel<T, DEEP>;
  static bool configured[64] = {false};
  int dev = 0;
  IRIS_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !configured[dev]) {
    IRIS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Rows<T, DEEP>::SMEM));
    if (dev < 64) configured[dev] = true;
  }
  p.token_tiles = (p.M + T - 1) / T;
  p.splits = splits;
  const int64_t ctas = static_cast<int64_t>(p.token_tiles) * ((p.N + BN - 1) / BN) * splits;
  IRIS_REQUIRE(ctas < (1ll << 31), "gemm_i8: too many rows");
  IRIS_CUDA(launch_early(kernel, dim3(static_cast<unsigned>(ctas)), THREADS, Rows<T, DEEP>::SMEM, st, static_cast<unsigned>(splits), tw,
                         tx, p));
  return IRIS_OK;
}

// rows_kernel that rounds its tokens itself, one launch instead of two: every CTA reads its rows
// whole for their largest magnitudes and lays its own part of K out in shared memory, as TMA
// would have. It is taken (few_tokens) where the device is done as early as with two launches or
// earlier; the host is, by some 3 us, in any case.
//  - T 32, 64 or 128, rows of one slab (SHORT_ROW bytes): all rows of a tile at once, a few lanes
//    each. More lanes a row are faster, so T 32 while its tiles have an SM each.
//  - T 16, up to MOST_ROWS longer rows: K in parts, a warp or more a row.
namespace few {
constexpr int STAGES = 4, RING = STAGES * BN * SLAB, X = 32768, PARTS = 16 * BN * 4;
constexpr int most_slabs(int T) { return X / (T * SLAB); }  // slabs of a CTA
constexpr int64_t SHORT_ROW = 256, MOST_TOKENS = 128, MOST_ROWS = 8;
struct Smem {
  uint64_t full[STAGES], empty[STAGES], x_full, done;
  uint32_t tmem_base;
  int abort, bad[8];
  uint32_t top[MOST_ROWS];
  float scale[128];
};
constexpr int SMEM = 1024 + RING + X + PARTS + static_cast<int>(sizeof(Smem));
}  // namespace few

template <typename V, int T, bool ALIGNED>
__global__ void __launch_bounds__(THREADS, 2)
    few_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ Params p, const V* x, int64_t ldx) {
  using namespace few;
  constexpr int N = Vec<V>::N, X_SLAB = T * SLAB, COLS = T < 32 ? 32 : T;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* rows = ring + RING;
  int* parts = reinterpret_cast<int*>(rows + X);  // [part][column][128]
  few::Smem* s = reinterpret_cast<few::Smem*>(rows + X + PARTS);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const int part = static_cast<int>(blockIdx.x % p.splits), unit = static_cast<int>(blockIdx.x / p.splits);
  const int m0 = unit % p.token_tiles * T, n0 = unit / p.token_tiles * BN;
  const int tokens = min(T, p.M - m0);
  const int slabs = (p.K + SLAB - 1) / SLAB;
  const int first = slabs * part / p.splits, count = slabs * (part + 1) / p.splits - first;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&s->full[i], 1);
      mbar_init(&s->empty[i], 1);
    }
    mbar_init(&s->x_full, EPILOGUE);
    mbar_init(&s->done, 1);
    s->abort = 0;
    for (int i = 0; i < 8; ++i) s->bad[i] = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tw);
  }
  if (threadIdx.x < MOST_ROWS) s->top[threadIdx.x] = 0u;
  __syncthreads();
  volatile int* abort = &s->abort;
  if (p.splits > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  grid_wait();

  bool ok = true;
  float my_scale = 0.f, my_bias = 0.f;
  uint32_t tmem = 0;
  const int quarter = warp & 3, half = warp >= 6;
  const int n = n0 + quarter * 32 + lane;
  if (warp == 0) {
    // ----------------------------------------------------------------- TMA
    if (lane == 0) {
      int issued = 0;
      for (; issued < count; ++issued) {
        const int st = issued % STAGES;
        ok = mbar_wait(&s->empty[st], static_cast<uint32_t>((issued / STAGES) & 1) ^ 1u, abort);
        if (!ok) break;
        mbar_arrive_expect_tx(&s->full[st], BN * SLAB);
        tma_load_2d(&tw, &s->full[st], ring + st * BN * SLAB, (first + issued) * SLAB, n0);
      }
      if (!ok) {  // no copy may land after the CTA is gone
        int dummy = 0;
        for (int i = max(0, issued - STAGES); i < issued; ++i)
          mbar_wait(&s->full[i % STAGES], static_cast<uint32_t>((i / STAGES) & 1), &dummy);
      }
    }
  } else if (warp == 1) {
    // ----------------------------------------------------------------- MMA
    tmem_alloc(&s->tmem_base, COLS);  // after the wait and before the successor, as in rows_kernel
    grid_trigger();
    tc_fence_before();
    __syncwarp();
    barrier_tell<2, 32 + 32 * EPILOGUE>();
    tmem = *reinterpret_cast<volatile uint32_t*>(&s->tmem_base);
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_i8(BN, T);
      ok = mbar_wait(&s->x_full, 0, abort);
      for (int i = 0; i < count && ok; ++i) {
        const int st = i % STAGES;
        ok = mbar_wait(&s->full[st], static_cast<uint32_t>((i / STAGES) & 1), abort);
        if (!ok) break;
        tc_fence_after();
        const uint32_t w_addr = smem_addr(ring + st * BN * SLAB), x_addr = smem_addr(rows + i * X_SLAB);
#pragma unroll
        for (int k = 0; k < SLAB / 32; ++k)
          umma_i8(tmem, umma_desc(w_addr + k * 32, 16, 1024, kLayoutSw128), umma_desc(x_addr + k * 32, 16, 1024, kLayoutSw128),
                  idesc, (i | k) != 0 ? 1u : 0u);
        umma_commit(&s->empty[st]);
      }
      umma_commit(&s->done);  // also after a wait that gave up: all that was issued ends before TMEM is freed
      int dummy = 0;
      mbar_wait(&s->done, 0, &dummy);
    }
  } else {
    // ------------------------------------------------------------- the rows
    if (n < p.N) {
      my_scale = p.w_scale[n];
      if (p.bias) my_bias = p.bias[n];
    }
    const int vecs = (p.K + N - 1) / N;
    constexpr int OF_SLAB = SLAB / N;
    const V* row0 = x + m0 * ldx;
    // the 8-bit values of vector i of this part, of row m, in their swizzled place: 16-byte piece c of row r at c ^ (r & 7)
    auto place = [&](int m, int i, const Factors& f) {
      const int v = first * OF_SLAB + i;
      const uint4 value = v < vecs && f.up != 0.f ? load_vec<V, ALIGNED>(row0 + m * ldx, v, p.K) : make_uint4(0u, 0u, 0u, 0u);
      const uint2 q = round_vec<V>(value, f);
      const int byte = i % OF_SLAB * N;
      uint8_t* to = rows + i / OF_SLAB * X_SLAB + m * SLAB + (((byte >> 4) ^ (m & 7)) * 16) + (byte & 15);
      if (N == 8) *reinterpret_cast<uint2*>(to) = q;
      else *reinterpret_cast<uint32_t*>(to) = q.x;
    };
    // rows that are not there are zeros
    for (int i = threadIdx.x - 64; i < count * (T - tokens) * (SLAB / 16); i += 32 * EPILOGUE) {
      const int piece = i % (SLAB / 16), row = tokens + i / (SLAB / 16) % (T - tokens), slab = i / (SLAB / 16) / (T - tokens);
      *reinterpret_cast<uint4*>(rows + slab * X_SLAB + row * SLAB + piece * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
    if (T > 16) {
      // all rows at once, a few lanes each
      constexpr int LANES = 32 * EPILOGUE / T;
      const int m = (threadIdx.x - 64) / LANES, l = threadIdx.x % LANES;
      uint32_t top = 0u;
      if (m < tokens) {
#pragma unroll 4
        for (int v = l; v < vecs; v += LANES) top = top_of<V>(load_vec<V, ALIGNED>(row0 + m * ldx, v, p.K), top);
      }
      if (sizeof(V) == 2) top = max(top & 0xffffu, top >> 16);
#pragma unroll
      for (int o = 1; o < LANES; o *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (m < tokens) {
        float scale;
        const Factors f = factors_of<V>(top, &scale);
        if (l == 0) s->scale[m] = scale;
#pragma unroll 2
        for (int i = l; i < count * OF_SLAB; i += LANES) place(m, i, f);
      }
    } else {
      const int w = warp - 2, share = tokens == 1 ? 8 : tokens == 2 ? 4 : tokens <= 4 ? 2 : 1, m = w / share;  // warps of a row
      if (m < tokens) {
        uint32_t top = 0u;
#pragma unroll 2
        for (int v = w % share * 32 + lane; v < vecs; v += share * 32)
          top = top_of<V>(load_vec<V, ALIGNED>(row0 + m * ldx, v, p.K), top);
        if (sizeof(V) == 2) top = max(top & 0xffffu, top >> 16);
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) atomicMax(&s->top[m], top);
      }
      barrier_wait<1, 32 * EPILOGUE>();
      if (m < tokens) {
        float scale;
        const Factors f = factors_of<V>(s->top[m], &scale);
        if (lane == 0) s->scale[m] = scale;
#pragma unroll 1
        for (int i = w % share * 32 + lane; i < count * OF_SLAB; i += share * 32) place(m, i, f);
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&s->x_full);
    barrier_wait<2, 32 + 32 * EPILOGUE>();  // every row's scale is there, and TMEM
    tmem = s->tmem_base;
    ok = __all_sync(0xffffffffu, mbar_wait(&s->done, 0, abort));
    ok = ok && *abort == 0;
    tc_fence_after();
  }
  __syncwarp();
  // ------------------------------------------------------------- epilogue
  const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  if (T > 16) {
    Params mine = p;  // of the tile's tokens
    mine.x_scale = s->scale;
    mine.M = tokens;
    mine.out = static_cast<uint8_t*>(p.out) + static_cast<int64_t>(m0) * p.N * (p.out_dtype == IRIS_F32 ? 4 : 2);
    constexpr int SHARE = T / 2;
    if (warp >= 2) store_columns(mine, lanes + half * SHARE, half * SHARE, SHARE, n, ok);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(s->tmem_base, COLS);
    return;
  }
  const int own = T / p.splits, log_own = __ffs(own) - 1;  // columns of a CTA: a power of two, 2 at least
  if (p.splits > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (warp >= 2 && !half) {
    uint32_t r[16];
    tmem_ld16(lanes, r);
    tmem_wait_ld();
#pragma unroll
    for (int col = 0; col < 16; ++col) {
      const uint32_t to = map_to_cta(parts + (part * own + (col & (own - 1))) * BN + quarter * 32 + lane,
                                     static_cast<uint32_t>(col >> log_own));
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(r[col]) : "memory");
    }
  }
  if (warp >= 2 && !ok && lane < p.splits) {
    const uint32_t to = map_to_cta(&s->bad[part], static_cast<uint32_t>(lane));
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(1) : "memory");
  }
  if (p.splits > 1) cluster_sync();
  else __syncthreads();
  if (warp >= 2) {
    bool bad = false;
    for (int i = 0; i < p.splits; ++i) bad = bad || s->bad[i] != 0;
#pragma unroll 1
    for (int c = half; c < own; c += 2) {
      const int m = part * own + c;
      if (m >= p.M) break;
      int sum = 0;
#pragma unroll 2
      for (int i = 0; i < p.splits; ++i) sum += parts[(i * own + c) * BN + quarter * 32 + lane];
      if (n < p.N) store_out(p, static_cast<int64_t>(m) * p.N + n, bad ? NAN : scaled(sum, s->scale[m], my_scale, my_bias));
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(s->tmem_base, COLS);
}

template <typename V, int T, bool ALIGNED>
int launch_few_as(const CUtensorMap& tw, Params p, int splits, const void* x, int64_t ldx, cudaStream_t st) {
  auto kernel = few_kernel<V, T, ALIGNED>;
  static bool configured[64] = {false};
  int dev = 0;
  IRIS_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !configured[dev]) {
    IRIS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, few::SMEM));
    if (dev < 64) configured[dev] = true;
  }
  p.token_tiles = (p.M + T - 1) / T;
  p.splits = splits;
  const int64_t ctas = static_cast<int64_t>(p.token_tiles) * ((p.N + BN - 1) / BN) * splits;
  IRIS_REQUIRE(ctas < (1ll << 31), "gemm_i8: too many rows");
  IRIS_CUDA(launch_early(kernel, dim3(static_cast<unsigned>(ctas)), THREADS, few::SMEM, st, static_cast<unsigned>(splits), tw, p,
                         static_cast<const V*>(x), ldx));
  return IRIS_OK;
}

template <typename V>
int launch_few(const CUtensorMap& tw, const Params& p, int tokens, int splits, const void* x, int64_t ldx, cudaStream_t st) {
  const bool aligned = aligned16(x) && (p.M <= 1 || ldx * static_cast<int64_t>(sizeof(V)) % 16 == 0);
  switch (tokens + aligned) {
    case 16: return launch_few_as<V, 16, false>(tw, p, splits, x, ldx, st);
    case 17: return launch_few_as<V, 16, true>(tw, p, splits, x, ldx, st);
    case 32: return launch_few_as<V, 32, false>(tw, p, 1, x, ldx, st);
    case 33: return launch_few_as<V, 32, true>(tw, p, 1, x, ldx, st);
    case 64: return launch_few_as<V, 64, false>(tw, p, 1, x, ldx, st);
    case 65: return launch_few_as<V, 64, true>(tw, p, 1, x, ldx, st);
    case 128: return launch_few_as<V, 128, false>(tw, p, 1, x, ldx, st);
    default: return launch_few_as<V, 128, true>(tw, p, 1, x, ldx, st);
  }
}

// ---------------------------------------------------------------- many tokens
// CTA pairs (cta_group::2), persistent: a cluster of two CTAs on paired SMs computes 256
// weight rows by up to 256 tokens. Each CTA brings its own 128 weight rows and half of the
// tokens' rows by TMA, 256 wide in k (two slabs) into a three-stage ring; both CTAs' copies complete
// on the leader's barrier. The leader's MMA thread issues tcgen05.mma.cta_group::2, which
// leaves each CTA's 128 rows by all tokens in that CTA's TMEM, twice: the next tile's
// products run under the epilogue. The tile's tokens (a multiple of 32) follow M, so that
// the last tile is not mostly padding.
namespace pair {
constexpr int STAGES = 3, SLABS = 2;
constexpr int W_BYTES = 128 * SLAB, X_BYTES = 128 * SLAB;  // of a slab, at most
constexpr int STAGE = SLABS * (W_BYTES + X_BYTES);
constexpr int GROUP = 16;  // neighbouring tiles: 16 of weight rows share their tokens, then tokens go on
struct Smem {
  uint64_t full[STAGES];  // used in the leader only: both CTAs' copies complete here
  uint64_t empty[STAGES];
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];  // used in the leader only: both CTAs' epilogue warps
  uint64_t teardown;
  uint32_t tmem_base;
  int abort;
};
constexpr int SMEM = 1024 + STAGES * STAGE + static_cast<int>(sizeof(Smem));
static_assert(SMEM <= 232448, "pair kernel shared memory");

struct Tile {
  int nb, mb;
};
IRIS_DEVICE Tile locate(int t, int num_n, int num_m) {
  const int group = t / (GROUP * num_m), first = group * GROUP;
  const int in_group = t - group * GROUP * num_m, wide = min(GROUP, num_n - first);
  return Tile{first + in_group % wide, in_group / wide};
}
IRIS_DEVICE void umma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
}  // namespace pair

__global__ void __launch_bounds__(THREADS, 1)
    pair_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tx,
                const __grid_constant__ Params p, int tokens) {
  using namespace pair;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  pair::Smem* s = reinterpret_cast<pair::Smem*>(ring + STAGES * STAGE);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const int rank = static_cast<int>(cluster_ctarank());
  const bool leader = rank == 0;
  const int pair_id = static_cast<int>(blockIdx.x / 2), pairs = static_cast<int>(gridDim.x / 2);
  const int num_n = (p.N + 255) / 256, num_m = (p.M + tokens - 1) / tokens, tiles = num_n * num_m;
  const int slabs = (p.K + SLAB - 1) / SLAB, steps = (slabs + SLABS - 1) / SLABS;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&s->full[i], 1);
      mbar_init(&s->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s->tmem_full[i], 1);
      mbar_init(&s->tmem_empty[i], 2 * EPILOGUE);
    }
    mbar_init(&s->teardown, 1);
    s->abort = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tw);
    tma_prefetch_desc(&tx);
  }
  cluster_sync();  // every barrier of both CTAs exists before any remote arrival
  volatile int* abort = &s->abort;
  grid_wait();
  if (warp == 1) {
    tmem_alloc_pair(&s->tmem_base, 512);  // after the wait and before the successor, as in rows_kernel
    grid_trigger();
  }
  // both CTAs' TMEM before any product; the producers go on meanwhile
  tc_fence_before();
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  if (warp != 0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&s->tmem_base);

  if (warp == 0) {
    // ------------------------------------------------------------ producer (both CTAs)
    if (lane == 0) {
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      const int half = tokens / 2;
      for (int t = pair_id; t < tiles && ok; t += pairs) {
        const Tile tl = locate(t, num_n, num_m);
        for (int step = 0; step < steps; ++step) {
          if (!mbar_wait(&s->empty[stage], phase ^ 1u, abort)) {
            ok = false;
            break;
          }
          const uint32_t full_leader = map_to_cta(&s->full[stage], 0);
          const int n = min(SLABS, slabs - step * SLABS);
          if (leader) mbar_arrive_expect_tx(&s->full[stage], 2 * n * (W_BYTES + half * SLAB));
          for (int i = 0; i < n; ++i) {
            const int k = (step * SLABS + i) * SLAB;
            tma_load_2d_pair(&tw, full_leader, ring + stage * STAGE + i * W_BYTES, k, tl.nb * 256 + rank * 128);
            tma_load_2d_pair(&tx, full_leader, ring + stage * STAGE + SLABS * W_BYTES + i * X_BYTES, k, tl.mb * tokens + rank * half);
          }
          ++issued;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok && issued > 0) {
        // the loads in flight target both CTAs' shared memory: give them time to land
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 1000000ull) {
        }
      }
    }
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader)
    if (lane == 0 && leader) {
      const uint32_t idesc = idesc_i8(256, tokens);
      int stage = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = pair_id; t < tiles && ok; t += pairs, ++it) {
        const int acc = it & 1;
        if (!mbar_wait_cluster(&s->tmem_empty[acc], static_cast<uint32_t>((it >> 1) & 1) ^ 1u, abort)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem + static_cast<uint32_t>(acc * 256);
        for (int step = 0; step < steps; ++step) {
          if (!mbar_wait(&s->full[stage], phase, abort)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const int n = min(SLABS, slabs - step * SLABS);
          for (int i = 0; i < n; ++i) {
            const uint32_t w_addr = smem_addr(ring + stage * STAGE + i * W_BYTES);
            const uint32_t x_addr = smem_addr(ring + stage * STAGE + SLABS * W_BYTES + i * X_BYTES);
#pragma unroll
            for (int k = 0; k < SLAB / 32; ++k)
              umma_i8_pair(d_tmem, umma_desc(w_addr + k * 32, 16, 1024, kLayoutSw128), umma_desc(x_addr + k * 32, 16, 1024, kLayoutSw128),
                           idesc, (step | i | k) != 0 ? 1u : 0u);
          }
          umma_commit_pair(map_to_cta(&s->empty[stage], 0));
          umma_commit_pair(map_to_cta(&s->empty[stage], 1));
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok) {
          umma_commit_pair(map_to_cta(&s->tmem_full[acc], 0));
          umma_commit_pair(map_to_cta(&s->tmem_full[acc], 1));
        }
      }
      umma_commit_pair(map_to_cta(&s->teardown, 0));
      int dummy = 0;
      mbar_wait(&s->teardown, 0, &dummy);
    }
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int quarter = warp & 3, first = warp >= 6 ? tokens / 2 : 0;
    const uint32_t empty_leader = map_to_cta(&s->tmem_empty[0], 0);
    int it = 0;
    bool ok = true;  // a wait gave up: NaN rather than wrong values
    for (int t = pair_id; t < tiles; t += pairs, ++it) {
      const Tile tl = locate(t, num_n, num_m);
      const int acc = it & 1;
      ok = ok && __all_sync(0xffffffffu, mbar_wait_cluster(&s->tmem_full[acc], static_cast<uint32_t>((it >> 1) & 1), abort));
      tc_fence_after();
      const int n = tl.nb * 256 + rank * 128 + quarter * 32 + lane;
      store_columns(p, tmem + static_cast<uint32_t>(acc * 256 + first) + (static_cast<uint32_t>(quarter * 32) << 16), tl.mb * tokens + first,
                    tokens / 2, n, ok);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(empty_leader + static_cast<uint32_t>(acc) * 8u);
    }
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync();  // no CTA leaves while the other may still address its barriers or TMEM
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

// Not every SM has a partner SM that a cluster of two can use: the persistent grid has the
// clusters that are resident at once.
int resident_pairs(int* pairs) {
  static int cache[64] = {0};
  int dev = 0;
  IRIS_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || cache[dev] == 0) {
    IRIS_CUDA(cudaFuncSetAttribute(pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, pair::SMEM));
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(num_sms() / 2 * 2));
    config.blockDim = dim3(THREADS);
    config.dynamicSmemBytes = pair::SMEM;
    config.attrs = &attr;
    config.numAttrs = 1;
    IRIS_CUDA(cudaOccupancyMaxActiveClusters(pairs, pair_kernel, &config));
    IRIS_REQUIRE(*pairs > 0, "gemm_i8: no CTA pair fits on this device");
    if (dev < 64) cache[dev] = *pairs;
    return IRIS_OK;
  }
  *pairs = cache[dev];
  return IRIS_OK;
}

// Tokens of a tile: as few tiles as 256 gives, evenly filled.
inline int pair_tokens(int64_t M) {
  const int64_t tiles = (M + 255) / 256;
  return static_cast<int>(((M + tiles - 1) / tiles + 31) / 32 * 32);
}

int launch_pair(const void* w, int64_t ldw, const void* x, int64_t ldx, const Params& p, cudaStream_t st) {
  const int tokens = pair_tokens(p.M);
  CUtensorMap tw, tx;
  IRIS_CHECK_STATUS(make_tmap_2d_bytes(&tw, w, p.K, p.N, ldw, SLAB, 128));
  IRIS_CHECK_STATUS(make_tmap_2d_bytes(&tx, x, p.K, p.M, ldx, SLAB, tokens / 2));
  int pairs = 0;
  IRIS_CHECK_STATUS(resident_pairs(&pairs));
  const int64_t tiles = static_cast<int64_t>((p.N + 255) / 256) * ((p.M + tokens - 1) / tokens);
  IRIS_REQUIRE(tiles < (1ll << 30), "gemm_i8: too many tiles");
  IRIS_CUDA(launch_early(pair_kernel, dim3(static_cast<unsigned>(2 * std::min<int64_t>(tiles, pairs))), THREADS, pair::SMEM, st, 2, tw, tx,
                         p, tokens));
  return IRIS_OK;
}

// ------------------------------------------------------------------- which form
// By an estimate of its time in us. A rows_kernel CTA of T tokens takes START and, for each
// of its slabs, what its ring of stages gives (SLAB_US alone on its SM; two on one PAIRED times
// that, DEEP_SLAB of it for a deep ring), the weights' bytes HBM_RATE or L2_RATE at most; parts of K
// cost their exchange; an SM's second CTA begins SECOND later. A pair's tile takes its tokens'
// products. Measured, us, (tokens, K -> N): 64, 2560 -> 2560: T 64 deep in 4 parts 7.0, T 32 in 4
// parts 7.9, T 64 whole 8.7, pair 9.2; 16, 8192 -> 8192: 4 parts 10.2, deep 2 parts 11.6,
// whole 19.7; 256, 8192 -> 8192: T 128 deep 20.6, T 64 23.8, T 128 24.4, pair 25.6; 1024, 2560 ->
// 2560: T 128 13.3, pair 13.7; 301, 2560 -> 15360: pair 18.1, T 128 21.7; 64, 8192 -> 32768: T 64
// 49, deep 52, pair 53.
struct Choice {
  int tokens, splits;  // 0 tokens: CTA pairs
  bool deep;
};

Choice choose(int64_t M, int64_t N, int64_t K) {
  constexpr float START = 2.6f, START_TOKEN = 0.0115f, SLAB_US = 0.24f, SLAB_TOKEN = 0.0006f, HBM_RATE = 6.3e6f, L2_RATE = 9.0e6f;
  constexpr int64_t IN_L2 = 96 << 20;  // weights that L2 may hold from the last step
  constexpr float EXCHANGE = 0.3f, EXCHANGE_TOKEN = 0.024f, SECOND = 1.2f, DEEP_SLAB = 0.85f, DEEP_HBM = 1.07f, PAIRED = 1.45f;
  constexpr float PAIR_START = 6.3f, PAIR_TILE = 1.2f, PAIR_SLAB = 0.08f, PAIR_TOKEN = 0.0009f;
  const int64_t sms = num_sms(), slabs = (K + SLAB - 1) / SLAB, wide = (N + BN - 1) / BN;
  const int64_t per = pair_tokens(M), tiles = (M + per - 1) / per * ((N + 255) / 256), waves = (tiles + sms / 2 - 1) / (sms / 2);
  Choice best = {0, 1, false};
  if (waves > 4) return best;
  const float hbm = N * K / (N * K > IN_L2 ? HBM_RATE : L2_RATE);
  float least = PAIR_START + std::max(hbm, waves * (PAIR_TILE + slabs * (PAIR_SLAB + PAIR_TOKEN * per)));
  for (int T = 16; T <= 128 && T < 2 * M + 16; T *= 2) {
    const int64_t units = (M + T - 1) / T * wide;
    if (units > 4 * sms) continue;
    const float start = START + START_TOKEN * T, slab = SLAB_US + SLAB_TOKEN * T;
    for (int splits = 1; splits <= 8 && splits <= slabs; splits *= 2) {
      const int64_t ctas = units * splits, mine = (slabs + splits - 1) / splits;
      const float exchange = splits > 1 ? EXCHANGE + EXCHANGE_TOKEN * T : 0.f;
      for (int deep = 0; deep < 2; ++deep) {
        const int64_t slots = deep ? sms : 2 * sms, turns = (ctas + slots - 1) / slots;
        const float each = mine * slab * (deep ? DEEP_SLAB : ctas > sms ? PAIRED : 1.f);
        // an SM's second CTA starts when the first has its TMEM, which is after the wait for the predecessor
        const float late = !deep && ctas > sms ? SECOND : 0.f;
        const float t = start + exchange + late + std::max(deep ? DEEP_HBM * hbm : hbm, turns * each + (turns - 1) * (start + exchange - 1.f));
        if (t < least) least = t, best = Choice{T, splits, deep != 0};
      }
    }
  }
  return best;
}

// The tokens of few_kernel's tile that takes a call's rows; 0: two launches do, `c` being the
// product's form. us of graph replays over weights that come from memory, one launch against
// two (rows x K -> N, bf16 unless said):
//  - short rows: 1 x 16 -> 2560 3.0 / 3.9, 16 x 128 -> 2560 3.3 / 3.7, 128 x 40 -> 2560 3.3 / 4.4. T 32 where its
//    tiles have an SM each, 33 x 128 -> 9000 3.6 / 4.4 (T 64 4.5); T 64, 128 x 80 -> 6848 4.6 / 5.2 (T 32 5.2, T 128
//    6.4), 64 x 128 -> 15360 4.8 / 5.0 (T 32 5.1), -> 40000 9.5 / 8.8, 64 x 80 -> 70000 11.4 / 13.7; T 128, 128 x 80
//    -> 15360 6.5 / 7.5 (T 64 6.6), 128 x 128 -> 15360 7.4 / 6.1, 128 x 40 -> 40000 12.6 / 13.2 (T 64 13.7), 128 x 64
//    -> 40000 13.1 / 11.4.
//  - K in parts: 1 x 2560 -> 2560 5.6 / 7.2, 4 x 2560 -> 2560 6.4 / 7.3, 8 x 1280 -> 2560 5.8 / 6.4; 10 KB a CTA
//    level: fp32, 1 x 10240 -> 2560 11.8 / 11.9. Few long rows cost the rounding kernel most: fp32, 1 x 10240
//    -> 256 8.1 / 9.2, 3 x 3000 -> 256 6.5 / 6.3, 4 x 2560 -> 2560 7.5 / 7.3.
//  - K whole: 5 KB a CTA about level (4 x 640 -> 2560 5.6 / 5.3; fp32 5.8 / 5.2; 8 x 640 6.0 / 5.2). CTAs in
//    turn: 4 x 640 -> 40000 13.1 / 10.4, 1 x 1280 -> 70000 18.6 / 19.4; where the product would have a
//    deep ring, one CTA an SM, in three turns, 3 x 1280 -> 40000 17.7 / 20.6.
inline int few_tokens(const iris_i8_problem& q, const Choice& c) {
  if (q.x_dtype == IRIS_I8 || q.M > few::MOST_TOKENS) return 0;
  const int64_t row = q.K * (q.x_dtype == IRIS_F32 ? 4 : 2), wide = (q.N + BN - 1) / BN, sms = num_sms();
  if (row <= few::SHORT_ROW) {
    if (q.M <= 32 || (q.M + 31) / 32 * wide <= sms) return 32;
    const int tokens = q.M <= 64 || 2 * wide <= sms ? 64 : 128;
    const bool resident = (q.M + tokens - 1) / tokens * wide <= 2 * sms;
    return row <= (tokens == 64 ? resident ? few::SHORT_ROW : 192 : resident ? 192 : 96) ? tokens : 0;
  }
  if (q.M > few::MOST_ROWS || c.tokens != 16 || (q.M - 1) * row > 20480) return 0;
  const int64_t slabs = (q.K + SLAB - 1) / SLAB, part = q.M * row / c.splits;
  const int64_t most = c.splits > 1 ? 10240 : q.M > 4 ? 0 : wide <= 2 * sms ? 5120 : c.deep ? 10240 : 4096;
  return part <= most && (slabs + c.splits - 1) / c.splits <= few::most_slabs(16) ? 16 : 0;
}

inline int check_rows(int64_t M, int64_t K, int64_t ldx) {
  IRIS_REQUIRE(M >= 0 && M < (1ll << 31) - 256 && K >= 1 && K <= 131071, "quantize_i8: M rows of 1 to 131071 values");
  IRIS_REQUIRE(ldx >= 0, "quantize_i8: the row stride must not be negative");
  return IRIS_OK;
}

inline int64_t row_bytes(int64_t K) { return (K + 15) / 16 * 16; }
inline int64_t workspace_bytes(const iris_i8_problem& q) {
  return q.x_dtype == IRIS_I8 ? 0 : q.M * row_bytes(q.K) + (q.M + 3) / 4 * 16;
}

inline int launch_quantize_any(const QuantizeParams& p, int64_t dtype, cudaStream_t st) {
  return dtype == IRIS_F32 ? quantize<float>(p, st) : dtype == IRIS_BF16 ? quantize<__nv_bfloat16>(p, st) : quantize<__half>(p, st);
}

int check_product(const iris_i8_problem& q) {
  IRIS_REQUIRE(q.x_dtype >= IRIS_F32 && q.x_dtype <= IRIS_I8 && q.out_dtype >= IRIS_F32 && q.out_dtype <= IRIS_F16,
               "gemm_i8: unsupported dtype");
  IRIS_REQUIRE(q.M >= 0 && q.M < (1ll << 31) - 256 && q.N >= 0 && q.N < (1ll << 31) - 256, "gemm_i8: sizes");
  IRIS_REQUIRE(q.K >= 1 && q.K <= 131071, "gemm_i8: 1 <= K <= 131071 (longer sums could leave int32)");
  return IRIS_OK;
}

}  // namespace i8
}  // namespace iris

using namespace iris;

extern "C" int iris_quantize_i8(const iris_quantize_problem* q, void* stream) {
  using namespace iris::i8;
  IRIS_REQUIRE(q != nullptr, "quantize_i8: null pointer");
  IRIS_REQUIRE(q->x_dtype >= IRIS_F32 && q->x_dtype <= IRIS_F16, "quantize_i8: unsupported dtype");
  IRIS_CHECK_STATUS(check_rows(q->M, q->K, q->ldx));
  IRIS_REQUIRE(q->ldq >= q->K && q->ldq % 8 == 0, "quantize_i8: rows of q at multiples of 8 bytes, at least K");
  if (q->M == 0) return IRIS_OK;
  IRIS_REQUIRE(q->x && q->q && q->scale, "quantize_i8: null pointer");
  IRIS_REQUIRE(aligned_n(q->q, 8) && aligned_n(q->scale, 4) && aligned_n(q->x, q->x_dtype == IRIS_F32 ? 4 : 2),
               "quantize_i8: misaligned pointer");
  const QuantizeParams p = {q->x, static_cast<int8_t*>(q->q), q->scale, q->ldx, q->ldq, static_cast<int>(q->M),
                            static_cast<int>(q->K)};
  return launch_quantize_any(p, q->x_dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int iris_gemm_i8_workspace(const iris_i8_problem* q, int64_t* bytes) {
  using namespace iris::i8;
  IRIS_REQUIRE(q != nullptr && bytes != nullptr, "gemm_i8_workspace: null pointer");
  IRIS_CHECK_STATUS(check_product(*q));
  *bytes = q->M * q->N == 0 || few_tokens(*q, choose(q->M, q->N, q->K)) != 0 ? 0 : workspace_bytes(*q);
  return IRIS_OK;
}

extern "C" int iris_gemm_i8(const iris_i8_problem* q, void* stream) {
  using namespace iris::i8;
  IRIS_REQUIRE(q != nullptr, "gemm_i8: null pointer");
  IRIS_CHECK_STATUS(check_product(*q));
  if (q->M == 0 || q->N == 0) return IRIS_OK;
  const bool fresh = q->x_dtype != IRIS_I8;
  IRIS_REQUIRE(q->x && q->w && q->w_scale && q->out && (fresh || q->x_scale), "gemm_i8: null pointer");
  IRIS_REQUIRE(aligned16(q->w) && q->ldw % 16 == 0 && q->ldw >= q->K, "gemm_i8: weight rows at multiples of 16 bytes");
  IRIS_REQUIRE(aligned_n(q->w_scale, 4) && aligned_n(q->bias, 4) && aligned_n(q->x_scale, 4) &&
                   aligned_n(q->out, q->out_dtype == IRIS_F32 ? 4 : 2) && aligned_n(q->x, q->x_dtype == IRIS_F32 ? 4 : fresh ? 2 : 1),
               "gemm_i8: misaligned pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const void* x = q->x;
  int64_t ldx = q->ldx;
  Params p = {};
  p.x_scale = q->x_scale;
  p.w_scale = q->w_scale, p.bias = q->bias, p.out = q->out;
  p.M = static_cast<int>(q->M), p.N = static_cast<int>(q->N), p.K = static_cast<int>(q->K);
  p.out_dtype = static_cast<int>(q->out_dtype);
  const Choice c = choose(p.M, p.N, p.K);
  CUtensorMap tw, tx;
  if (fresh) {
    IRIS_CHECK_STATUS(check_rows(q->M, q->K, q->ldx));
    if (const int tokens = few_tokens(*q, c)) {
      IRIS_CHECK_STATUS(make_tmap_2d_bytes(&tw, q->w, q->K, q->N, q->ldw, SLAB, BN));
      return q->x_dtype == IRIS_F32    ? launch_few<float>(tw, p, tokens, c.splits, x, ldx, st)
             : q->x_dtype == IRIS_BF16 ? launch_few<__nv_bfloat16>(tw, p, tokens, c.splits, x, ldx, st)
                                       : launch_few<__half>(tw, p, tokens, c.splits, x, ldx, st);
    }
    IRIS_REQUIRE(q->workspace && aligned16(q->workspace) && q->workspace_bytes >= workspace_bytes(*q), "gemm_i8: workspace too small");
    ldx = row_bytes(q->K);
    float* scale = reinterpret_cast<float*>(static_cast<uint8_t*>(q->workspace) + q->M * ldx);
    const QuantizeParams rows = {q->x, static_cast<int8_t*>(q->workspace), scale, q->ldx, ldx, static_cast<int>(q->M),
                                 static_cast<int>(q->K)};
    IRIS_CHECK_STATUS(launch_quantize_any(rows, q->x_dtype, st));
    x = q->workspace;
    p.x_scale = scale;
  } else {
    if (q->M == 1) ldx = row_bytes(q->K);  // a lone row's stride says nothing
    IRIS_REQUIRE(aligned16(x) && ldx % 16 == 0 && ldx >= q->K, "gemm_i8: 8-bit rows of x at multiples of 16 bytes");
  }
  p.early = fresh;
  if (c.tokens == 0) return launch_pair(q->w, q->ldw, x, ldx, p, st);
  IRIS_CHECK_STATUS(make_tmap_2d_bytes(&tw, q->w, q->K, q->N, q->ldw, SLAB, BN));
  IRIS_CHECK_STATUS(make_tmap_2d_bytes(&tx, x, q->K, q->M, ldx, SLAB, c.tokens));
  switch (c.tokens + c.deep) {
    case 16: return launch_rows<16, false>(tw, tx, p, c.splits, st);
    case 32: return launch_rows<32, false>(tw, tx, p, c.splits, st);
    case 64: return launch_rows<64, false>(tw, tx, p, c.splits, st);
    case 128: return launch_rows<128, false>(tw, tx, p, c.splits, st);
    case 17: return launch_rows<16, true>(tw, tx, p, c.splits, st);
    case 33: return launch_rows<32, true>(tw, tx, p, c.splits, st);
    case 65: return launch_rows<64, true>(tw, tx, p, c.splits, st);
    default: return launch_rows<128, true>(tw, tx, p, c.splits, st);
  }
}
