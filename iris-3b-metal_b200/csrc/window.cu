// Attention with a window and first tokens that stay visible, for a text side's
// prompts, chunks and single tokens over a cache (the denoiser's own attention,
// attention.cu, is unmasked). Query i of sample b is at position p = starts[b] + i;
// it sees key j < lengths[b] where j <= p + right and (j >= p - left or j < sinks):
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j,   0 where no key is visible.
// A row's visible keys are two runs, [0, early) and [lo, hi) (struct Span).
#include <math.h>

#include <algorithm>

#include "attend.cuh"
#include "iris_abi_internal.h"

namespace iris {
namespace window {
using namespace attend;

struct Params {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  int64_t qb, qh, qn, kb, kh, kn, vb, vh, vn, ob, on;  // element strides of batch, head, token
  int batch, heads_q, heads_kv, n, n_kv;
  const int* starts;   // null: n_kv - n
  const int* lengths;  // null: n_kv
  int64_t left, right;  // kNoBound: none
  int sinks;
  float scale_log2;
};

constexpr int64_t kNoBound = 1ll << 40;

// Visible keys of one query: [0, early) and [lo, hi).
struct Span {
  int early, lo, hi;
  IRIS_DEVICE int count() const { return early + hi - lo; }
  IRIS_DEVICE int key(int c) const { return c < early ? c : lo + (c - early); }
};

IRIS_DEVICE int sample_length(const Params& p, int b) {
  return p.lengths ? max(0, min(p.lengths[b], p.n_kv)) : p.n_kv;
}
IRIS_DEVICE int64_t sample_start(const Params& p, int b) { return p.starts ? p.starts[b] : p.n_kv - p.n; }

IRIS_DEVICE Span visible(const Params& p, int64_t pos, int length) {
  Span s;
  s.hi = static_cast<int>(max(int64_t(0), min(int64_t(length), pos + p.right + 1)));
  s.lo = static_cast<int>(max(int64_t(0), min(int64_t(s.hi), pos - p.left)));
  s.early = min(p.sinks, s.lo);
  return s;
}

// One output row by one warp, keys 32 at a time (a lane scores one), from global
// memory: columns [64 c + 2 lane, + 2) of chunk c < D / 64. Only visible keys are
// read, so what lies in masked places cannot reach the row. The row is kept as the
// mean so far, for sums over values near the end of bf16's range would leave fp32, where
// the result does not.
template <typename T, int D>
__device__ __noinline__ void attend_row(const Params& p, int b, int h, int i, float2 (&acc)[D / 64]) {
  const int lane = threadIdx.x & 31;
  const int hk = h / (p.heads_q / p.heads_kv);
  const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) + b * p.qb + h * p.qh + i * p.qn);
  const T* k = reinterpret_cast<const T*>(p.k) + b * p.kb + hk * p.kh;
  const T* v = reinterpret_cast<const T*>(p.v) + b * p.vb + hk * p.vh;
  const Span s = visible(p, sample_start(p, b) + i, sample_length(p, b));
  // f16 products stay far below fp32's end, bf16's only once they are scaled
  const float first = IsHalf<T>::value ? 1.f : p.scale_log2, then = IsHalf<T>::value ? p.scale_log2 : 1.f;
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int c = 0; c < D / 64; ++c) acc[c] = make_float2(0.f, 0.f);
  const int count = s.count();
  for (int c0 = 0; c0 < count; c0 += 32) {
    const bool real = c0 + lane < count;
    float dot = 0.f;
    if (real) {
      const uint4* kr = reinterpret_cast<const uint4*>(k + static_cast<int64_t>(s.key(c0 + lane)) * p.kn);
      for (int d = 0; d < D / 8; ++d) {
        const uint4 a = q[d], e = kr[d];
        const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float2 f = unpack2<T>(x[u]), g = unpack2<T>(y[u]);
          dot = fmaf(f.x * first, g.x, fmaf(f.y * first, g.y, dot));
        }
      }
    }
    const float score = real ? dot * then : -INFINITY;
    float top = score;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float m_new = fmaxf(m, top);
    const float base = m_new == -INFINITY ? 0.f : m_new;  // nothing above -inf so far: every weight 0
    float w = real ? exp2f(score - base) : 0.f;
    const float before = m == -INFINITY ? 0.f : l * exp2f(m - base);
    l = before + warp_sum(w);
    m = m_new;
    const float inv = l == 0.f ? 0.f : 1.f / l, keep = before * inv;
    w *= inv;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) acc[c] = make_float2(acc[c].x * keep, acc[c].y * keep);
    const int keys = min(32, count - c0);
    for (int j = 0; j < keys; ++j) {
      const float wj = __shfl_sync(0xffffffffu, w, j);
      const T* vr = v + static_cast<int64_t>(s.key(c0 + j)) * p.vn + 2 * lane;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const float2 f = unpack2<T>(*reinterpret_cast<const uint32_t*>(vr + 64 * c));
        acc[c] = make_float2(fmaf(wj, f.x, acc[c].x), fmaf(wj, f.y, acc[c].y));
      }
    }
  }
  // every visible score -inf: 0 / 0, as softmax has it
#pragma unroll
  for (int c = 0; c < D / 64; ++c)
    acc[c] = count == 0 ? make_float2(0.f, 0.f) : l == 0.f ? make_float2(NAN, NAN) : acc[c];
}

// ------------------------------------------------------------- tensor cores
// Prompts and chunks on the 5th-generation tensor cores: a CTA takes 128 query rows of
// one head, S, P and O in TMEM, over the blocks of 64 keys that some row sees (the blocks
// of the first `sinks` keys, then the window's), two CTAs to an SM. Warp 0 brings Q once
// and K and V through two-slot rings by TMA; warp 1 issues the MMAs; warps 2 to 5 do
// the softmax, a thread per row (TMEM lane), its 64 scores in registers: no exchange
// between threads. Exponentials (2048 a quarter and block at 4 a clock) take as long as
// the MMAs, so what costs is waiting: S alternates between two buffers and runs a block
// ahead of P V, so that a block's scores are there when the softmax of the one before
// ends, and the other CTA fills what waits are left (its start and its epilogue too).
//
// A block that every row of a warp sees in full takes no mask; others get one bit per
// key from the row's span. Keys behind the sample's length are zeroed in shared
// memory (their K only reaches masked scores), so cache rows never written cost
// nothing. A masked key's weight is exactly 0, and 0 times a NaN or infinity of
// its V row is NaN: a row that comes out not finite is computed again by attend_row,
// which reads visible keys alone (also rows that see no key: 0 / 0 here).
//
// Measured, 128 wide, FLOP of visible pairs: 16384 tokens, 20 over 5 heads, window 1024
// 205 us (0.82 PFLOP/s; 239 inside long runs under the power cap), 2 x 4352 f16 rows of
// 24 heads, 512 to each side 154 us (0.82; 180 in long runs); 8192 tokens 1.0 unmasked, 1.12 causal. Tensor
// pipe and exponentials 45% busy each: a block takes a warp about 1730 cycles, 870 of them
// weights, 320 the wait for S. Two row tiles a CTA 281 us, one tile with 128-key blocks
// 262, eight softmax warps 465 (registers spill), a part of the exponentials as
// polynomials 213 to 219, against 204 in the same runs.
constexpr int BQ = 128, BKV = 64, KV = 2;  // rows, keys of a block, slots of the K and V rings
constexpr int TILE_THREADS = 192;
constexpr int Q_HALF = BQ * 128, KV_HALF = BKV * 128;  // bytes of 64 columns of a tile
constexpr uint32_t COL_S = 0, COL_O = 2 * BKV, TILE_COLS = 256;

struct TileSmem {
  uint64_t q_full, k_full[KV], k_free[KV], v_full[KV], v_free[KV], v_tail;
  uint64_t s_full[2], p_full[2], pv_done, o_final, teardown;
  uint32_t tmem_base;
  int abort;
};

template <int D>
constexpr int tile_smem() {
  return 1024 + (D / 64) * (Q_HALF + 2 * KV * KV_HALF) + static_cast<int>(sizeof(TileSmem));
}

// Key blocks that rows at positions [pos, pos + rows) see: [0, early) and [lo, hi).
struct Blocks {
  int early, lo, hi;
  IRIS_DEVICE int count() const { return early + hi - lo; }
  IRIS_DEVICE int at(int it) const { return it < early ? it : lo + it - early; }
};

IRIS_DEVICE Blocks key_blocks(const Params& p, int64_t pos, int rows, int length) {
  // lo, hi and early grow with the row
  const Span first = visible(p, pos, length), last = visible(p, pos + rows - 1, length);
  Blocks x;
  x.early = (last.early + BKV - 1) / BKV;
  x.lo = first.lo / BKV;
  x.hi = (last.hi + BKV - 1) / BKV;
  if (last.hi <= first.lo) x.lo = x.hi = x.early;
  x.early = min(x.early, x.lo);
  return x;
}

template <typename T, int D>
__global__ void __launch_bounds__(TILE_THREADS, 2)
    tiles_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                 const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap to,
                 const __grid_constant__ Params p) {
  constexpr int HALVES = D / 64, KV_BYTES = HALVES * KV_HALF;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* q_tile = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* k_tile = q_tile + HALVES * Q_HALF;
  uint8_t* v_tile = k_tile + KV * KV_BYTES;
  TileSmem* s = reinterpret_cast<TileSmem*>(v_tile + KV * KV_BYTES);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  // later rows first: under a causal mask they see the most keys
  const int per_row = p.heads_q * p.batch;
  const int row0 = (static_cast<int>(gridDim.x / per_row) - 1 - static_cast<int>(blockIdx.x / per_row)) * BQ;
  const int b = blockIdx.x % per_row / p.heads_q, h = blockIdx.x % p.heads_q;
  const int hk = h / (p.heads_q / p.heads_kv);
  grid_wait();
  const int length = sample_length(p, b);
  const int64_t start = sample_start(p, b);
  const Blocks blocks = key_blocks(p, start + row0, min(BQ, p.n - row0), length);
  const int iters = blocks.count();

  if (threadIdx.x == 0) {
    mbar_init(&s->q_full, 1);
    for (int i = 0; i < KV; ++i) {
      mbar_init(&s->k_full[i], 1);
      mbar_init(&s->k_free[i], 1);
      mbar_init(&s->v_full[i], 1);
      mbar_init(&s->v_free[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s->s_full[i], 1);
      mbar_init(&s->p_full[i], 4);
    }
    mbar_init(&s->pv_done, 1);
    mbar_init(&s->o_final, 1);
    mbar_init(&s->v_tail, 1);
    mbar_init(&s->teardown, 1);
    s->abort = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&s->tmem_base, TILE_COLS);
    grid_trigger();  // behind TMEM: a successor that takes some could keep a CTA from ever getting its own
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s->tmem_base;
  volatile int* abort = &s->abort;

  if (warp == 0) {
    // ----------------------------------------------------------------- TMA
    const int kb = p.kb != 0 ? b : 0, kh = p.kh != 0 ? hk : 0;
    const int vb = p.vb != 0 ? b : 0, vh = p.vh != 0 ? hk : 0;
    int issued_k[KV], issued_v[KV];
    for (int i = 0; i < KV; ++i) issued_k[i] = issued_v[i] = -1;
    bool tail_issued = false;
    bool ok = true;
    if (lane == 0 && iters > 0) {
      tma_prefetch_desc(&tk);
      tma_prefetch_desc(&tv);
      mbar_arrive_expect_tx(&s->q_full, HALVES * Q_HALF);
      for (int c = 0; c < HALVES; ++c)
        tma_load_4d(&tq, &s->q_full, q_tile + c * Q_HALF, c * 64, row0, p.qh != 0 ? h : 0, p.qb != 0 ? b : 0);
    }
    auto load_k = [&](int it) {
      const int st = it % KV;
      const uint32_t ph = static_cast<uint32_t>((it / KV) & 1);
      ok = mbar_wait(&s->k_free[st], ph ^ 1u, abort);
      if (!ok) return;
      mbar_arrive_expect_tx(&s->k_full[st], KV_BYTES);
      for (int c = 0; c < HALVES; ++c)
        tma_load_4d(&tk, &s->k_full[st], k_tile + st * KV_BYTES + c * KV_HALF, c * 64, blocks.at(it) * BKV, kh, kb);
      issued_k[st] = static_cast<int>(ph);
    };
    if (lane == 0 && iters > 0) load_k(0);
    for (int it = 0; it < iters; ++it) {
      const int st = it % KV;
      const uint32_t ph = static_cast<uint32_t>((it / KV) & 1);
      const int key = blocks.at(it) * BKV;
      // keys behind the length that the tensor map does not end before
      const bool tail = key + BKV > length && length < p.n_kv;
      if (lane == 0 && ok) {
        if (it + 1 < iters) load_k(it + 1);  // scores run a block ahead
        ok = ok && mbar_wait(&s->v_free[st], ph ^ 1u, abort);
        if (ok) {
          uint64_t* bar = tail ? &s->v_tail : &s->v_full[st];
          mbar_arrive_expect_tx(bar, KV_BYTES);
          for (int c = 0; c < HALVES; ++c)
            tma_load_4d(&tv, bar, v_tile + st * KV_BYTES + c * KV_HALF, c * 64, key, vh, vb);
          tail_issued = tail_issued || tail;
          issued_v[st] = tail ? -1 : static_cast<int>(ph);  // the copy before in this slot has been read
        }
      }
      if (!__shfl_sync(0xffffffffu, ok, 0)) break;
      if (tail) {  // one block of the CTA at most: the one that the length ends in
        ok = __all_sync(0xffffffffu, mbar_wait(&s->v_tail, 0, abort));
        if (!ok) break;
        for (int e = (length - key) * 8 + lane; e < BKV * 8; e += 32)
          for (int c = 0; c < HALVES; ++c)
            *reinterpret_cast<uint4*>(v_tile + st * KV_BYTES + c * KV_HALF + e * 16) = make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s->v_full[st]);
      }
    }
    if (lane == 0 && iters > 0) {  // whichever warp gives up: no copy may land after the CTA is gone
      int dummy = 0;
      mbar_wait(&s->q_full, 0, &dummy);
      for (int i = 0; i < KV; ++i) {
        if (issued_k[i] >= 0) mbar_wait(&s->k_full[i], static_cast<uint32_t>(issued_k[i]), &dummy);
        if (issued_v[i] >= 0) mbar_wait(&s->v_full[i], static_cast<uint32_t>(issued_v[i]), &dummy);
      }
      if (tail_issued) mbar_wait(&s->v_tail, 0, &dummy);
    }
  } else if (warp == 1) {
    // ----------------------------------------------------------------- MMA
    if (lane == 0 && iters > 0) {
      constexpr uint32_t f16 = (1u << 7) | (1u << 10);  // the BF16 bits of idesc_bf16_f32; F16 is 0
      constexpr uint32_t clear = IsHalf<T>::value ? f16 : 0u;
      const uint32_t idesc_s = idesc_bf16_f32(BQ, BKV) & ~clear;
      const uint32_t idesc_o = idesc_bf16_f32(BQ, D, false, true) & ~clear;  // V is MN-major (columns contiguous)
      bool ok = mbar_wait(&s->q_full, 0, abort);
      // scores of block `it` into buffer it % 2
      auto issue_s = [&](int it) {
        ok = ok && mbar_wait(&s->k_full[it % KV], static_cast<uint32_t>((it / KV) & 1), abort);
        if (!ok) return;
        tc_fence_after();
        const uint32_t q_addr = smem_addr(q_tile), k_addr = smem_addr(k_tile + (it % KV) * KV_BYTES);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_ss(tmem + COL_S + (it & 1) * BKV, umma_desc(q_addr + (kk >> 2) * Q_HALF + (kk & 3) * 32, 16, 1024, kLayoutSw128),
                  umma_desc(k_addr + (kk >> 2) * KV_HALF + (kk & 3) * 32, 16, 1024, kLayoutSw128), idesc_s, kk > 0 ? 1u : 0u);
        umma_commit(&s->s_full[it & 1]);
        umma_commit(&s->k_free[it % KV]);
      };
      issue_s(0);
      if (iters > 1) issue_s(1);
      for (int it = 0; it < iters && ok; ++it) {
        const int st = it % KV;
        ok = mbar_wait(&s->v_full[st], static_cast<uint32_t>((it / KV) & 1), abort) &&
             mbar_wait(&s->p_full[it & 1], static_cast<uint32_t>((it >> 1) & 1), abort);
        if (!ok) break;
        tc_fence_after();
        const uint32_t v_addr = smem_addr(v_tile + st * KV_BYTES);
#pragma unroll
        for (int kk = 0; kk < BKV / 16; ++kk)  // P lies packed over the first half of its scores
          umma_ts(tmem + COL_O, tmem + COL_S + (it & 1) * BKV + kk * 8,
                  umma_desc(v_addr + kk * 16 * 128, KV_HALF, 1024, kLayoutSw128), idesc_o, (it > 0 || kk > 0) ? 1u : 0u);
        umma_commit(&s->pv_done);
        umma_commit(&s->v_free[st]);
        // into the buffer of the P just read: one thread's MMAs run in order
        if (it + 2 < iters) issue_s(it + 2);
      }
      if (ok) umma_commit(&s->o_final);
      umma_commit(&s->teardown);
      int dummy = 0;
      mbar_wait(&s->teardown, 0, &dummy);
    }
  } else {
    // ------------------------------------------------------------- softmax
    const int quarter = warp & 3;
    const int i = row0 + quarter * 32 + lane;  // query row
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const Span span = visible(p, start + i, length);
    // what every row of the warp sees: keys below hi_all that are sinks or from lo_all on
    const int hi_all = __shfl_sync(0xffffffffu, span.hi, 0), lo_all = __shfl_sync(0xffffffffu, span.lo, 31);
    float m_run = -INFINITY, l_run = 0.f;
    bool ok = true;
    for (int it = 0; it < iters; ++it) {
      const int key0 = blocks.at(it) * BKV;
      const bool full = key0 + BKV <= hi_all && (key0 >= lo_all || key0 + BKV <= p.sinks);
      const uint32_t s_at = lanes + COL_S + (it & 1) * BKV;
      ok = __all_sync(0xffffffffu, mbar_wait(&s->s_full[it & 1], static_cast<uint32_t>((it >> 1) & 1), abort));
      if (!ok) break;
      tc_fence_after();
      uint32_t r[2][32];
      tmem_ld32(s_at, r[0]);
      tmem_ld32(s_at + 32, r[1]);
      tmem_wait_ld();
      if (!full) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int k0 = key0 + c * 32;
          const uint32_t see = low_bits(span.hi - k0) & (~low_bits(span.lo - k0) | low_bits(p.sinks - k0));
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!(see >> e & 1u)) r[c][e] = __float_as_uint(-INFINITY);
        }
      }
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 32; e += 2)
          top[e / 2 % 4] = max3(top[e / 2 % 4], __uint_as_float(r[c][e]), __uint_as_float(r[c][e + 1]));
      const float mx = fmaxf(max3(top[0], top[1], top[2]), top[3]) * p.scale_log2;
      // the maximum is kept until a row exceeds it by 2^8 (O and l share it: exact); a row
      // that has seen nothing yet (-inf) has weights and sums of 0
      const bool grow = mx > m_run + RESCALE;
      const float m_new = grow ? mx : m_run;
      const bool rescale = grow && m_run != -INFINITY;
      if (__any_sync(0xffffffffu, rescale)) {
        const float corr = rescale ? ex2(m_run - m_new) : 1.f;
        l_run *= corr;
        ok = __all_sync(0xffffffffu, mbar_wait(&s->pv_done, static_cast<uint32_t>((it - 1) & 1), abort));
        if (!ok) break;
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < D / 16; ++c) {
          uint32_t o[16];
          tmem_ld16(lanes + COL_O + c * 16, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
          tmem_st16(lanes + COL_O + c * 16, o);
        }
      }
      m_run = m_new;
      // weights 2^(s * scale - m), rounded once to the operand type of the P V product:
      // the tensor cores take 16 bits, and the remainders would be a second product beside
      // two that already share the pipe. The rounding is relative to each weight and
      // averages out over the keys (bf16 rows 0.0020-0.0023 off the 64-bit ones, 0.0016 with
      // fp32 weights); the sum takes the fp32 values. Masked keys give exact zeros
      const float shift = m_new == -INFINITY ? 0.f : -m_new;
      const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), shift2 = make_float2(shift, shift);
      float2 sum2 = make_float2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float2 x =
              __ffma2_rn(make_float2(__uint_as_float(r[c][2 * e]), __uint_as_float(r[c][2 * e + 1])), scale2, shift2);
          const float2 w = make_float2(ex2(x.x), ex2(x.y));
          sum2 = __fadd2_rn(sum2, w);
          pk[e] = pack2<T>(w.x, w.y);
        }
        tmem_st16(s_at + c * 16, pk);
      }
      l_run += sum2.x + sum2.y;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s->p_full[it & 1]);
    }
    if (iters > 0) ok = ok && __all_sync(0xffffffffu, mbar_wait(&s->o_final, 0, abort));
    ok = ok && *abort == 0;
    T* out = reinterpret_cast<T*>(p.out) + b * p.ob + static_cast<int64_t>(h) * D;
    if (!ok) {  // a wait gave up (device error word): NaN rather than a wrong row
      if (i < p.n)
        for (int c = 0; c < D; c += 2) *reinterpret_cast<uint32_t*>(out + i * p.on + c) = pack2<T>(NAN, NAN);
    } else {
      tc_fence_after();
      const float inv = 1.f / l_run;
      bool finite = true;
      // the rows into Q's place (every score is computed), in the store's swizzle
      auto place = [&](int row, int piece) { return row * 128 + ((piece ^ (row & 7)) * 16); };
      const int row = quarter * 32 + lane;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t r[32];
        if (iters > 0) {
          tmem_ld32(lanes + COL_O + c * 32, r);
          tmem_wait_ld();
        }
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float a = iters > 0 ? __uint_as_float(r[2 * e]) * inv : 0.f;
          const float z = iters > 0 ? __uint_as_float(r[2 * e + 1]) * inv : 0.f;
          finite = finite && isfinite(a) && isfinite(z);
          pk[e] = pack2<T>(a, z);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<uint4*>(q_tile + (c >> 1) * Q_HALF + place(row, (c & 1) * 4 + e)) =
              make_uint4(pk[4 * e], pk[4 * e + 1], pk[4 * e + 2], pk[4 * e + 3]);
      }
      __syncwarp();  // a row that is computed again comes after what was written of it
      for (uint32_t again = __ballot_sync(0xffffffffu, !finite && i < p.n); again != 0; again &= again - 1) {
        const int r = quarter * 32 + __ffs(again) - 1;
        float2 acc[D / 64];
        attend_row<T, D>(p, b, h, row0 + r, acc);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          *reinterpret_cast<uint32_t*>(q_tile + c * Q_HALF + place(r, lane >> 2) + (lane & 3) * 4) = pack2<T>(acc[c].x, acc[c].y);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0 && row0 + quarter * 32 < p.n) {  // rows from n on are not written
        for (int c = 0; c < HALVES; ++c)
          tma_store_4d(&to, q_tile + c * Q_HALF + quarter * 32 * 128, c * 64, row0 + quarter * 32, h, p.ob != 0 ? b : 0);
        tma_store_wait();
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, TILE_COLS);
}

template <typename T, int D>
int launch_tiles(const Params& p, int dtype, cudaStream_t st) {
  const int64_t ctas = static_cast<int64_t>((p.n + BQ - 1) / BQ) * p.heads_q * p.batch;
  IRIS_REQUIRE(ctas < (1ll << 31), "window_attn_fwd: too many rows");
  CUtensorMap tq, tk, tv, to;
  IRIS_CHECK_STATUS(make_tmap_heads(&tq, p.q, dtype, D, p.n, p.heads_q, p.batch, p.qn, p.qh, p.qb, BQ));
  IRIS_CHECK_STATUS(make_tmap_heads(&tk, p.k, dtype, D, p.n_kv, p.heads_kv, p.batch, p.kn, p.kh, p.kb, BKV));
  IRIS_CHECK_STATUS(make_tmap_heads(&tv, p.v, dtype, D, p.n_kv, p.heads_kv, p.batch, p.vn, p.vh, p.vb, BKV));
  IRIS_CHECK_STATUS(make_tmap_heads(&to, p.out, dtype, D, p.n, p.heads_q, p.batch, p.on, D, p.ob, 32));
  auto kernel = tiles_kernel<T, D>;
  static bool configured[64] = {false};
  int dev = 0;
  IRIS_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !configured[dev]) {
    IRIS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, tile_smem<D>()));
    if (dev < 64) configured[dev] = true;
  }
  IRIS_CUDA(launch_early(kernel, dim3(static_cast<unsigned>(ctas)), TILE_THREADS, tile_smem<D>(), st, 1, tq, tk, tv, to, p));
  return IRIS_OK;
}

// ------------------------------------------------- few rows over many keys
// Single tokens and short chunks: the keys are split over CTAs and the parts joined.
// A CTA takes 16 query rows (the tokens' query heads of one key head, so K and V are
// read once for all of them) and a chunk of the keys that some of them sees; its
// warps walk 16-key tiles of their own, each with its own softmax state and its own
// ring of cp.async copies (no barrier until the end), scores and P V on mma.sync
// m16n8k16: HBM-bound, one K and V byte is used for 16 rows at most, which leaves the
// 5th-generation tensor cores' 128-row tiles seven eighths empty. Chunks are the same
// length for every sample, so samples of different lengths give equal work. Up to
// eight chunks are a cluster's CTAs: each stores its rows' states into the shared
// memory of the CTA that owns the row, which joins them: one launch, nothing in global
// memory. More chunks are joined by a second kernel.
//
// Measured, one token, 128 wide: 16 samples of 21400 keys on average, 32768 at most, 32
// over 8 heads 217 us (6.45 TB/s, 0.98 of a plain copy; 1280 keys a chunk instead of
// 2560: 220, 512: 239); one sample, 20 over 5 heads: 64 keys 3.7 us, 256 4.6,
// 1028 6.5 (each CTA reading the others' states at the end, scores in one chain of mmas:
// 8.1 us, and 228 us the long caches), 65536 keys 34 (4.9 TB/s). Six ring slots instead
// of three 5.6 us at 64 keys and 9.6 at 1028; eight warps a CTA slower on long caches.
constexpr int STEP_WARPS = 4, STEP_STAGES = 3, STEP_KEYS = 16, STEP_ROWS = 16;

struct Split {
  int row_tiles;  // 16-row tiles of a key head's query rows
  int chunk;      // keys per CTA
  int splits;     // chunks of the longest list
  bool cluster;   // the chunks of a row tile are a cluster
  float* parts;   // else [batch, heads_kv, row_tiles, splits, 16, D] sums, then [.., 16] maxima and totals; null: one chunk
};

constexpr int MOST_CLUSTER = 8;
// Rows that a cluster's CTA owns, and places for the states of all chunks of them.
IRIS_DEVICE int rows_owned(int splits) { return (STEP_ROWS + splits - 1) / splits; }
constexpr int STATES = STEP_ROWS + MOST_CLUSTER;  // at least splits * rows_owned(splits)

template <int D>
constexpr int STEP_RINGS = STEP_WARPS * STEP_STAGES * 2 * STEP_KEYS * D * 2;  // bytes
template <int D>
constexpr int step_smem() {
  return STEP_RINGS<D> + STATES * (D + 2) * 4;
}

// Writes row (b, h, i), columns [64 c + 2 lane, + 2); rows that are not finite again
// from visible keys alone (a masked key's V may be NaN or infinite: 0 times it is NaN).
template <typename T, int D>
IRIS_DEVICE void finish_row(const Params& p, int b, int h, int i, float2 (&acc)[D / 64], float total) {
  const float inv = 1.f / total;
  bool finite = true;
#pragma unroll
  for (int c = 0; c < D / 64; ++c) {
    acc[c] = make_float2(acc[c].x * inv, acc[c].y * inv);
    finite = finite && isfinite(acc[c].x) && isfinite(acc[c].y);
  }
  if (!__all_sync(0xffffffffu, finite)) attend_row<T, D>(p, b, h, i, acc);
  T* o = reinterpret_cast<T*>(p.out) + b * p.ob + i * p.on + static_cast<int64_t>(h) * D + 2 * (threadIdx.x & 31);
#pragma unroll
  for (int c = 0; c < D / 64; ++c) *reinterpret_cast<uint32_t*>(o + 64 * c) = pack2<T>(acc[c].x, acc[c].y);
}

template <typename T, int D>
__global__ void __launch_bounds__(STEP_WARPS * 32) step_kernel(const __grid_constant__ Params p,
                                                               const __grid_constant__ Split sp) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  constexpr int TILE = STEP_KEYS * D * 2;  // bytes of one K or V tile
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (sp.cluster) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  grid_wait();
  grid_trigger();
  const int split = static_cast<int>(blockIdx.x % sp.splits);
  const int unit = static_cast<int>(blockIdx.x / sp.splits);  // (b, hk, row tile)
  const int rt = unit % sp.row_tiles, hk = unit / sp.row_tiles % p.heads_kv, b = unit / sp.row_tiles / p.heads_kv;
  const int group = p.heads_q / p.heads_kv;
  const int rows = p.n * group;  // of this key head: row r is token r / group, head hk * group + r % group
  const int r0 = rt * STEP_ROWS, r_last = min(r0 + STEP_ROWS, rows) - 1;
  const int length = sample_length(p, b);
  const int64_t start = sample_start(p, b);
  // keys that some row of the tile sees: [0, early) and [lo, hi)
  const Span first = visible(p, start + r0 / group, length), last = visible(p, start + r_last / group, length);
  Span all = last;
  all.lo = first.lo;
  all.early = min(last.early, first.lo);
  const bool same = r0 / group == r_last / group;  // one token: every row sees all of them
  const int count = all.early + max(0, all.hi - all.lo);
  const int c_begin = min(split * sp.chunk, count), c_end = min(c_begin + sp.chunk, count);

  const T* k = reinterpret_cast<const T*>(p.k) + b * p.kb + hk * p.kh;
  const T* v = reinterpret_cast<const T*>(p.v) + b * p.vb + hk * p.vh;
  const uint32_t ring = smem_addr(smem_raw) + warp * (STEP_STAGES * 2 * TILE);
  const int tiles = (c_end - c_begin + STEP_KEYS - 1) / STEP_KEYS;
  const int mine = tiles > warp ? (tiles - warp + STEP_WARPS - 1) / STEP_WARPS : 0;
  // tile t of the warp into its slot: rows of D / 8 16-byte pieces, piece x of row r at x ^ (r & 7)
  constexpr int PIECES = D / 8;
  auto load = [&](int t) {
    if (t < mine) {
      const int c0 = c_begin + (warp + t * STEP_WARPS) * STEP_KEYS;
      const uint32_t slot = ring + (t % STEP_STAGES) * 2 * TILE;
#pragma unroll
      for (int e = 0; e < STEP_KEYS * PIECES / 32; ++e) {
        const int at = e * 32 + lane, r = at / PIECES, x = at % PIECES;
        const bool real = c0 + r < c_end;
        const int64_t key = real ? all.key(c0 + r) : 0;
        const uint32_t dst = slot + r * (D * 2) + ((x ^ (r & 7)) * 16);
        copy16(dst, k + (real ? key * p.kn + x * 8 : 0), real);
        copy16(dst + TILE, v + (real ? key * p.vn + x * 8 : 0), real);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int t = 0; t < STEP_STAGES - 1; ++t) load(t);

  // Q rows as the A operand: this lane's rows g and g + 8, columns 2 (lane % 4) + {0, 1} of each 8
  const int g = lane >> 2, quad = lane & 3;
  uint32_t qa[D / 16][4];
  Span seen[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int r = r0 + g + 8 * u;
    const int i = min(r, rows - 1) / group, h = hk * group + min(r, rows - 1) % group;
    seen[u] = visible(p, start + i, length);
    const T* q = reinterpret_cast<const T*>(p.q) + b * p.qb + h * p.qh + static_cast<int64_t>(i) * p.qn + 2 * quad;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      qa[d][u] = *reinterpret_cast<const uint32_t*>(q + 16 * d);
      qa[d][u + 2] = *reinterpret_cast<const uint32_t*>(q + 16 * d + 8);
    }
  }
  float o[D / 8][4];
#pragma unroll
  for (int d = 0; d < D / 8; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[d][e] = 0.f;
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};

  for (int t = 0; t < mine; ++t) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STEP_STAGES - 2) : "memory");
    __syncwarp();  // every lane's copies of the tile have landed; the slot refilled next was read by all
    load(t + STEP_STAGES - 1);
    const uint32_t slot = ring + (t % STEP_STAGES) * 2 * TILE;
    const int c0 = c_begin + (warp + t * STEP_WARPS) * STEP_KEYS;
    // S: keys [8 j, 8 j + 8) in s[j]
    float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}, odd[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int d = 0; d < D / 32; ++d) {  // two k steps per load: pieces 4 d .. 4 d + 3 of the 8 key rows
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t kb[4];
        const int r = 8 * j + (lane & 7), x = 4 * d + (lane >> 3);
        ldmatrix4(kb, slot + r * (D * 2) + ((x ^ (r & 7)) * 16));
        mma_16816<T>(s[j], qa[2 * d], kb[0], kb[1]);
        mma_16816<T>(odd[j], qa[2 * d + 1], kb[2], kb[3]);  // two chains: half the wait for the last
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[j][e] += odd[j][e];
    if (!same || c0 + STEP_KEYS > c_end) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = c0 + 8 * j + 2 * quad + (e & 1);
          const Span& w = seen[e >> 1];
          const int key = all.key(c);
          if (c >= c_end || key >= w.hi || (key < w.lo && key >= p.sinks)) s[j][e] = -INFINITY;
        }
    }
    bool rescale = false;
    float corr[2], shift[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float mx = fmaxf(fmaxf(s[0][2 * u], s[0][2 * u + 1]), fmaxf(s[1][2 * u], s[1][2 * u + 1])) * p.scale_log2;
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const bool grow = mx > m_run[u] + RESCALE;
      const float m_new = grow ? mx : m_run[u];
      corr[u] = grow && m_run[u] != -INFINITY ? ex2(m_run[u] - m_new) : 1.f;
      rescale = rescale || corr[u] != 1.f;
      m_run[u] = m_new;
      shift[u] = m_new == -INFINITY ? 0.f : -m_new;
    }
    if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
      for (int d = 0; d < D / 8; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][e] *= corr[e >> 1];
      l_run[0] *= corr[0];
      l_run[1] *= corr[1];
    }
    // weights, rounded once to the operand type (the fp32 values go into the totals): as in
    // tiles_kernel, so that a row is as accurate in either form
    uint32_t pa[4];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float w0 = ex2(fmaf(s[j][2 * u], p.scale_log2, shift[u]));
        const float w1 = ex2(fmaf(s[j][2 * u + 1], p.scale_log2, shift[u]));
        l_run[u] += w0 + w1;
        pa[2 * j + u] = pack2<T>(w0, w1);
      }
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {  // 16 columns per load: key rows 0-7 and 8-15, pieces 2 d and 2 d + 1
      uint32_t vb[4];
      const int r = lane & 15, x = 2 * d + (lane >> 4);
      ldmatrix4_trans(vb, slot + TILE + r * (D * 2) + ((x ^ (r & 7)) * 16));
      mma_16816<T>(o[2 * d], pa, vb[0], vb[1]);
      mma_16816<T>(o[2 * d + 1], pa, vb[2], vb[3]);
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    l_run[u] += __shfl_xor_sync(0xffffffffu, l_run[u], 1);
    l_run[u] += __shfl_xor_sync(0xffffffffu, l_run[u], 2);
  }
  // the warps' states, joined per row: warp w finishes rows w, w + 4, ...
  __syncthreads();  // the rings are done with
  float* sums = reinterpret_cast<float*>(smem_raw);  // [warp][16][D]
  __shared__ float tops[STEP_WARPS][STEP_ROWS], totals[STEP_WARPS][STEP_ROWS];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    float* dst = sums + (warp * STEP_ROWS + g + 8 * u) * D + 2 * quad;
#pragma unroll
    for (int d = 0; d < D / 8; ++d) *reinterpret_cast<float2*>(dst + 8 * d) = make_float2(o[d][2 * u], o[d][2 * u + 1]);
    if (quad == 0) {
      tops[warp][g + 8 * u] = m_run[u];
      totals[warp][g + 8 * u] = l_run[u];
    }
  }
  __syncthreads();
  // cluster: states [chunk][owned row], sums then {maximum, total}; other CTAs store here once all have begun
  float* states = reinterpret_cast<float*>(smem_raw + STEP_RINGS<D>);
  const int owned = rows_owned(sp.splits);
  if (sp.cluster) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  for (int r = warp; r <= r_last - r0; r += STEP_WARPS) {
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int w = 0; w < STEP_WARPS; ++w) top = fmaxf(top, tops[w][r]);
    float2 acc[D / 64];
#pragma unroll
    for (int c = 0; c < D / 64; ++c) acc[c] = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < STEP_WARPS; ++w) {
      // a warp that saw nothing has sums of 0 (or NaN, from a masked V: kept, it marks the row)
      const float f = tops[w][r] == -INFINITY ? 1.f : ex2(tops[w][r] - top);
      total += f * totals[w][r];
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const float2 x = *reinterpret_cast<const float2*>(sums + (w * STEP_ROWS + r) * D + 64 * c + 2 * lane);
        acc[c] = make_float2(fmaf(f, x.x, acc[c].x), fmaf(f, x.y, acc[c].y));
      }
    }
    if (sp.cluster) {
      float* at = states + (split * owned + r % owned) * (D + 2);
      const uint32_t to = map_to_cta(at, static_cast<uint32_t>(r / owned));
#pragma unroll
      for (int c = 0; c < D / 64; ++c) store_remote(to + 4 * (64 * c + 2 * lane), acc[c]);
      if (lane == 0) store_remote(to + 4 * D, make_float2(top, total));
    } else if (sp.parts == nullptr) {
      finish_row<T, D>(p, b, hk * group + (r0 + r) % group, (r0 + r) / group, acc, total);
    } else {
      const int64_t part = (static_cast<int64_t>(unit) * sp.splits + split) * STEP_ROWS + r;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) *reinterpret_cast<float2*>(sp.parts + part * D + 64 * c + 2 * lane) = acc[c];
      if (lane == 0) {
        const int64_t all_rows = static_cast<int64_t>(p.batch) * p.heads_kv * sp.row_tiles * sp.splits * STEP_ROWS;
        float2* state = reinterpret_cast<float2*>(sp.parts + all_rows * D);
        state[part] = make_float2(top, total);
      }
    }
  }
  if (sp.cluster) {
    cluster_sync();
    for (int local = warp; local < owned && split * owned + local <= r_last - r0; local += STEP_WARPS) {
      const int r = r0 + split * owned + local;
      float top = -INFINITY, total = 0.f;
      for (int q = 0; q < sp.splits; ++q) top = fmaxf(top, states[(q * owned + local) * (D + 2) + D]);
      float2 acc[D / 64];
#pragma unroll
      for (int c = 0; c < D / 64; ++c) acc[c] = make_float2(0.f, 0.f);
      for (int q = 0; q < sp.splits; ++q) {
        const float* from = states + (q * owned + local) * (D + 2);
        const float f = from[D] == -INFINITY ? 1.f : ex2(from[D] - top);
        total = fmaf(f, from[D + 1], total);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          const float2 x = *reinterpret_cast<const float2*>(from + 64 * c + 2 * lane);
          acc[c] = make_float2(fmaf(f, x.x, acc[c].x), fmaf(f, x.y, acc[c].y));
        }
      }
      finish_row<T, D>(p, b, hk * group + r % group, r / group, acc, total);
    }
  }
}

// One row's chunks joined by a block: its warps take every fourth chunk.
template <typename T, int D>
__global__ void __launch_bounds__(STEP_WARPS * 32) join_kernel(const __grid_constant__ Params p,
                                                               const __grid_constant__ Split sp) {
  __shared__ float2 sums[STEP_WARPS][D / 2];
  __shared__ float totals[STEP_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = p.heads_q / p.heads_kv, rows = p.n * group;
  const int unit_rows = static_cast<int>(blockIdx.x) / rows;  // (b, hk)
  const int row = static_cast<int>(blockIdx.x) - unit_rows * rows;
  const int64_t unit = static_cast<int64_t>(unit_rows) * sp.row_tiles + row / STEP_ROWS;
  const int64_t part0 = unit * sp.splits * STEP_ROWS + row % STEP_ROWS;
  const int64_t all_rows = static_cast<int64_t>(p.batch) * p.heads_kv * sp.row_tiles * sp.splits * STEP_ROWS;
  const float2* state = reinterpret_cast<const float2*>(sp.parts + all_rows * D);
  grid_wait();
  grid_trigger();
  float top = -INFINITY;
  for (int c = lane; c < sp.splits; c += 32) top = fmaxf(top, state[part0 + c * STEP_ROWS].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float total = 0.f;
  float2 acc[D / 64];
#pragma unroll
  for (int c = 0; c < D / 64; ++c) acc[c] = make_float2(0.f, 0.f);
#pragma unroll 4
  for (int c = warp; c < sp.splits; c += STEP_WARPS) {
    const int64_t part = part0 + static_cast<int64_t>(c) * STEP_ROWS;
    const float2 st = state[part];
    const float f = st.x == -INFINITY ? 1.f : ex2(st.x - top);
    total = fmaf(f, st.y, total);
#pragma unroll
    for (int d = 0; d < D / 64; ++d) {
      const float2 x = *reinterpret_cast<const float2*>(sp.parts + part * D + 64 * d + 2 * lane);
      acc[d] = make_float2(fmaf(f, x.x, acc[d].x), fmaf(f, x.y, acc[d].y));
    }
  }
#pragma unroll
  for (int d = 0; d < D / 64; ++d) sums[warp][32 * d + lane] = acc[d];
  if (lane == 0) totals[warp] = total;
  __syncthreads();
  if (warp != 0) return;
#pragma unroll
  for (int w = 1; w < STEP_WARPS; ++w) {
    total += totals[w];
#pragma unroll
    for (int d = 0; d < D / 64; ++d) {
      const float2 x = sums[w][32 * d + lane];
      acc[d] = make_float2(acc[d].x + x.x, acc[d].y + x.y);
    }
  }
  const int b = unit_rows / p.heads_kv, hk = unit_rows % p.heads_kv;
  finish_row<T, D>(p, b, hk * group + row % group, row / group, acc, total);
}

// Clusters of `size` step_kernel CTAs that run at once: GPCs hold whole clusters, so
// fewer CTAs than the SMs hold alone.
int64_t clusters_at_once(int size) {
  static int cache[64][MOST_CLUSTER + 1] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return num_sms() * 2 / size;
  if (cache[dev][size] == 0) {
    auto kernel = step_kernel<__nv_bfloat16, 128>;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(size);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(size));
    config.blockDim = dim3(STEP_WARPS * 32);
    config.dynamicSmemBytes = step_smem<128>();
    config.attrs = &attr;
    config.numAttrs = 1;
    int n = 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, step_smem<128>()) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kernel, &config) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = num_sms() * 2 / size;
    }
    cache[dev][size] = n;
  }
  return cache[dev][size];
}

// How a call's keys are split, or that whole 128-row tiles are the better form.
//
// Split: from a bound on the keys that a row tile sees. The CTAs that the SMs hold at
// once are a wave; w waves take about w times a chunk and a CTA's own time (CTA_KEYS),
// so the number of waves whose chunks waste least is taken, and more of them for
// several samples, whose lengths may differ, where that costs little and leaves long
// chunks. One token, 128 wide, us (chunks of one wave against six or against LONG_CHUNK
// alone): one sample, 5 key heads, 65536 keys 34 against 60 and 48; 4 samples, 8 key
// heads, 4096 keys 18.6 against 27 and 21.
// Tiles: a CTA walks its keys at TILE_NS each whatever rows it has, and starts and ends
// in the time of TILE_KEYS; a split CTA's keys take STEP_NS. One sample, 20 over 5 heads, 2048 keys, us split / tiles: 8 tokens 9.7 / 30,
// 128 tokens 43 / 32; 16384 keys: 64 tokens 110 / 216, 128 tokens 214 / 217.
constexpr int64_t STEP_WAVES = 6, STEP_CTAS = 2, LONG_CHUNK = 1024, SHORT_CHUNK = 192, CTA_KEYS = 96, JOIN_KEYS = 64;
constexpr int64_t STEP_NS = 25, TILE_NS = 13, TILE_KEYS = 288;

struct Sizes {
  int64_t batch, heads_q, heads_kv, n, n_kv, left, right, sinks;
};

bool split_keys(const Sizes& z, Split* sp) {
  const int64_t group = z.heads_q / z.heads_kv, slots = num_sms() * STEP_CTAS;
  auto span_of = [&](int64_t tokens) {  // keys that so many neighbouring rows see at most
    return z.left < kNoBound && z.right < kNoBound ? std::min(z.n_kv, z.left + z.right + tokens + z.sinks) : z.n_kv;
  };
  const int64_t row_tiles = (z.n * group + STEP_ROWS - 1) / STEP_ROWS, units = z.batch * z.heads_kv * row_tiles;
  const int64_t span = span_of(std::min(z.n, (STEP_ROWS - 1) / group + 2));
  constexpr int64_t unit = STEP_WARPS * STEP_KEYS;
  auto pieces = [&](int64_t splits) { return std::max(unit, ((span + splits - 1) / splits + unit - 1) / unit * unit); };
  auto cost_of = [&](int64_t chunk, int64_t waves) {
    const int64_t splits = (span + chunk - 1) / chunk;
    if (splits > MOST_CLUSTER) return waves * (chunk + CTA_KEYS) + JOIN_KEYS;
    if (splits > 1) waves = (units + clusters_at_once(static_cast<int>(splits)) - 1) / clusters_at_once(static_cast<int>(splits));
    return waves * (chunk + CTA_KEYS);
  };
  const int64_t first = (units + slots - 1) / slots;  // fewer waves do not hold every unit
  int64_t chunk = pieces(1), least = cost_of(chunk, first);
  auto consider = [&](int64_t c, int64_t waves) {
    const int64_t cost = cost_of(c, waves);
    if (cost < least || (z.batch > 1 && c < chunk && c >= LONG_CHUNK && cost < least + least / 12)) {
      chunk = c;
      least = std::min(least, cost);
    }
  };
  for (int64_t splits = 2; splits <= MOST_CLUSTER; ++splits) consider(pieces(splits), (units * splits + slots - 1) / slots);
  for (int64_t w = first; w < first + STEP_WAVES; ++w)
    if (w * slots / units > MOST_CLUSTER) consider(pieces(w * slots / units), w);
  // eight short chunks rather than more of them and a second launch
  if (span > MOST_CLUSTER * chunk && pieces(MOST_CLUSTER) <= SHORT_CHUNK) chunk = pieces(MOST_CLUSTER);
  sp->row_tiles = static_cast<int>(std::min<int64_t>(row_tiles, 1 << 30));
  sp->chunk = static_cast<int>(chunk);
  sp->splits = static_cast<int>(span > chunk ? (span + chunk - 1) / chunk : 1);
  sp->cluster = sp->splits > 1 && sp->splits <= MOST_CLUSTER;
  const int64_t tiles = z.batch * z.heads_q * ((z.n + BQ - 1) / BQ);
  const int64_t tile_cost = (tiles + slots - 1) / slots * (span_of(std::min<int64_t>(z.n, BQ)) + TILE_KEYS);
  return z.n_kv == 0 || least * STEP_NS < tile_cost * TILE_NS;
}

template <typename T, int D>
int launch_step(const Params& p, Split sp, float* parts, int64_t parts_bytes, cudaStream_t st) {
  const int64_t units = static_cast<int64_t>(p.batch) * p.heads_kv * sp.row_tiles;
  const int64_t rows = static_cast<int64_t>(p.batch) * p.heads_q * p.n;
  IRIS_REQUIRE(units * sp.splits < (1ll << 31) && rows < (1ll << 31), "window_attn_fwd: too many rows");
  if (sp.splits > 1 && !sp.cluster) {
    IRIS_REQUIRE(parts != nullptr && aligned16(parts) && parts_bytes >= units * sp.splits * STEP_ROWS * (D + 2) * 4,
                 "window_attn_fwd: workspace too small");
    sp.parts = parts;
  }
  auto kernel = step_kernel<T, D>;
  static bool configured[64] = {false};
  int dev = 0;
  IRIS_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !configured[dev]) {
    IRIS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, step_smem<D>()));
    if (dev < 64) configured[dev] = true;
  }
  IRIS_CUDA(launch_early(kernel, dim3(static_cast<unsigned>(units * sp.splits)), STEP_WARPS * 32, step_smem<D>(), st,
                         sp.cluster ? static_cast<unsigned>(sp.splits) : 1u, p, sp));
  if (sp.parts == nullptr) return IRIS_OK;
  IRIS_CUDA(launch_early(join_kernel<T, D>, dim3(static_cast<unsigned>(rows)), STEP_WARPS * 32, 0, st, 1, p, sp));
  return IRIS_OK;
}

template <typename T, int D>
int launch(const Params& p, int dtype, void* workspace, int64_t workspace_bytes, cudaStream_t st) {
  Split sp = {};
  if (split_keys(Sizes{p.batch, p.heads_q, p.heads_kv, p.n, p.n_kv, p.left, p.right, p.sinks}, &sp))
    return launch_step<T, D>(p, sp, static_cast<float*>(workspace), workspace_bytes, st);
  return launch_tiles<T, D>(p, dtype, st);
}

inline int64_t bound(int64_t v) { return v < 0 || v > kNoBound ? kNoBound : v; }

inline int check_sizes(const iris_window_problem& q) {
  IRIS_REQUIRE(q.dtype == IRIS_BF16 || q.dtype == IRIS_F16, "window_attn_fwd: bf16 or f16");
  IRIS_REQUIRE(q.head_dim == 64 || q.head_dim == 128, "window_attn_fwd: head_dim must be 64 or 128");
  IRIS_REQUIRE(q.heads_q > 0 && q.heads_kv > 0 && q.heads_q % q.heads_kv == 0,
               "window_attn_fwd: heads_q must be a positive multiple of heads_kv");
  IRIS_REQUIRE(q.batch >= 0 && q.n >= 0 && q.n_kv >= 0 && q.batch <= 65535 && q.heads_q <= 65535 &&
                   q.n < (1ll << 30) && q.n_kv < (1ll << 30),
               "window_attn_fwd: sizes");
  IRIS_REQUIRE(q.left >= -1 && q.right >= -1 && q.sinks >= 0, "window_attn_fwd: window bounds are -1 (none) or more");
  return IRIS_OK;
}

inline bool rows_aligned(const iris_head_rows& r) {
  return aligned16(r.data) && r.stride_b % 8 == 0 && r.stride_h % 8 == 0 && r.stride_n % 8 == 0;
}
inline bool rows_apart(const iris_head_rows& r, int64_t n) {
  return r.stride_b >= 0 && r.stride_h >= 0 && (n <= 1 || r.stride_n > 0);
}

}  // namespace window
}  // namespace iris

using namespace iris;

extern "C" int iris_window_attn_workspace(const iris_window_problem* q, int64_t* bytes) {
  using namespace iris::window;
  IRIS_REQUIRE(q != nullptr && bytes != nullptr, "window_attn_workspace: null pointer");
  IRIS_CHECK_STATUS(check_sizes(*q));
  *bytes = 0;
  if (q->batch * q->n == 0) return IRIS_OK;
  Split sp = {};
  if (split_keys(Sizes{q->batch, q->heads_q, q->heads_kv, q->n, q->n_kv, bound(q->left), bound(q->right),
                       std::min(q->sinks, q->n_kv)}, &sp) &&
      sp.splits > 1 && !sp.cluster)
    *bytes = q->batch * q->heads_kv * sp.row_tiles * sp.splits * STEP_ROWS * (q->head_dim + 2) * 4;
  return IRIS_OK;
}

extern "C" int iris_window_attn_fwd(const iris_window_problem* q, void* stream) {
  using namespace iris::window;
  IRIS_REQUIRE(q != nullptr, "window_attn_fwd: null pointer");
  IRIS_CHECK_STATUS(check_sizes(*q));
  const float scale = static_cast<float>(q->scale);
  // and so must its product with log2(e) be: 0 times infinity is NaN
  IRIS_REQUIRE(scale > 0.f && scale * 1.4426950408889634f < INFINITY, "window_attn_fwd: scale must be positive and finite");
  const iris_head_rows rows = used_strides(q->q, q->batch, q->heads_q, q->n);
  const iris_head_rows k = used_strides(q->k, q->batch, q->heads_kv, q->n_kv), v = used_strides(q->v, q->batch, q->heads_kv, q->n_kv);
  IRIS_REQUIRE(rows_aligned(rows) && rows_aligned(k) && rows_aligned(v) && aligned16(q->out) &&
                   q->out_stride_b % 8 == 0 && q->out_stride_n % 8 == 0,
               "window_attn_fwd: pointers and strides must be multiples of 16 bytes");
  IRIS_REQUIRE(rows_apart(rows, q->n) && rows_apart(k, q->n_kv) && rows_apart(v, q->n_kv),
               "window_attn_fwd: rows must not repeat along the tokens");
  if (q->batch * q->n == 0) return IRIS_OK;
  IRIS_REQUIRE(rows.data && q->out && ((k.data && v.data) || q->n_kv == 0), "window_attn_fwd: null pointer");
  Params p = {};
  p.q = rows.data, p.k = k.data, p.v = v.data, p.out = q->out;
  p.qb = rows.stride_b, p.qh = rows.stride_h, p.qn = rows.stride_n;
  p.kb = k.stride_b, p.kh = k.stride_h, p.kn = k.stride_n;
  p.vb = v.stride_b, p.vh = v.stride_h, p.vn = v.stride_n;
  p.ob = q->out_stride_b, p.on = q->out_stride_n;
  p.batch = static_cast<int>(q->batch), p.heads_q = static_cast<int>(q->heads_q);
  p.heads_kv = static_cast<int>(q->heads_kv), p.n = static_cast<int>(q->n), p.n_kv = static_cast<int>(q->n_kv);
  p.starts = q->starts, p.lengths = q->lengths;
  p.left = bound(q->left), p.right = bound(q->right);
  p.sinks = static_cast<int>(q->sinks < q->n_kv ? q->sinks : q->n_kv);
  p.scale_log2 = scale * 1.4426950408889634f;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int dtype = static_cast<int>(q->dtype);
  if (dtype == IRIS_BF16)
    return q->head_dim == 128 ? launch<__nv_bfloat16, 128>(p, dtype, q->workspace, q->workspace_bytes, st)
                              : launch<__nv_bfloat16, 64>(p, dtype, q->workspace, q->workspace_bytes, st);
  return q->head_dim == 128 ? launch<__half, 128>(p, dtype, q->workspace, q->workspace_bytes, st)
                            : launch<__half, 64>(p, dtype, q->workspace, q->workspace_bytes, st);
}
