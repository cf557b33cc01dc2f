// Attention of a batch whose samples share a long prefix: groups of batch / groups
// neighbouring samples have one prefix's keys and values in common and a cache of their
// own behind it. Query i of sample b (group g) sees the prefix's keys j < prefix_lengths[g]
// and its own keys j < lengths[b] with j <= starts[b] + i + right, in one softmax:
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j over both,   0 where no key is visible.
//
// The prefix is read once for a group: its rows, tokens times query heads of all samples, fill the
// 128-row tiles of the 5th-generation tensor cores (tile_cta), which split the prefix's keys
// between CTAs; a sample's own keys go by 8 or 16 rows (step_cta), and the parts are joined by their
// maxima and totals. Prompts, whose rows fill tiles by themselves, see all keys in one pass; few
// rows over a short prefix take all keys by step_cta. make_plan chooses.
//
// Measured in graph replays, 128 wide, caches full, us: one token of 4 samples behind 300 tokens, 20
// over 5 heads 4.9; of 32 behind 2048 with 512 of their own, 32 over 8 heads 16.4; of 64 behind 32768
// with 1024 80 (402 MB, 5.0 TB/s, 0.77 of a plain copy: the tiles' start, the uneven end and the join
// take the rest); 8 prompts of 300 behind 4096 113 (0.92 PFLOP/s; 131, 0.79, in long runs under the
// power cap); 2 x 1024 rows of 24 heads behind 16384 392 to 403 (1.1 PFLOP/s; 476, 0.92, in long runs).
#include <math.h>

#include <algorithm>

#include "attend.cuh"
#include "iris_abi_internal.h"

namespace iris {
namespace prefix {
using namespace attend;

struct Params {
  const void* q;
  const void* pk;
  const void* pv;
  const void* k;
  const void* v;
  void* out;
  int64_t qb, qh, qn, pkb, pkh, pkn, pvb, pvh, pvn, kb, kh, kn, vb, vh, vn, ob, on;  // element strides of batch, head, token
  int batch, per_group, heads_q, heads_kv, n, n_prefix, n_kv;
  const int* prefix_lengths;  // null: n_prefix
  const int* starts;          // null: n_kv - n
  const int* lengths;         // null: n_kv
  int64_t right;              // kNoBound: none
  float scale_log2;
};

constexpr int64_t kNoBound = 1ll << 40;

IRIS_DEVICE int prefix_length(const Params& p, int b) {
  return p.prefix_lengths ? max(0, min(p.prefix_lengths[b / p.per_group], p.n_prefix)) : p.n_prefix;
}
IRIS_DEVICE int own_length(const Params& p, int b) { return p.lengths ? max(0, min(p.lengths[b], p.n_kv)) : p.n_kv; }
IRIS_DEVICE int64_t own_start(const Params& p, int b) { return p.starts ? p.starts[b] : p.n_kv - p.n; }
// Own keys [0, n) that the query at position pos sees.
IRIS_DEVICE int own_keys(const Params& p, int64_t pos, int length) {
  return static_cast<int>(max(int64_t(0), min(int64_t(length), pos + p.right + 1)));
}

// One output row by one warp, keys 32 at a time (a lane scores one), from global
// memory: columns [64 c + 2 lane, + 2) of chunk c < D / 64. Only visible keys are
// read, so what lies in masked places cannot reach the row. The row is kept as the
// mean so far, for sums over values near the end of bf16's range would leave fp32, where
// the result does not.
template <typename T, int D>
__device__ __noinline__ void attend_row(const Params& p, int b, int h, int i, float2 (&acc)[D / 64]) {
  const int lane = threadIdx.x & 31;
  const int hk = h / (p.heads_q / p.heads_kv), g = b / p.per_group;
  const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) + b * p.qb + h * p.qh + i * p.qn);
  const T* pk = reinterpret_cast<const T*>(p.pk) + g * p.pkb + hk * p.pkh;
  const T* pv = reinterpret_cast<const T*>(p.pv) + g * p.pvb + hk * p.pvh;
  const T* k = reinterpret_cast<const T*>(p.k) + b * p.kb + hk * p.kh;
  const T* v = reinterpret_cast<const T*>(p.v) + b * p.vb + hk * p.vh;
  const int early = prefix_length(p, b);
  const int64_t count = early + static_cast<int64_t>(own_keys(p, own_start(p, b) + i, own_length(p, b)));
  // f16 products stay far below fp32's end, bf16's only once they are scaled
  const float first = IsHalf<T>::value ? 1.f : p.scale_log2, then = IsHalf<T>::value ? p.scale_log2 : 1.f;
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int c = 0; c < D / 64; ++c) acc[c] = make_float2(0.f, 0.f);
  for (int64_t c0 = 0; c0 < count; c0 += 32) {
    const bool real = c0 + lane < count;
    float dot = 0.f;
    if (real) {
      const int64_t c = c0 + lane;
      const uint4* kr = reinterpret_cast<const uint4*>(c < early ? pk + c * p.pkn : k + (c - early) * p.kn);
      for (int d = 0; d < D / 8; ++d) {
        const uint4 a = q[d], e = kr[d];
        const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float2 f = unpack2<T>(x[u]), w = unpack2<T>(y[u]);
          dot = fmaf(f.x * first, w.x, fmaf(f.y * first, w.y, dot));
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
    const int keys = static_cast<int>(min(int64_t(32), count - c0));
    for (int j = 0; j < keys; ++j) {
      const float wj = __shfl_sync(0xffffffffu, w, j);
      const int64_t c = c0 + j;
      const T* vr = (c < early ? pv + c * p.pvn : v + (c - early) * p.vn) + 2 * lane;
#pragma unroll
      for (int e = 0; e < D / 64; ++e) {
        const float2 f = unpack2<T>(*reinterpret_cast<const uint32_t*>(vr + 64 * e));
        acc[e] = make_float2(fmaf(wj, f.x, acc[e].x), fmaf(wj, f.y, acc[e].y));
      }
    }
  }
  // every visible score -inf: 0 / 0, as softmax has it
#pragma unroll
  for (int c = 0; c < D / 64; ++c)
    acc[c] = count == 0 ? make_float2(0.f, 0.f) : l == 0.f ? make_float2(NAN, NAN) : acc[c];
}

// -------------------------------------------------------- 128-row tiles (tcgen05)
// A tile is 128 query rows of one key head: tokens times query heads of `per` samples, row
// r being sample r / (n group), token r / group % n, head r % group. The prefix is the
// same for all samples of a group, so its rows are taken together (per = per_group): one
// token of 32 samples and 4 heads each fills a tile that would hold 4 rows. Where one
// sample's rows fill tiles (per = 1), they see its own keys too, in the same pass.
//
// A CTA takes a tile and a chunk of its blocks of 64 keys, two CTAs to an SM: warps 2 to 5
// bring Q's rows, which lie anywhere, into the swizzled place that the tensor cores read;
// warp 0 brings K and V through two-slot rings by TMA; warp 1 issues the MMAs; warps 2 to 5
// do the softmax, a thread per row (TMEM lane). S alternates between two buffers and runs a
// block ahead of P V. Chunks' states are joined by join_kernel.
//
// A block that every row of a warp sees in full takes no mask. Keys behind a length
// are zeroed in shared memory (their K only reaches masked scores). A masked key's weight is
// exactly 0, and 0 times a NaN or infinity of its V row is NaN: a row that comes out
// not finite is computed again by attend_row, which reads visible keys alone.
//
// A commit holds the tensor pipe for about 90 cycles before the next product (measured: 8 + 4
// products of a block 633 cycles, 989 with four commits), so a block has two: one
// barrier tells the softmax of its scores and the TMA warp of its slot of K, another of
// P V and its slot of V. (One for both tells of V's slot later: 114 -> 112 us where keys are in L2, 88 -> 97
// where they come from memory.)
//
// A block takes a CTA about 1800 cycles: 65 to 70% of them the tensor pipe, which two CTAs share (the
// scores' products read 6 KB of shared memory each, 49 cycles instead of 32), 55% the
// exponentials. Tried, 2 x 1024 rows behind 16384: weights by the maximum before the block's own is
// known, so that the exponentials need not wait for it, 489 -> 529 us; blocks brought into L2
// ahead of the rings 407 -> 425.
constexpr int BQ = 128, BKV = 64, KV = 2;  // rows, keys of a block, slots of the K and V rings
constexpr int THREADS = 192;
// Two CTAs to an SM: warp w of each sits in quarter w % 4 of the SM, whose registers hold
// four such warps (two of either CTA) at 128 each, not at the 168 that 2 x 192 threads would share
constexpr int BOUND_THREADS = 256;
constexpr int Q_HALF = BQ * 128, KV_HALF = BKV * 128;  // bytes of 64 columns of a tile
constexpr uint32_t COL_S = 0, COL_O = 2 * BKV, TILE_COLS = 256;

struct TileSmem {
  uint64_t q_full, k_full[KV], v_full[KV], v_tail;
  uint64_t s_full[2];   // block it's scores are there, and its slot of K is free: [it % 2]
  uint64_t p_full[2];
  uint64_t pv_done[2];  // block it's products are in O, and its slot of V is free
  uint64_t teardown;
  uint32_t tmem_base;
  int abort;
};

template <int D>
constexpr int tile_smem() {
  return 1024 + (D / 64) * (Q_HALF + 2 * KV * KV_HALF) + static_cast<int>(sizeof(TileSmem));
}

// ------------------------------------------------- few rows over many keys
// A sample's own keys where its rows fill no tile, and all of its keys where they are
// few: a CTA takes 8 or 16 query rows of a sample and key head (K and V are read once for all of
// them) and a chunk of the keys; its warps walk 16-key tiles of their own, each with its own
// softmax state and its own ring of cp.async copies (no barrier until the end). Scores and
// P V on mma.sync m16n8k16 with the keys, then the columns of V, as the 16-row operand: S^T = K
// Q^T, O^T = V^T P^T. So 8 rows (one token's query heads, mostly) need half the products and
// registers that a 16-row operand of queries would: HBM-bound where the keys are many.
constexpr int STEP_WARPS = 4, STEP_STAGES = 3, STEP_KEYS = 16;
constexpr int MOST_CLUSTER = 8;

// How a call is cut up.
struct Plan {
  int per;           // samples whose rows share tiles; 1: tiles see the samples' own keys too
  int units;         // of `per` samples and a key head
  int tiles;         // 128-row tiles of a unit
  int whole_tiles;   // the first tiles (all units') have one CTA each, which finishes their rows
  int tile_chunk;    // blocks of 64 keys that a CTA of the others walks
  int tile_splits;   // chunks of such a tile
  int tile_ctas;
  int row_tiles;     // tiles of 8 or 16 rows of a sample and key head
  int step_rows;     // 8 or 16
  int step_prefix;   // whether they see the prefix (no tiles do)
  int cluster;       // a row tile's chunks are a cluster and joined there (step_prefix alone)
  int step_chunk;    // keys of such a tile's CTA
  int step_splits;   // chunks; 0: tiles see all keys
  int step_ctas;
  float* tile_sums;  // [tile behind the whole ones, split, 128, D], then maxima and totals [.., 128]
  float2* tile_states;
  float* step_sums;  // [sample, key head, row tile, split, step_rows, D], then [.., step_rows]; null: rows are finished by their CTA
  float2* step_states;
};

template <int D>
constexpr int STEP_RINGS = STEP_WARPS * STEP_STAGES * 2 * STEP_KEYS * D * 2;  // bytes
// Rows that a cluster's CTA owns, and places behind the rings for the states of all chunks of them.
IRIS_DEVICE int rows_owned(int rows, int splits) { return (rows + splits - 1) / splits; }
template <int D>
constexpr int cluster_smem() {
  return STEP_RINGS<D> + (16 + MOST_CLUSTER) * (D + 2) * 4;  // at least splits * rows_owned(splits) of them
}
template <int D>
constexpr int most_smem() {
  return tile_smem<D>() > STEP_RINGS<D> ? tile_smem<D>() : STEP_RINGS<D>;
}

struct Row {
  int b, h, i;
};
// Row r of unit (u, hk).
IRIS_DEVICE Row row_of(const Params& p, int per, int u, int hk, int r) {
  const int group = p.heads_q / p.heads_kv;
  const int token = r / group;
  return Row{u * per + token / p.n, hk * group + r - token * group, token % p.n};
}

// Tile `index` of all units': later rows first, for under a causal mask they see the most keys.
struct Place {
  int u, hk, tile;
};
IRIS_DEVICE Place tile_place(const Params& p, const Plan& plan, int index) {
  const int unit = index % plan.units;
  return Place{unit / p.heads_kv, unit % p.heads_kv, plan.tiles - 1 - index / plan.units};
}

template <typename T, int D>
IRIS_DEVICE void tile_cta(const CUtensorMap& tpk, const CUtensorMap& tpv, const CUtensorMap& tk, const CUtensorMap& tv,
                          const Params& p, const Plan& plan, int cta, uint8_t* smem_raw) {
  constexpr int HALVES = D / 64, KV_BYTES = HALVES * KV_HALF;
  uint8_t* q_tile = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* k_tile = q_tile + HALVES * Q_HALF;
  uint8_t* v_tile = k_tile + KV * KV_BYTES;
  TileSmem* s = reinterpret_cast<TileSmem*>(v_tile + KV * KV_BYTES);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const int group = p.heads_q / p.heads_kv, rows = plan.per * p.n * group;
  if (threadIdx.x == 0) {
    mbar_init(&s->q_full, 4);
    for (int i = 0; i < KV; ++i) {
      mbar_init(&s->k_full[i], 1);
      mbar_init(&s->v_full[i], 1);
      mbar_init(&s->s_full[i], 1);
      mbar_init(&s->p_full[i], 4);
      mbar_init(&s->pv_done[i], 1);
    }
    mbar_init(&s->v_tail, 1);
    mbar_init(&s->teardown, 1);
    s->abort = 0;
    fence_barrier_init();
  }
  __syncthreads();
  volatile int* abort = &s->abort;
  grid_wait();
  const bool finish = cta < plan.whole_tiles;
  const int split = finish ? 0 : (cta - plan.whole_tiles) % plan.tile_splits;
  const int unit_tile = finish ? cta : plan.whole_tiles + (cta - plan.whole_tiles) / plan.tile_splits;
  const Place place_of = tile_place(p, plan, unit_tile);
  const int tile = place_of.tile, hk = place_of.hk, u = place_of.u;
  const int row0 = tile * BQ, last = min(row0 + BQ, rows) - 1;
  const int b0 = u * plan.per, g = b0 / p.per_group;
  const bool own = plan.per == 1 && plan.step_splits == 0;
  const int early = prefix_length(p, b0);
  const int length = own ? own_length(p, b0) : 0;
  const int64_t start = own ? own_start(p, b0) : 0;
  const int early_blocks = (early + BKV - 1) / BKV;
  const int all_blocks = early_blocks + (own ? (own_keys(p, start + last / group, length) + BKV - 1) / BKV : 0);
  const int first = finish ? 0 : min(split * plan.tile_chunk, all_blocks);
  const int iters = finish ? all_blocks : min(plan.tile_chunk, all_blocks - first);

  if (warp == 0) {
    // ----------------------------------------------------------------- TMA
    int issued_k[KV], issued_v[KV];
    for (int i = 0; i < KV; ++i) issued_k[i] = issued_v[i] = -1;
    int tails = 0;
    bool ok = true;
    if (lane == 0 && first < early_blocks) {
      tma_prefetch_desc(&tpk);
      tma_prefetch_desc(&tpv);
    }
    if (lane == 0 && all_blocks > early_blocks) {
      tma_prefetch_desc(&tk);
      tma_prefetch_desc(&tv);
    }
    // one block's 64 rows of keys or values into a slot
    auto load = [&](const CUtensorMap& of_prefix, const CUtensorMap& of_own, uint64_t* bar, uint8_t* slot, int block, int ph, int pb,
                    int oh, int ob) {
      mbar_arrive_expect_tx(bar, KV_BYTES);
      for (int c = 0; c < HALVES; ++c)
        if (block < early_blocks) tma_load_4d(&of_prefix, bar, slot + c * KV_HALF, c * 64, block * BKV, ph, pb);
        else tma_load_4d(&of_own, bar, slot + c * KV_HALF, c * 64, (block - early_blocks) * BKV, oh, ob);
    };
    auto load_k = [&](int it) {
      const int st = it % KV;
      const uint32_t ph = static_cast<uint32_t>((it / KV) & 1);
      ok = mbar_wait(&s->s_full[st], ph ^ 1u, abort);
      if (!ok) return;
      load(tpk, tk, &s->k_full[st], k_tile + st * KV_BYTES, first + it, p.pkh != 0 ? hk : 0, p.pkb != 0 ? g : 0, p.kh != 0 ? hk : 0,
           p.kb != 0 ? b0 : 0);
      issued_k[st] = static_cast<int>(ph);
    };
    if (lane == 0 && iters > 0) load_k(0);
    for (int it = 0; it < iters; ++it) {
      const int st = it % KV;
      const uint32_t ph = static_cast<uint32_t>((it / KV) & 1);
      const int block = first + it;
      // keys behind the length that the tensor map does not end before
      const int left = block < early_blocks ? early - block * BKV : length - (block - early_blocks) * BKV;
      const bool tail = left < BKV && (block < early_blocks ? early < p.n_prefix : length < p.n_kv);
      if (lane == 0 && ok) {
        if (it + 1 < iters) load_k(it + 1);  // scores run a block ahead
        ok = ok && mbar_wait(&s->pv_done[st], ph ^ 1u, abort);
        if (ok) {
          load(tpv, tv, tail ? &s->v_tail : &s->v_full[st], v_tile + st * KV_BYTES, block, p.pvh != 0 ? hk : 0, p.pvb != 0 ? g : 0,
               p.vh != 0 ? hk : 0, p.vb != 0 ? b0 : 0);
          issued_v[st] = tail ? -1 : static_cast<int>(ph);  // the copy before in this slot has been read
        }
      }
      if (!__shfl_sync(0xffffffffu, ok, 0)) break;
      if (tail) {  // two blocks of the CTA at most: those that the lengths end in
        ++tails;
        ok = __all_sync(0xffffffffu, mbar_wait(&s->v_tail, static_cast<uint32_t>(tails - 1) & 1u, abort));
        if (!ok) break;
        for (int e = left * 8 + lane; e < BKV * 8; e += 32)
          for (int c = 0; c < HALVES; ++c)
            *reinterpret_cast<uint4*>(v_tile + st * KV_BYTES + c * KV_HALF + e * 16) = make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s->v_full[st]);
      }
    }
    if (lane == 0 && iters > 0) {  // whichever warp gives up: no copy may land after the CTA is gone
      int dummy = 0;
      for (int i = 0; i < KV; ++i) {
        if (issued_k[i] >= 0) mbar_wait(&s->k_full[i], static_cast<uint32_t>(issued_k[i]), &dummy);
        if (issued_v[i] >= 0) mbar_wait(&s->v_full[i], static_cast<uint32_t>(issued_v[i]), &dummy);
      }
      if (tails > 0) mbar_wait(&s->v_tail, static_cast<uint32_t>(tails - 1) & 1u, &dummy);
    }
  } else if (warp == 1) {
    // ----------------------------------------------------------------- MMA
    // TMEM only after the wait (a CTA that held some while it waits could keep its predecessor's,
    // which still have to allocate theirs, from ever ending), and the successor only after TMEM
    tmem_alloc(&s->tmem_base, TILE_COLS);
    grid_trigger();
    tc_fence_before();
    __syncwarp();
    barrier_tell<1, 32 + BQ>();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&s->tmem_base);
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
        umma_commit(&s->pv_done[st]);
        // into the buffer of the P just read: one thread's MMAs run in order
        if (it + 2 < iters) issue_s(it + 2);
      }
      umma_commit(&s->teardown);
      int dummy = 0;
      mbar_wait(&s->teardown, 0, &dummy);
    }
  } else {
    // ------------------------------------------------------------- softmax
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane, r = row0 + row;  // of the tile, of the unit
    const Row at = row_of(p, plan.per, u, hk, min(r, rows - 1));
    auto place = [&](int row, int piece) { return row * 128 + ((piece ^ (row & 7)) * 16); };
    // Q: the warp's 32 rows, each by D / 8 lanes; rows from the unit's end on are zeros
    if (iters > 0) {
      constexpr int LANES = D / 8, STEP = 32 / LANES;
      const int piece = lane % LANES;
      const int64_t mine = at.b * p.qb + at.h * p.qh + at.i * p.qn;
      const uint32_t to = smem_addr(q_tile) + (piece >> 3) * Q_HALF;
#pragma unroll 1
      for (int x = 0; x < 32; x += STEP) {
        const int w = x + lane / LANES;
        const T* from = reinterpret_cast<const T*>(p.q) + __shfl_sync(0xffffffffu, mine, w) + piece * 8;
        copy16(to + place(quarter * 32 + w, piece & 7), from, row0 + quarter * 32 + w < rows);
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s->q_full);
    }
    barrier_wait<1, 32 + BQ>();
    tc_fence_after();
    const uint32_t lanes = s->tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const int own_hi = own ? own_keys(p, start + at.i, length) : 0;
    // what every row of the warp sees
    const int hi_all = __shfl_sync(0xffffffffu, own_hi, 0);
    float m_run = -INFINITY, l_run = 0.f;
    bool ok = true;
    for (int it = 0; it < iters; ++it) {
      const int block = first + it;
      const int key0 = (block < early_blocks ? block : block - early_blocks) * BKV;
      const int seen = (block < early_blocks ? early : own_hi) - key0;  // leading keys of the block that the row sees
      const bool full = (block < early_blocks ? early : hi_all) - key0 >= BKV;
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
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (c * 32 + e >= seen) r[c][e] = __float_as_uint(-INFINITY);
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
        ok = __all_sync(0xffffffffu, mbar_wait(&s->pv_done[(it - 1) & 1], static_cast<uint32_t>(((it - 1) >> 1) & 1), abort));
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
      // the tensor cores take 16 bits. The rounding is relative to each weight and averages
      // out over the keys; the sum takes the fp32 values. Masked keys give exact zeros
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
    if (iters > 0)
      ok = ok && __all_sync(0xffffffffu, mbar_wait(&s->pv_done[(iters - 1) & 1], static_cast<uint32_t>(((iters - 1) >> 1) & 1), abort));
    ok = ok && *abort == 0;
    tc_fence_after();
    // rows leave from the place of Q and the rings (every product is computed), each as one
    // bulk copy; 16 bytes of padding spread a piece of 8 rows over the banks
    if (!finish) {
      // this chunk's state; a wait that gave up (device error word) makes the row NaN
      const int64_t part = (static_cast<int64_t>(unit_tile - plan.whole_tiles) * plan.tile_splits + split) * BQ + row;
      if (r < rows) plan.tile_states[part] = ok ? make_float2(m_run, l_run) : make_float2(NAN, NAN);
      if (ok && iters > 0) {
        uint8_t* mine = q_tile + row * (D * 4 + 16);
#pragma unroll 1
        for (int c = 0; c < D / 16; ++c) {
          uint32_t o[16];
          tmem_ld16(lanes + COL_O + c * 16, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<uint4*>(mine + c * 64 + e * 16) = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        }
        fence_proxy_async_smem();
        if (r < rows) bulk_store(plan.tile_sums + part * D, mine, D * 4);
        tma_store_wait();
      }
    } else {
      const float inv = ok ? 1.f / l_run : NAN;
      bool finite = true;
      uint8_t* mine = q_tile + row * (D * 2 + 16);
#pragma unroll 1
      for (int c = 0; c < D / 16; ++c) {
        uint32_t o[16], pk[8];
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = 0u;
        if (iters > 0) {
          tmem_ld16(lanes + COL_O + c * 16, o);
          tmem_wait_ld();
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = iters > 0 ? __uint_as_float(o[2 * e]) * inv : 0.f;
          const float z = iters > 0 ? __uint_as_float(o[2 * e + 1]) * inv : 0.f;
          finite = finite && isfinite(x) && isfinite(z);
          pk[e] = pack2<T>(x, z);
        }
        *reinterpret_cast<uint4*>(mine + c * 32) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
        *reinterpret_cast<uint4*>(mine + c * 32 + 16) = make_uint4(pk[4], pk[5], pk[6], pk[7]);
      }
      __syncwarp();  // a row that is computed again comes after what was written of it
      for (uint32_t again = __ballot_sync(0xffffffffu, ok && !finite && r < rows); again != 0; again &= again - 1) {
        const int from = __ffs(again) - 1;
        float2 acc[D / 64];
        attend_row<T, D>(p, __shfl_sync(0xffffffffu, at.b, from), __shfl_sync(0xffffffffu, at.h, from),
                         __shfl_sync(0xffffffffu, at.i, from), acc);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          *reinterpret_cast<uint32_t*>(q_tile + (quarter * 32 + from) * (D * 2 + 16) + c * 128 + lane * 4) = pack2<T>(acc[c].x, acc[c].y);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (r < rows) bulk_store(reinterpret_cast<T*>(p.out) + at.b * p.ob + at.i * p.on + static_cast<int64_t>(at.h) * D, mine, D * 2);
      tma_store_wait();
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(s->tmem_base, TILE_COLS);
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

// Rows of keys or values: row c at `at` + 16 stride c, which is row c - first of the tensor.
struct KeyRows {
  uint64_t at;
  uint32_t stride;  // 16-byte pieces: strides are below 2^34 elements
};
template <typename T>
IRIS_DEVICE KeyRows key_rows(const void* data, int64_t offset, int64_t stride, int first) {
  return KeyRows{reinterpret_cast<uint64_t>(reinterpret_cast<const T*>(data) + offset - first * stride), static_cast<uint32_t>(stride / 8)};
}

// 8 x 8 16-bit elements of a warp's registers transposed.
IRIS_DEVICE uint32_t movmatrix(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// 8 NQ rows of a sample and key head over a chunk of their keys: the prefix's (PREFIX) and
// then the sample's own. Four warps; the block's others only meet the barriers.
template <typename T, int D, int NQ, bool PREFIX>
IRIS_DEVICE void step_cta(const Params& p, const Plan& plan, int cta, uint8_t* smem_raw) {
  constexpr int ROWS = 8 * NQ, TILE = STEP_KEYS * D * 2;  // bytes of one K or V tile
  constexpr int PAD = D + 4;  // floats of a row of sums: the four lanes of a column pair in different banks
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x & 31;
  const int split = cta % plan.step_splits, unit = cta / plan.step_splits;  // (b, hk, row tile)
  const int rt = unit % plan.row_tiles, hk = unit / plan.row_tiles % p.heads_kv, b = unit / plan.row_tiles / p.heads_kv;
  const int group = p.heads_q / p.heads_kv, rows = p.n * group;
  const int r0 = rt * ROWS, r_last = min(r0 + ROWS, rows) - 1;
  if (PREFIX && plan.cluster) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  grid_wait();
  grid_trigger();
  const int early = PREFIX ? prefix_length(p, b) : 0;
  const int length = own_length(p, b);
  const int64_t start = own_start(p, b);
  const int count = early + own_keys(p, start + r_last / group, length);  // some row of the tile sees them
  const bool same = r0 / group == r_last / group;  // one token: every row sees all of them
  const int c_begin = min(split * plan.step_chunk, count), c_end = min(c_begin + plan.step_chunk, count);

  // where key c of each lot would start, and its rows' stride in 16-byte pieces: one multiplication a copy
  const int pb = b / p.per_group;
  const KeyRows pk = key_rows<T>(p.pk, pb * p.pkb + hk * p.pkh, p.pkn, 0), pv = key_rows<T>(p.pv, pb * p.pvb + hk * p.pvh, p.pvn, 0);
  const KeyRows k = key_rows<T>(p.k, b * p.kb + hk * p.kh, p.kn, early), v = key_rows<T>(p.v, b * p.vb + hk * p.vh, p.vn, early);
  const uint32_t ring = smem_addr(smem_raw) + warp * (STEP_STAGES * 2 * TILE);
  const int tiles = (c_end - c_begin + STEP_KEYS - 1) / STEP_KEYS;
  const int mine = tiles > warp ? (tiles - warp + STEP_WARPS - 1) / STEP_WARPS : 0;
  // tile t of the warp into its slot: rows of D / 8 16-byte pieces, piece x of row r at x ^ (r & 7)
  constexpr int PIECES = D / 8;
  auto load = [&](int t) {
    if (t < mine) {
      const int c0 = c_begin + (warp + t * STEP_WARPS) * STEP_KEYS;
      const uint32_t slot = ring + (t % STEP_STAGES) * 2 * TILE;
#pragma unroll 1
      for (int e = 0; e < STEP_KEYS * PIECES / 32; ++e) {
        const int at = e * 32 + lane, r = at / PIECES, x = at % PIECES;
        const int c = c0 + r;
        const bool real = c < c_end;
        const bool of_prefix = PREFIX && c < early;
        const uint64_t key = static_cast<uint32_t>(real ? c : c_begin);
        const uint64_t from_k = (of_prefix ? pk.at : k.at) + key * (of_prefix ? pk.stride : k.stride) * 16 + x * 16;
        const uint64_t from_v = (of_prefix ? pv.at : v.at) + key * (of_prefix ? pv.stride : v.stride) * 16 + x * 16;
        const uint32_t dst = slot + r * (D * 2) + ((x ^ (r & 7)) * 16);
        copy16(dst, reinterpret_cast<const void*>(from_k), real);
        copy16(dst + TILE, reinterpret_cast<const void*>(from_v), real);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // this lane's queries: 8 j + 2 (lane % 4) + {0, 1}; its key of a tile's halves, column of O^T's: lane / 4
  const int g = lane >> 2, quad = lane & 3;
  float o[D / 16][NQ][4];
  float m_run[NQ][2], l_run[NQ][2];
  if (warp < STEP_WARPS) {
    // Q's rows into the slot that is filled last, then the first tiles
    const uint32_t q_slot = ring + (STEP_STAGES - 1) * 2 * TILE;
#pragma unroll 1
    for (int e = 0; e < ROWS * PIECES / 32; ++e) {
      const int at = e * 32 + lane, w = at / PIECES, x = at % PIECES;
      const int r = min(r0 + w, rows - 1);
      const T* q = reinterpret_cast<const T*>(p.q) + b * p.qb + (hk * group + r % group) * p.qh + static_cast<int64_t>(r / group) * p.qn;
      copy16(q_slot + w * (D * 2) + ((x ^ (w & 7)) * 16), q + x * 8, r0 + w < rows);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll 1
    for (int t = 0; t < STEP_STAGES - 1; ++t) load(t);

    uint32_t qb[D / 16][NQ][2];
    int seen[NQ][2];
#pragma unroll
    for (int j = 0; j < NQ; ++j)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        seen[j][u] = early + own_keys(p, start + min(r0 + 8 * j + 2 * quad + u, rows - 1) / group, length);
        m_run[j][u] = -INFINITY;
        l_run[j][u] = 0.f;
      }
    asm volatile("cp.async.wait_group %0;" ::"n"(STEP_STAGES - 1) : "memory");
    __syncwarp();
#pragma unroll
    for (int j = 0; j < NQ; ++j)
#pragma unroll
      for (int d = 0; d < D / 32; ++d) {  // pieces 4 d .. 4 d + 3 of 8 query rows
        uint32_t r4[4];
        const int r = 8 * j + (lane & 7), x = 4 * d + (lane >> 3);
        ldmatrix4(r4, q_slot + r * (D * 2) + ((x ^ (r & 7)) * 16));
        qb[2 * d][j][0] = r4[0], qb[2 * d][j][1] = r4[1], qb[2 * d + 1][j][0] = r4[2], qb[2 * d + 1][j][1] = r4[3];
      }
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
      for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][j][e] = 0.f;

    for (int t = 0; t < mine; ++t) {
      asm volatile("cp.async.wait_group %0;" ::"n"(STEP_STAGES - 2) : "memory");
      __syncwarp();  // every lane's copies of the tile have landed; the slot refilled next was read by all
      load(t + STEP_STAGES - 1);
      const uint32_t slot = ring + (t % STEP_STAGES) * 2 * TILE;
      const int c0 = c_begin + (warp + t * STEP_WARPS) * STEP_KEYS;
      float s[NQ][4], odd[NQ][4];
#pragma unroll
      for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = odd[j][e] = 0.f;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {  // 16 keys of pieces 2 d and 2 d + 1
        uint32_t ka[4];
        const int r = lane & 15, x = 2 * d + (lane >> 4);
        ldmatrix4(ka, slot + r * (D * 2) + ((x ^ (r & 7)) * 16));
#pragma unroll
        for (int j = 0; j < NQ; ++j) mma_16816<T>(d & 1 ? odd[j] : s[j], ka, qb[d][j][0], qb[d][j][1]);  // two chains
      }
#pragma unroll
      for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] += odd[j][e];
      if (!same || c0 + STEP_KEYS > c_end) {
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int c = c0 + g + 8 * (e >> 1);
            if (c >= c_end || c >= seen[j][e & 1]) s[j][e] = -INFINITY;
          }
      }
      // a row's maximum is kept until a score exceeds it by 2^8, seen by any lane
      bool grow = false;
#pragma unroll
      for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int u = 0; u < 2; ++u) grow = grow || fmaxf(s[j][u], s[j][u + 2]) * p.scale_log2 > m_run[j][u] + RESCALE;
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float mx = fmaxf(s[j][u], s[j][u + 2]) * p.scale_log2;
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const bool more = mx > m_run[j][u] + RESCALE;
            const float corr = more && m_run[j][u] != -INFINITY ? ex2(m_run[j][u] - mx) : 1.f;
            if (more) m_run[j][u] = mx;
            l_run[j][u] *= corr;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
              o[d][j][u] *= corr;
              o[d][j][u + 2] *= corr;
            }
          }
      }
      // weights, rounded once to the operand type (the fp32 values go into the totals): as in
      // tile_cta, so that a row is as accurate in either form
      uint32_t pw[NQ][2];
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float m = m_run[j][e & 1];
          w[e] = ex2(fmaf(s[j][e], p.scale_log2, m == -INFINITY ? 0.f : -m));
          l_run[j][e & 1] += w[e];
        }
        pw[j][0] = movmatrix(pack2<T>(w[0], w[1]));
        pw[j][1] = movmatrix(pack2<T>(w[2], w[3]));
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {  // 16 columns of V (pieces 2 d and 2 d + 1) as rows, by 16 keys
        uint32_t va[4];
        const int r = (lane & 7) + (lane >> 4) * 8, x = 2 * d + (lane >> 3 & 1);
        ldmatrix4_trans(va, slot + TILE + r * (D * 2) + ((x ^ (r & 7)) * 16));
#pragma unroll
        for (int j = 0; j < NQ; ++j) mma_16816<T>(o[d][j], va, pw[j][0], pw[j][1]);
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int j = 0; j < NQ; ++j)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int x = 4; x <= 16; x *= 2) l_run[j][u] += __shfl_xor_sync(0xffffffffu, l_run[j][u], x);
  }
  // the warps' states, joined per row: warp w finishes rows w, w + 4, ...
  __syncthreads();  // the rings are done with
  float* sums = reinterpret_cast<float*>(smem_raw);  // [warp][ROWS][PAD]
  __shared__ float tops[STEP_WARPS][16], totals[STEP_WARPS][16];
  if (warp < STEP_WARPS) {
#pragma unroll
    for (int j = 0; j < NQ; ++j)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int row = 8 * j + 2 * quad + u;
        float* dst = sums + (warp * ROWS + row) * PAD + g;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          dst[16 * d] = o[d][j][u];
          dst[16 * d + 8] = o[d][j][u + 2];
        }
        if (g == 0) {
          tops[warp][row] = m_run[j][u];
          totals[warp][row] = l_run[j][u];
        }
      }
  }
  __syncthreads();
  // cluster: states [chunk][owned row], sums then {maximum, total}; other CTAs store here once all have begun
  float* states = reinterpret_cast<float*>(smem_raw + STEP_RINGS<D>);
  const int owned = rows_owned(ROWS, plan.step_splits);
  if (PREFIX && plan.cluster) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (warp < STEP_WARPS) {
    for (int r = warp; r <= r_last - r0; r += STEP_WARPS) {
      float top = -INFINITY, total = 0.f;
#pragma unroll
      for (int w = 0; w < STEP_WARPS; ++w) top = fmaxf(top, tops[w][r]);
      float2 acc[D / 64];
#pragma unroll
      for (int c = 0; c < D / 64; ++c) acc[c] = make_float2(0.f, 0.f);
#pragma unroll 1
      for (int w = 0; w < STEP_WARPS; ++w) {
        // a warp that saw nothing has sums of 0 (or NaN, from a masked V: kept, it marks the row)
        const float f = tops[w][r] == -INFINITY ? 1.f : ex2(tops[w][r] - top);
        total += f * totals[w][r];
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          const float2 x = *reinterpret_cast<const float2*>(sums + (w * ROWS + r) * PAD + 64 * c + 2 * lane);
          acc[c] = make_float2(fmaf(f, x.x, acc[c].x), fmaf(f, x.y, acc[c].y));
        }
      }
      if (PREFIX && plan.cluster) {
        float* at = states + (split * owned + r % owned) * (D + 2);
        const uint32_t to = map_to_cta(at, static_cast<uint32_t>(r / owned));
#pragma unroll
        for (int c = 0; c < D / 64; ++c) store_remote(to + 4 * (64 * c + 2 * lane), acc[c]);
        if (lane == 0) store_remote(to + 4 * D, make_float2(top, total));
      } else if (plan.step_sums == nullptr) {
        finish_row<T, D>(p, b, hk * group + (r0 + r) % group, (r0 + r) / group, acc, total);
      } else {
        const int64_t part = (static_cast<int64_t>(unit) * plan.step_splits + split) * ROWS + r;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) *reinterpret_cast<float2*>(plan.step_sums + part * D + 64 * c + 2 * lane) = acc[c];
        if (lane == 0) plan.step_states[part] = make_float2(top, total);
      }
    }
  }
  if (PREFIX && plan.cluster) {
    cluster_sync();
    for (int local = warp; local < owned && split * owned + local <= r_last - r0; local += STEP_WARPS) {
      const int r = r0 + split * owned + local;
      float top = -INFINITY, total = 0.f;
      for (int q = 0; q < plan.step_splits; ++q) top = fmaxf(top, states[(q * owned + local) * (D + 2) + D]);
      float2 acc[D / 64];
#pragma unroll
      for (int c = 0; c < D / 64; ++c) acc[c] = make_float2(0.f, 0.f);
      for (int q = 0; q < plan.step_splits; ++q) {
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

// Few rows over few keys: no tiles.
template <typename T, int D, int NQ>
__global__ void __launch_bounds__(STEP_WARPS * 32) step_kernel(const __grid_constant__ Params p, const __grid_constant__ Plan plan) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  step_cta<T, D, NQ, true>(p, plan, static_cast<int>(blockIdx.x), smem_raw);
}

// What a CTA runs once is kept in loops, here and in tile_cta: straight code waits for its
// instructions (Q's 16 copies a lane unrolled took 4.9 us of a tile's 14).

// Both kinds of CTA in one launch, the longer ones first: tiles are bound by the tensor cores
// and exponentials, the others by memory, and they share the SMs (mixed evenly, tiles that
// started late ended last: 64 samples behind 32768 tokens 111 us).
//
// 128 registers a thread hold both kinds of CTA but for 16 rows of 128 columns (NQ 2), where the compiler
// spills 140 bytes; that instance also runs where there are tiles alone.
template <typename T, int D, int NQ>
__global__ void __launch_bounds__(BOUND_THREADS, 2)
    attend_kernel(const __grid_constant__ CUtensorMap tpk, const __grid_constant__ CUtensorMap tpv,
                  const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                  const __grid_constant__ Params p, const __grid_constant__ Plan plan) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  if (static_cast<int>(blockIdx.x) < plan.tile_ctas) {
    tile_cta<T, D>(tpk, tpv, tk, tv, p, plan, static_cast<int>(blockIdx.x), smem_raw);
  } else {
    // no second CTA starts on the SM while one of a kernel that allocates TMEM may still do so
    // (measured: step CTAs ran one at a time, 41 us instead of 30 for 512 of them)
    if (threadIdx.x < 32) tmem_relinquish();
    step_cta<T, D, NQ, false>(p, plan, static_cast<int>(blockIdx.x) - plan.tile_ctas, smem_raw);
  }
}

// A row's chunks joined by a warp.
template <typename T, int D>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ Params p, const __grid_constant__ Plan plan) {
  const int lane = threadIdx.x & 31;
  const int group = p.heads_q / p.heads_kv, rows = plan.per * p.n * group;
  const int index = static_cast<int>(blockIdx.x / (BQ / 4));  // of the tiles behind the whole ones
  const int in_tile = static_cast<int>(blockIdx.x % (BQ / 4)) * 4 + (threadIdx.x >> 5);
  const Place at = tile_place(p, plan, plan.whole_tiles + index);
  const int r = at.tile * BQ + in_tile;
  if (r >= rows) return;
  const Row row = row_of(p, plan.per, at.u, at.hk, r);
  const int b = row.b, h = row.h, i = row.i;
  grid_wait();
  grid_trigger();
  int64_t tile0 = 0, step0 = 0;  // of its states: first place, and how many there are, BQ or step_rows apart
  int tile_parts = 0, step_parts = 0;
  if (plan.tile_sums != nullptr) {
    tile0 = static_cast<int64_t>(index) * plan.tile_splits * BQ + in_tile;
    tile_parts = plan.tile_splits;
  }
  if (plan.step_sums != nullptr) {
    const int of_sample = i * group + h % group;
    const int64_t unit = (static_cast<int64_t>(b) * p.heads_kv + at.hk) * plan.row_tiles + of_sample / plan.step_rows;
    step0 = unit * plan.step_splits * plan.step_rows + of_sample % plan.step_rows;
    step_parts = plan.step_splits;
  }
  const int parts = tile_parts + step_parts;
  auto state_of = [&](int c) {
    return c < tile_parts ? plan.tile_states[tile0 + static_cast<int64_t>(c) * BQ]
                          : plan.step_states[step0 + static_cast<int64_t>(c - tile_parts) * plan.step_rows];
  };
  float top = -INFINITY;
  for (int c = lane; c < parts; c += 32) top = fmaxf(top, state_of(c).x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float total = 0.f;
  bool lost = false;  // a wait gave up
  float2 acc[D / 64];
#pragma unroll
  for (int c = 0; c < D / 64; ++c) acc[c] = make_float2(0.f, 0.f);
  for (int c0 = 0; c0 < parts; c0 += 32) {
    // a lane's part: its factor; one that saw nothing has none (a tile without keys wrote no sums)
    const float2 st = c0 + lane < parts ? state_of(c0 + lane) : make_float2(-INFINITY, 0.f);
    const bool real = st.x != -INFINITY || st.y != 0.f;
    const float f = !real ? 0.f : st.x == -INFINITY ? 1.f : ex2(st.x - top);
    total += real ? f * st.y : 0.f;
    lost = lost || (isnan(st.x) && isnan(st.y));
    const uint32_t some = __ballot_sync(0xffffffffu, real);
    const int most = min(32, parts - c0);
#pragma unroll 4
    for (int e = 0; e < most; ++e) {
      const int c = c0 + e;
      const float* from = c < tile_parts ? plan.tile_sums + (tile0 + static_cast<int64_t>(c) * BQ) * D
                                         : plan.step_sums + (step0 + static_cast<int64_t>(c - tile_parts) * plan.step_rows) * D;
      const float fc = __shfl_sync(0xffffffffu, f, e);
#pragma unroll
      for (int d = 0; d < D / 64; ++d) {
        const float2 x = *reinterpret_cast<const float2*>(from + 64 * d + 2 * lane);
        if (some >> e & 1u) acc[d] = make_float2(fmaf(fc, x.x, acc[d].x), fmaf(fc, x.y, acc[d].y));
      }
    }
  }
  total = warp_sum(total);
  lost = __any_sync(0xffffffffu, lost);
  if (lost) {
    T* o = reinterpret_cast<T*>(p.out) + b * p.ob + i * p.on + static_cast<int64_t>(h) * D + 2 * lane;
    for (int c = 0; c < D / 64; ++c) *reinterpret_cast<uint32_t*>(o + 64 * c) = pack2<T>(NAN, NAN);
    return;
  }
  finish_row<T, D>(p, b, h, i, acc, total);
}

// How a call is cut up, from its sizes alone (lengths are on the device: n_prefix and
// n_kv bound them, and are taken for them: caches with much room to spare are cut as if they were
// full, one token of 32 samples behind 2048 with 256 of their own 15.9 us in a room of 256, 32.8 in
// 2048, 166 in 8192). Three forms, and the one whose estimate is least:
//  - joint: row tiles of a sample see all of its keys (step_kernel); few rows or short prefixes;
//  - shared: a group's rows see the prefix by tiles, row tiles their own keys;
//  - whole: a sample's rows see all keys by tiles; prompts.
// Estimates in us, from the SMs' two slots each. A tile's CTA takes TILE_START and TILE_BLOCK
// for each 64 keys, a row tile's STEP_START and, for each key, STEP_KEY alone on its SM or
// STEP_PAIRED beside another (8 rows; 16 rows 1.3 times that, heads of 64 0.6 times); joining
// parts takes JOIN and their bytes. Measured against the estimate, heads of 128, the form
// taken and the next: 4 samples behind 300 tokens, 4 rows each, joint 4.4 (3.7), shared 9.4 (9.7);
// 32 behind 2048 with 512 of their own, shared 20 (16), joint 36 (38); 8 behind 8192, shared
// 20 (16), joint 31 (32); one of 256 rows behind 16384, whole 27 (24), joint 99 (98); 4 of 128 rows
// behind 1000, whole 14 (13), joint 22 (16).
constexpr float TILE_START = 5.3f, TILE_BLOCK = 0.95f, STEP_START = 2.5f, STEP_KEY = 0.0096f, STEP_PAIRED = 0.0139f;
constexpr float JOIN = 2.5f, JOIN_BYTES = 5.0e6f;  // bytes per us, written and read

struct Sizes {
  int64_t batch, groups, heads_q, heads_kv, n, n_prefix, n_kv, head_dim;
};

struct Estimate {
  const Sizes& z;
  int64_t sms = num_sms(), slots = 2 * sms;
  int64_t group = z.heads_q / z.heads_kv, rows = z.n * group, all_rows = z.batch * z.heads_q * z.n;
  float width = z.head_dim == 64 ? 0.6f : 1.f;

  float tile(int64_t blocks) const { return TILE_START + TILE_BLOCK * (0.5f + 0.5f * width) * blocks; }
  // a row tile's CTA over so many keys, one of `ctas`
  float step(int64_t keys, int64_t ctas) const {
    return STEP_START + (ctas <= sms ? STEP_KEY : STEP_PAIRED) * (rows > 8 ? 1.3f : 1.f) * width * keys;
  }
  float join(int64_t joined, int64_t parts) const { return JOIN + joined * parts * z.head_dim * 8 / JOIN_BYTES; }
};

// Chunks of `keys` in units of `unit`, so many or fewer.
struct Cut {
  int64_t chunk, splits;
};
inline Cut cut(int64_t keys, int64_t splits, int64_t unit) {
  splits = std::max<int64_t>(1, std::min(splits, (keys + unit - 1) / unit));
  const int64_t chunk = std::max(unit, ((keys + splits - 1) / splits + unit - 1) / unit * unit);
  return Cut{chunk, std::max<int64_t>(1, (keys + chunk - 1) / chunk)};
}

int make_plan(const Sizes& z, Plan* out) {
  const Estimate e{z};
  const int64_t per_group = z.batch / z.groups;
  const int64_t step_rows = e.rows <= 8 ? 8 : 16, row_tiles = (e.rows + step_rows - 1) / step_rows;
  const int64_t step_units = z.batch * z.heads_kv * row_tiles, keys = z.n_prefix + z.n_kv;
  constexpr int64_t STEP_UNIT = STEP_WARPS * STEP_KEYS;
  float least = INFINITY;
  Plan plan = {};
  plan.step_rows = static_cast<int>(step_rows);
  plan.row_tiles = static_cast<int>(std::min<int64_t>(row_tiles, 1 << 30));
  Cut tile_cut = {1, 1}, step_cut = {STEP_UNIT, 1};
  int form = 0;  // 0 joint, 1 shared, 2 whole
  // joint: up to eight chunks are joined in a cluster
  for (int64_t s : {int64_t(1), int64_t(2), int64_t(4), int64_t(8), e.slots / std::max<int64_t>(1, step_units)}) {
    const Cut c = cut(keys, s, STEP_UNIT);
    const int64_t ctas = step_units * c.splits;
    const float t = ((ctas + e.slots - 1) / e.slots) * e.step(std::min(c.chunk, keys), ctas) +
                    (c.splits > MOST_CLUSTER ? e.join(e.all_rows, c.splits) : 0.f);
    if (t < least) least = t, step_cut = c;
  }
  const int64_t prefix_blocks = (z.n_prefix + BKV - 1) / BKV;
  if (per_group > 1 && z.n_prefix > 0) {
    // the samples' own keys: split only where they leave SMs idle
    const Cut own = cut(z.n_kv, step_units * 2 <= e.sms ? e.sms / step_units : 1, STEP_UNIT);
    const int64_t steps = step_units * own.splits, units = z.groups * z.heads_kv;
    const int64_t tiles = units * ((per_group * e.rows + BQ - 1) / BQ);
    for (int64_t s : {int64_t(1), int64_t(2), int64_t(4), int64_t(8), int64_t(16), int64_t(32), e.sms / std::max<int64_t>(1, tiles),
                      e.slots / std::max<int64_t>(1, tiles)}) {
      const Cut c = cut(prefix_blocks, s, 1);
      const int64_t ctas = tiles * c.splits;
      const float tile = e.tile(c.chunk), step = e.step(std::min(own.chunk, z.n_kv), steps + ctas);
      const int64_t beside = std::max<int64_t>(0, e.slots - ctas);  // slots that row tiles have from the start
      float t;
      if (ctas > e.slots) t = (ctas * tile + steps * step) / e.slots + 0.5f * tile;
      else if (steps * step <= beside * tile) t = std::max(tile, (steps + beside - 1) / beside * step);
      else t = tile + (steps * step - beside * tile) / e.slots + 0.5f * step;
      t += e.join(e.all_rows, c.splits + own.splits);
      if (t < least) least = t, form = 1, tile_cut = c, step_cut = own;
    }
  }
  {
    const int64_t blocks = prefix_blocks + (z.n_kv + BKV - 1) / BKV;
    const int64_t tiles = z.batch * z.heads_kv * ((e.rows + BQ - 1) / BQ);
    // tiles that fill the SMs are not split; the last of them, which would leave some idle, are
    const int64_t rest = tiles % e.slots != 0 ? tiles % e.slots : tiles;
    const Cut c = cut(blocks, std::min(e.slots / std::max<int64_t>(1, rest), std::max<int64_t>(1, blocks / 4)), 1);
    float t = ((tiles - 1) / e.slots) * e.tile(blocks) + e.tile(c.chunk);
    if (c.splits > 1) t += e.join(rest * std::min<int64_t>(BQ, e.rows), c.splits);
    if (t < least) least = t, form = 2, tile_cut = c;
  }
  plan.per = static_cast<int>(form == 1 ? per_group : 1);
  const int64_t units = z.batch / plan.per * z.heads_kv, tiles = (plan.per * e.rows + BQ - 1) / BQ, all = units * tiles;
  IRIS_REQUIRE(all < (1ll << 30) && step_units < (1ll << 30), "prefix_attn_fwd: too many rows");
  plan.units = static_cast<int>(units);
  plan.tiles = static_cast<int>(tiles);
  plan.tile_splits = 1;
  if (form != 0) {
    const int64_t rest = form == 2 && all % e.slots != 0 ? all % e.slots : all;
    plan.tile_chunk = static_cast<int>(tile_cut.chunk);
    plan.tile_splits = static_cast<int>(tile_cut.splits);
    plan.whole_tiles = static_cast<int>(form == 1 ? 0 : tile_cut.splits == 1 ? all : all - rest);
    const int64_t ctas = plan.whole_tiles + (all - plan.whole_tiles) * tile_cut.splits;
    IRIS_REQUIRE(ctas < (1ll << 30), "prefix_attn_fwd: too many rows");
    plan.tile_ctas = static_cast<int>(ctas);
  }
  if (form != 2) {
    IRIS_REQUIRE(step_units * step_cut.splits < (1ll << 30), "prefix_attn_fwd: too many rows");
    plan.step_prefix = form == 0;
    plan.step_chunk = static_cast<int>(step_cut.chunk);  // at most the keys (below 2^30) and 63
    plan.step_splits = static_cast<int>(step_cut.splits);
    plan.step_ctas = static_cast<int>(step_units * step_cut.splits);
    plan.cluster = form == 0 && plan.step_splits > 1 && plan.step_splits <= MOST_CLUSTER;
  }
  *out = plan;
  return IRIS_OK;
}

// Floats of the parts' sums, and as many pairs of a maximum and a total as rows of them.
struct Room {
  int64_t tile_rows, step_rows;
};
inline Room room_of(const Plan& plan) {
  Room x = {};
  x.tile_rows = static_cast<int64_t>(plan.tile_ctas - plan.whole_tiles) * BQ;
  if (x.tile_rows > 0 || (plan.step_splits > 1 && !plan.cluster)) x.step_rows = static_cast<int64_t>(plan.step_ctas) * plan.step_rows;
  return x;
}
// Tiles whose rows join_kernel takes.
inline int64_t joined_tiles(const Plan& plan) {
  return plan.tile_ctas > 0 ? (plan.tile_ctas - plan.whole_tiles) / plan.tile_splits : static_cast<int64_t>(plan.tiles) * plan.units;
}
inline int64_t room_bytes(const Room& x, int64_t d) { return (x.tile_rows + x.step_rows) * (d + 2) * 4; }

template <typename... Params_>
int allow_smem(void (*kernel)(Params_...), int bytes, bool (&configured)[64]) {
  int dev = 0;
  IRIS_CUDA(cudaGetDevice(&dev));
  if (dev < 64 && configured[dev]) return IRIS_OK;
  IRIS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  IRIS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
  if (dev < 64) configured[dev] = true;
  return IRIS_OK;
}

template <typename T, int D, int NQ>
int launch_rows(const Params& p, const Plan& plan, int dtype, cudaStream_t st) {
  if (plan.tile_ctas == 0) {
    static bool configured[64] = {false};
    IRIS_CHECK_STATUS(allow_smem(step_kernel<T, D, NQ>, cluster_smem<D>(), configured));
    IRIS_CUDA(launch_early(step_kernel<T, D, NQ>, dim3(static_cast<unsigned>(plan.step_ctas)), STEP_WARPS * 32,
                           plan.cluster ? cluster_smem<D>() : STEP_RINGS<D>, st,
                           plan.cluster ? static_cast<unsigned>(plan.step_splits) : 1u, p, plan));
    return IRIS_OK;
  }
  CUtensorMap tpk = {}, tpv = {}, tk = {}, tv = {};
  if (p.n_prefix > 0) {
    const int groups = p.batch / p.per_group;
    IRIS_CHECK_STATUS(make_tmap_heads(&tpk, p.pk, dtype, D, p.n_prefix, p.heads_kv, groups, p.pkn, p.pkh, p.pkb, BKV));
    IRIS_CHECK_STATUS(make_tmap_heads(&tpv, p.pv, dtype, D, p.n_prefix, p.heads_kv, groups, p.pvn, p.pvh, p.pvb, BKV));
  }
  if (plan.step_splits == 0 && p.n_kv > 0) {
    IRIS_CHECK_STATUS(make_tmap_heads(&tk, p.k, dtype, D, p.n_kv, p.heads_kv, p.batch, p.kn, p.kh, p.kb, BKV));
    IRIS_CHECK_STATUS(make_tmap_heads(&tv, p.v, dtype, D, p.n_kv, p.heads_kv, p.batch, p.vn, p.vh, p.vb, BKV));
  }
  static bool configured[64] = {false};
  IRIS_CHECK_STATUS(allow_smem(attend_kernel<T, D, NQ>, most_smem<D>(), configured));
  IRIS_CUDA(launch_early(attend_kernel<T, D, NQ>, dim3(static_cast<unsigned>(plan.tile_ctas + plan.step_ctas)), THREADS,
                         plan.step_splits == 0 ? tile_smem<D>() : most_smem<D>(), st, 1, tpk, tpv, tk, tv, p, plan));
  return IRIS_OK;
}

template <typename T, int D>
int launch(const Params& p, int dtype, void* workspace, int64_t workspace_bytes, cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(p.batch) * p.n * p.heads_q;
  IRIS_REQUIRE(rows < (1ll << 31), "prefix_attn_fwd: too many rows");
  Plan plan;
  IRIS_CHECK_STATUS(make_plan(Sizes{p.batch, p.batch / p.per_group, p.heads_q, p.heads_kv, p.n, p.n_prefix, p.n_kv, D}, &plan));
  const Room room = room_of(plan);
  const bool parts = room.tile_rows + room.step_rows > 0;
  if (parts) {
    IRIS_REQUIRE(workspace != nullptr && aligned16(workspace) && workspace_bytes >= room_bytes(room, D),
                 "prefix_attn_fwd: workspace too small");
    float* at = static_cast<float*>(workspace);
    if (room.tile_rows > 0) plan.tile_sums = at;
    at += room.tile_rows * D;
    if (room.step_rows > 0) plan.step_sums = at;
    at += room.step_rows * D;
    plan.tile_states = reinterpret_cast<float2*>(at);
    plan.step_states = plan.tile_states + room.tile_rows;
  }
  if (plan.step_rows == 16) IRIS_CHECK_STATUS((launch_rows<T, D, 2>(p, plan, dtype, st)));
  else IRIS_CHECK_STATUS((launch_rows<T, D, 1>(p, plan, dtype, st)));
  if (parts) {
    const int64_t blocks = joined_tiles(plan) * (BQ / 4);
    IRIS_REQUIRE(blocks < (1ll << 31), "prefix_attn_fwd: too many rows");
    IRIS_CUDA(launch_early(join_kernel<T, D>, dim3(static_cast<unsigned>(blocks)), 128, 0, st, 1, p, plan));
  }
  return IRIS_OK;
}

inline int64_t bound(int64_t v) { return v < 0 || v > kNoBound ? kNoBound : v; }

inline int check_sizes(const iris_prefix_problem& q) {
  IRIS_REQUIRE(q.dtype == IRIS_BF16 || q.dtype == IRIS_F16, "prefix_attn_fwd: bf16 or f16");
  IRIS_REQUIRE(q.head_dim == 64 || q.head_dim == 128, "prefix_attn_fwd: head_dim must be 64 or 128");
  IRIS_REQUIRE(q.heads_q > 0 && q.heads_kv > 0 && q.heads_q % q.heads_kv == 0,
               "prefix_attn_fwd: heads_q must be a positive multiple of heads_kv");
  IRIS_REQUIRE(q.batch >= 0 && q.n >= 0 && q.n_prefix >= 0 && q.n_kv >= 0 && q.batch <= 65535 && q.heads_q <= 65535 &&
                   q.n < (1ll << 30) && q.n_prefix < (1ll << 30) && q.n_kv < (1ll << 30) && q.n_prefix + q.n_kv < (1ll << 30),
               "prefix_attn_fwd: sizes");
  IRIS_REQUIRE(q.groups >= 1 && q.batch % q.groups == 0, "prefix_attn_fwd: the batch must be a multiple of the groups");
  IRIS_REQUIRE(q.right >= -1, "prefix_attn_fwd: right is -1 (no bound) or more");
  return IRIS_OK;
}

inline bool rows_aligned(const iris_head_rows& r) {
  return aligned16(r.data) && r.stride_b % 8 == 0 && r.stride_h % 8 == 0 && r.stride_n % 8 == 0;
}
inline bool rows_apart(const iris_head_rows& r, int64_t n) {
  return r.stride_b >= 0 && r.stride_h >= 0 && (n <= 1 || r.stride_n > 0);
}

}  // namespace prefix
}  // namespace iris

using namespace iris;

extern "C" int iris_prefix_attn_workspace(const iris_prefix_problem* q, int64_t* bytes) {
  using namespace iris::prefix;
  IRIS_REQUIRE(q != nullptr && bytes != nullptr, "prefix_attn_workspace: null pointer");
  IRIS_CHECK_STATUS(check_sizes(*q));
  *bytes = 0;
  if (q->batch * q->n == 0) return IRIS_OK;
  Plan plan;
  IRIS_CHECK_STATUS(make_plan(Sizes{q->batch, q->groups, q->heads_q, q->heads_kv, q->n, q->n_prefix, q->n_kv, q->head_dim}, &plan));
  *bytes = room_bytes(room_of(plan), q->head_dim);
  return IRIS_OK;
}

extern "C" int iris_prefix_attn_fwd(const iris_prefix_problem* q, void* stream) {
  using namespace iris::prefix;
  IRIS_REQUIRE(q != nullptr, "prefix_attn_fwd: null pointer");
  IRIS_CHECK_STATUS(check_sizes(*q));
  const float scale = static_cast<float>(q->scale);
  // and so must its product with log2(e) be: 0 times infinity is NaN
  IRIS_REQUIRE(scale > 0.f && scale * 1.4426950408889634f < INFINITY, "prefix_attn_fwd: scale must be positive and finite");
  const iris_head_rows all[5] = {used_strides(q->q, q->batch, q->heads_q, q->n),
                                 used_strides(q->prefix_k, q->groups, q->heads_kv, q->n_prefix),
                                 used_strides(q->prefix_v, q->groups, q->heads_kv, q->n_prefix),
                                 used_strides(q->k, q->batch, q->heads_kv, q->n_kv),
                                 used_strides(q->v, q->batch, q->heads_kv, q->n_kv)};
  const int64_t tokens[5] = {q->n, q->n_prefix, q->n_prefix, q->n_kv, q->n_kv};
  for (int i = 0; i < 5; ++i) {
    IRIS_REQUIRE(rows_aligned(all[i]), "prefix_attn_fwd: pointers and strides must be multiples of 16 bytes");
    IRIS_REQUIRE(rows_apart(all[i], tokens[i]), "prefix_attn_fwd: rows must not repeat along the tokens");
    IRIS_REQUIRE(all[i].stride_n < (1ll << 34), "prefix_attn_fwd: rows must lie less than 2^34 elements apart");
  }
  IRIS_REQUIRE(aligned16(q->out) && q->out_stride_b % 8 == 0 && q->out_stride_n % 8 == 0,
               "prefix_attn_fwd: pointers and strides must be multiples of 16 bytes");
  if (q->batch * q->n == 0) return IRIS_OK;
  IRIS_REQUIRE(q->out, "prefix_attn_fwd: null pointer");
  for (int i = 0; i < 5; ++i) IRIS_REQUIRE(all[i].data || tokens[i] == 0, "prefix_attn_fwd: null pointer");
  Params p = {};
  p.q = all[0].data, p.pk = all[1].data, p.pv = all[2].data, p.k = all[3].data, p.v = all[4].data, p.out = q->out;
  p.qb = all[0].stride_b, p.qh = all[0].stride_h, p.qn = all[0].stride_n;
  p.pkb = all[1].stride_b, p.pkh = all[1].stride_h, p.pkn = all[1].stride_n;
  p.pvb = all[2].stride_b, p.pvh = all[2].stride_h, p.pvn = all[2].stride_n;
  p.kb = all[3].stride_b, p.kh = all[3].stride_h, p.kn = all[3].stride_n;
  p.vb = all[4].stride_b, p.vh = all[4].stride_h, p.vn = all[4].stride_n;
  p.ob = q->out_stride_b, p.on = q->out_stride_n;
  p.batch = static_cast<int>(q->batch), p.per_group = static_cast<int>(q->batch / q->groups);
  p.heads_q = static_cast<int>(q->heads_q), p.heads_kv = static_cast<int>(q->heads_kv);
  p.n = static_cast<int>(q->n), p.n_prefix = static_cast<int>(q->n_prefix), p.n_kv = static_cast<int>(q->n_kv);
  p.prefix_lengths = q->prefix_lengths, p.starts = q->starts, p.lengths = q->lengths;
  p.right = bound(q->right);
  p.scale_log2 = scale * 1.4426950408889634f;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int dtype = static_cast<int>(q->dtype);
  if (dtype == IRIS_BF16)
    return q->head_dim == 128 ? launch<__nv_bfloat16, 128>(p, dtype, q->workspace, q->workspace_bytes, st)
                              : launch<__nv_bfloat16, 64>(p, dtype, q->workspace, q->workspace_bytes, st);
  return q->head_dim == 128 ? launch<__half, 128>(p, dtype, q->workspace, q->workspace_bytes, st)
                            : launch<__half, 64>(p, dtype, q->workspace, q->workspace_bytes, st);
}
