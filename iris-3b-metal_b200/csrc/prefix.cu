// Attention of a batch whose samples share a long prefix: groups of batch / groups
// neighbouring samples have one prefix's keys and values in common and a cache of their
// own behind it. Query i of sample b (group g) sees the prefix's keys j < prefix_lengths[g]
// and its own keys j < lengths[b] with j <= starts[b] + i + right, in one softmax:
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j over both,   0 where no key is visible.
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

template <typename T, int D>
__global__ void __launch_bounds__(128) rows_kernel(const __grid_constant__ Params p) {
  grid_wait();
  grid_trigger();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= static_cast<int64_t>(p.batch) * p.n * p.heads_q) return;
  const int h = static_cast<int>(row % p.heads_q), i = static_cast<int>(row / p.heads_q % p.n);
  const int b = static_cast<int>(row / p.heads_q / p.n);
  float2 acc[D / 64];
  attend_row<T, D>(p, b, h, i, acc);
  T* o = reinterpret_cast<T*>(p.out) + b * p.ob + i * p.on + static_cast<int64_t>(h) * D + 2 * (threadIdx.x & 31);
#pragma unroll
  for (int c = 0; c < D / 64; ++c) *reinterpret_cast<uint32_t*>(o + 64 * c) = pack2<T>(acc[c].x, acc[c].y);
}

template <typename T, int D>
int launch(const Params& p, int dtype, void* workspace, int64_t workspace_bytes, cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(p.batch) * p.n * p.heads_q;
  IRIS_REQUIRE(rows < (1ll << 31), "prefix_attn_fwd: too many rows");
  IRIS_CUDA(launch_early(rows_kernel<T, D>, dim3(static_cast<unsigned>((rows + 3) / 4)), 128, 0, st, 1, p));
  return IRIS_OK;
}

inline int64_t bound(int64_t v) { return v < 0 || v > kNoBound ? kNoBound : v; }

inline int check_sizes(const iris_prefix_problem& q) {
  IRIS_REQUIRE(q.dtype == IRIS_BF16 || q.dtype == IRIS_F16, "prefix_attn_fwd: bf16 or f16");
  IRIS_REQUIRE(q.head_dim == 64 || q.head_dim == 128, "prefix_attn_fwd: head_dim must be 64 or 128");
  IRIS_REQUIRE(q.heads_q > 0 && q.heads_kv > 0 && q.heads_q % q.heads_kv == 0,
               "prefix_attn_fwd: heads_q must be a positive multiple of heads_kv");
  IRIS_REQUIRE(q.batch >= 0 && q.n >= 0 && q.n_prefix >= 0 && q.n_kv >= 0 && q.batch <= 65535 && q.heads_q <= 65535 &&
                   q.n < (1ll << 30) && q.n_prefix < (1ll << 30) && q.n_kv < (1ll << 30),
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
  return IRIS_OK;
}

extern "C" int iris_prefix_attn_fwd(const iris_prefix_problem* q, void* stream) {
  using namespace iris::prefix;
  IRIS_REQUIRE(q != nullptr, "prefix_attn_fwd: null pointer");
  IRIS_CHECK_STATUS(check_sizes(*q));
  const float scale = static_cast<float>(q->scale);
  // and so must its product with log2(e) be: 0 times infinity is NaN
  IRIS_REQUIRE(scale > 0.f && scale * 1.4426950408889634f < INFINITY, "prefix_attn_fwd: scale must be positive and finite");
  const iris_head_rows all[5] = {q->q, q->prefix_k, q->prefix_v, q->k, q->v};
  const int64_t tokens[5] = {q->n, q->n_prefix, q->n_prefix, q->n_kv, q->n_kv};
  for (int i = 0; i < 5; ++i) {
    IRIS_REQUIRE(rows_aligned(all[i]), "prefix_attn_fwd: pointers and strides must be multiples of 16 bytes");
    IRIS_REQUIRE(rows_apart(all[i], tokens[i]), "prefix_attn_fwd: rows must not repeat along the tokens");
  }
  IRIS_REQUIRE(aligned16(q->out) && q->out_stride_b % 8 == 0 && q->out_stride_n % 8 == 0,
               "prefix_attn_fwd: pointers and strides must be multiples of 16 bytes");
  if (q->batch * q->n == 0) return IRIS_OK;
  IRIS_REQUIRE(q->out, "prefix_attn_fwd: null pointer");
  for (int i = 0; i < 5; ++i) IRIS_REQUIRE(all[i].data || tokens[i] == 0, "prefix_attn_fwd: null pointer");
  Params p = {};
  p.q = q->q.data, p.pk = q->prefix_k.data, p.pv = q->prefix_v.data, p.k = q->k.data, p.v = q->v.data, p.out = q->out;
  p.qb = q->q.stride_b, p.qh = q->q.stride_h, p.qn = q->q.stride_n;
  p.pkb = q->prefix_k.stride_b, p.pkh = q->prefix_k.stride_h, p.pkn = q->prefix_k.stride_n;
  p.pvb = q->prefix_v.stride_b, p.pvh = q->prefix_v.stride_h, p.pvn = q->prefix_v.stride_n;
  p.kb = q->k.stride_b, p.kh = q->k.stride_h, p.kn = q->k.stride_n;
  p.vb = q->v.stride_b, p.vh = q->v.stride_h, p.vn = q->v.stride_n;
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
