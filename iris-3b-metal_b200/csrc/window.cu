// Attention with a window and first tokens that stay visible, for a text side's
// prompts, chunks and single tokens over a cache (the denoiser's own attention,
// attention.cu, is unmasked). Query i of sample b is at position p = starts[b] + i;
// it sees key j < lengths[b] where j <= p + right and (j >= p - left or j < sinks):
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j,   0 where no key is visible.
// A row's visible keys are two runs, [0, early) and [lo, hi) (struct Span).
#include <math.h>

#include "common.cuh"
#include "iris_abi_internal.h"

namespace iris {
namespace window {

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

template <typename T>
IRIS_DEVICE float2 unpack2(uint32_t v);
template <>
IRIS_DEVICE float2 unpack2<__nv_bfloat16>(uint32_t v) { return unpack_bf16x2(v); }
template <>
IRIS_DEVICE float2 unpack2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
template <typename T>
IRIS_DEVICE uint32_t pack2(float a, float b);
template <>
IRIS_DEVICE uint32_t pack2<__nv_bfloat16>(float a, float b) { return pack_bf16x2(a, b); }
template <>
IRIS_DEVICE uint32_t pack2<__half>(float a, float b) { return pack_f16x2(a, b); }

// One output row by one warp, keys 32 at a time (a lane scores one), from global
// memory: columns [64 c + 2 lane, + 2) of chunk c < D / 64. Only visible keys are
// read, so what lies in masked places cannot reach the row.
template <typename T, int D>
IRIS_DEVICE void attend_row(const Params& p, int b, int h, int i, float2 (&acc)[D / 64]) {
  const int lane = threadIdx.x & 31;
  const int hk = h / (p.heads_q / p.heads_kv);
  const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) + b * p.qb + h * p.qh + i * p.qn);
  const T* k = reinterpret_cast<const T*>(p.k) + b * p.kb + hk * p.kh;
  const T* v = reinterpret_cast<const T*>(p.v) + b * p.vb + hk * p.vh;
  const Span s = visible(p, sample_start(p, b) + i, sample_length(p, b));
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
          dot = fmaf(f.x, g.x, fmaf(f.y, g.y, dot));
        }
      }
    }
    const float score = real ? dot * p.scale_log2 : -INFINITY;
    float top = score;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float m_new = fmaxf(m, top);
    const float base = m_new == -INFINITY ? 0.f : m_new;  // nothing above -inf so far: every weight 0
    const float w = real ? exp2f(score - base) : 0.f;
    const float corr = m == -INFINITY ? 0.f : exp2f(m - base);
    l = l * corr + warp_sum(w);
    m = m_new;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) acc[c] = make_float2(acc[c].x * corr, acc[c].y * corr);
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
  const float inv = count == 0 ? 0.f : 1.f / l;
#pragma unroll
  for (int c = 0; c < D / 64; ++c)
    acc[c] = count == 0 ? make_float2(0.f, 0.f) : l == 0.f ? make_float2(NAN, NAN) : make_float2(acc[c].x * inv, acc[c].y * inv);
}

constexpr int ROW_WARPS = 8;

template <typename T, int D>
__global__ void __launch_bounds__(ROW_WARPS * 32) rows_kernel(const __grid_constant__ Params p) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * ROW_WARPS + (threadIdx.x >> 5);
  const int64_t per_sample = static_cast<int64_t>(p.heads_q) * p.n;
  if (row >= p.batch * per_sample) return;
  const int b = static_cast<int>(row / per_sample);
  const int64_t rest = row - b * per_sample;
  const int i = static_cast<int>(rest / p.heads_q), h = static_cast<int>(rest - static_cast<int64_t>(i) * p.heads_q);
  float2 acc[D / 64];
  attend_row<T, D>(p, b, h, i, acc);
  T* o = reinterpret_cast<T*>(p.out) + b * p.ob + i * p.on + static_cast<int64_t>(h) * D + 2 * (threadIdx.x & 31);
#pragma unroll
  for (int c = 0; c < D / 64; ++c) *reinterpret_cast<uint32_t*>(o + 64 * c) = pack2<T>(acc[c].x, acc[c].y);
}

template <typename T, int D>
int launch(const Params& p, cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(p.batch) * p.heads_q * p.n;
  const int64_t blocks = (rows + ROW_WARPS - 1) / ROW_WARPS;
  IRIS_REQUIRE(blocks < (1ll << 31), "window_attn_fwd: too many rows");
  rows_kernel<T, D><<<static_cast<unsigned>(blocks), ROW_WARPS * 32, 0, st>>>(p);
  IRIS_CUDA(cudaGetLastError());
  return IRIS_OK;
}

}  // namespace window
}  // namespace iris

using namespace iris;

extern "C" int iris_window_attn_fwd(const void* q, const void* k, const void* v, void* out, int dtype, int64_t batch,
                                    int64_t heads_q, int64_t heads_kv, int64_t n, int64_t n_kv, int64_t head_dim,
                                    int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_n, int64_t k_stride_b,
                                    int64_t k_stride_h, int64_t k_stride_n, int64_t v_stride_b, int64_t v_stride_h,
                                    int64_t v_stride_n, int64_t out_stride_b, int64_t out_stride_n, const int* starts,
                                    const int* lengths, int64_t left, int64_t right, int64_t sinks, float scale,
                                    void* stream) {
  using namespace iris::window;
  IRIS_REQUIRE(dtype == IRIS_BF16 || dtype == IRIS_F16, "window_attn_fwd: bf16 or f16");
  IRIS_REQUIRE(head_dim == 64 || head_dim == 128, "window_attn_fwd: head_dim must be 64 or 128");
  IRIS_REQUIRE(heads_q > 0 && heads_kv > 0 && heads_q % heads_kv == 0,
               "window_attn_fwd: heads_q must be a positive multiple of heads_kv");
  IRIS_REQUIRE(batch >= 0 && n >= 0 && n_kv >= 0 && batch <= 65535 && heads_q <= 65535 && n < (1ll << 30) &&
                   n_kv < (1ll << 30),
               "window_attn_fwd: sizes");
  IRIS_REQUIRE(left >= -1 && right >= -1 && sinks >= 0, "window_attn_fwd: window bounds are -1 (none) or more");
  IRIS_REQUIRE(scale > 0.f && scale < INFINITY, "window_attn_fwd: scale must be positive and finite");
  IRIS_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out) && q_stride_b % 8 == 0 &&
                   q_stride_h % 8 == 0 && q_stride_n % 8 == 0 && k_stride_b % 8 == 0 && k_stride_h % 8 == 0 &&
                   k_stride_n % 8 == 0 && v_stride_b % 8 == 0 && v_stride_h % 8 == 0 && v_stride_n % 8 == 0 &&
                   out_stride_b % 8 == 0 && out_stride_n % 8 == 0,
               "window_attn_fwd: pointers and strides must be multiples of 16 bytes");
  if (batch * n == 0) return IRIS_OK;
  IRIS_REQUIRE(q && out && ((k && v) || n_kv == 0), "window_attn_fwd: null pointer");
  Params p = {};
  p.q = q, p.k = k, p.v = v, p.out = out;
  p.qb = q_stride_b, p.qh = q_stride_h, p.qn = q_stride_n;
  p.kb = k_stride_b, p.kh = k_stride_h, p.kn = k_stride_n;
  p.vb = v_stride_b, p.vh = v_stride_h, p.vn = v_stride_n;
  p.ob = out_stride_b, p.on = out_stride_n;
  p.batch = static_cast<int>(batch), p.heads_q = static_cast<int>(heads_q), p.heads_kv = static_cast<int>(heads_kv);
  p.n = static_cast<int>(n), p.n_kv = static_cast<int>(n_kv);
  p.starts = starts, p.lengths = lengths;
  p.left = left < 0 || left > kNoBound ? kNoBound : left;
  p.right = right < 0 || right > kNoBound ? kNoBound : right;
  p.sinks = static_cast<int>(sinks < n_kv ? sinks : n_kv);
  p.scale_log2 = scale * 1.4426950408889634f;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == IRIS_BF16)
    return head_dim == 128 ? launch<__nv_bfloat16, 128>(p, st) : launch<__nv_bfloat16, 64>(p, st);
  return head_dim == 128 ? launch<__half, 128>(p, st) : launch<__half, 64>(p, st);
}
