// Rotary positions on head rows in any strides, and the same with the append
// to a key / value cache (text side: the denoiser's own heads go through
// qk_norm_rope, heads.cu). A pair (a, b) of a head row at position p becomes
// (a c - b s, a s + b c) with c, s = cos / sin[p] of that pair; pairs are
// (2 i, 2 i + 1) or (i, i + R / 2), the columns from R on are copied.
// Arithmetic in fp32, one rounding to the row's type.
//
// HBM-bound (3 flops per element read and written once). A thread owns one unit
// of a token's rows, two vectors of V elements: V neighbouring pairs (interleaved)
// or V columns and their partners R / 2 further (half), so both layouts read and
// write whole vectors. It takes that unit in several heads, so the token's table
// entries are read once for all of them.
#include "common.cuh"
#include "iris_abi_internal.h"

namespace iris {
namespace rope {

constexpr int THREADS = 256;

struct View {  // [batch, heads, n, D] rows, element strides
  const void* src;
  int64_t sb, sh, sn;
  void* dst;
  int64_t db, dh, dn;
};

struct Params {
  View q, k, v;           // rope: q alone
  int heads_q, heads_kv;  // heads_kv = 0: rope
  int n, head_dim, rotary;
  int64_t tokens;  // batch * n
  const float* cos;
  const float* sin;
  int64_t table_rows;
  const void* positions;  // rope: null, int32 or int64 [batch or 1, n]
  int64_t pos_stride;
  int pos64;
  float sign;          // -1: the inverse rotation
  const int* starts;   // append: position of each sample's first row
  const int* counts;   // append: rows of each sample, or null (all n)
  int64_t capacity;    // append: slots of the cache
  int64_t sinks;       // append: -1 plain cache, else slots that a rolling cache never overwrites
  bool zero_rest;      // append: zeros in out's rows from counts[b] on
  int units, hslots, tokens_per_block;
};

template <typename T>
IRIS_DEVICE float to_f32(T v);
template <>
IRIS_DEVICE float to_f32(float v) { return v; }
template <>
IRIS_DEVICE float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
IRIS_DEVICE float to_f32(__half v) { return __half2float(v); }
template <typename T>
IRIS_DEVICE T from_f32(float v);
template <>
IRIS_DEVICE float from_f32(float v) { return v; }
template <>
IRIS_DEVICE __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <>
IRIS_DEVICE __half from_f32(float v) { return __float2half_rn(v); }

// The turned pair, contracted the same way in every variant: a row's bits do not
// depend on its alignment.
IRIS_DEVICE float turn_a(float a, float b, float c, float s) { return fmaf(a, c, -__fmul_rn(b, s)); }
IRIS_DEVICE float turn_b(float a, float b, float c, float s) { return fmaf(a, s, __fmul_rn(b, c)); }

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T e[V];
};

// Slot of position p, or -1 where it is not kept. `last`: the sample's last new
// position; a rolling cache skips tokens whose slot a later one of the call takes.
IRIS_DEVICE int64_t cache_slot(const Params& a, int64_t p, int64_t last, bool* bad) {
  if (a.sinks < 0) {
    *bad = p >= a.capacity;
    return *bad ? -1 : p;
  }
  const int64_t turn = a.capacity - a.sinks;
  if (p < a.sinks) return p;
  if (p + turn <= last) return -1;
  return a.sinks + (p - a.sinks) % turn;
}

template <typename T, int V, bool HALF, bool APPEND>
__global__ void __launch_bounds__(THREADS) rope_kernel(const __grid_constant__ Params a) {
  const int items = a.tokens_per_block * a.hslots * a.units;
  const int heads = a.heads_q + 2 * a.heads_kv;
  for (int item = threadIdx.x; item < items; item += THREADS) {
    const int u = item % a.units;
    const int rest = item / a.units;
    const int slot = rest % a.hslots;
    const int64_t token = static_cast<int64_t>(blockIdx.x) * a.tokens_per_block + rest / a.hslots;
    if (token >= a.tokens) return;
    const int b = static_cast<int>(token / a.n), t = static_cast<int>(token - static_cast<int64_t>(b) * a.n);
    int64_t p = t, row = t;  // position; row of the cache
    bool bad = false;
    if constexpr (APPEND) {
      const int64_t first = a.starts[b];
      const int64_t count = a.counts ? min(a.counts[b], a.n) : a.n;
      if (t >= count) {
        if (!a.zero_rest) continue;
        const Vec<T, V> none = {};
        for (int h = slot; h < a.heads_q; h += a.hslots) {
          T* dst = reinterpret_cast<T*>(a.q.dst) + b * a.q.db + h * a.q.dh + t * a.q.dn + u * 2 * V;
          *reinterpret_cast<Vec<T, V>*>(dst) = none;
          *reinterpret_cast<Vec<T, V>*>(dst + V) = none;
        }
        continue;
      }
      p = first + t;
      bad = p < 0 || p >= a.table_rows;
      bool full = false;
      row = bad ? -1 : cache_slot(a, p, first + count - 1, &full);
      if ((bad || full) && u == 0 && slot == 0) atomicOr(&g_device_error, kErrBadArgument);
    } else {
      if (a.positions) {
        const int64_t at = b * a.pos_stride + t;
        p = a.pos64 ? reinterpret_cast<const int64_t*>(a.positions)[at] : reinterpret_cast<const int*>(a.positions)[at];
      }
      bad = p < 0 || p >= a.table_rows;
      if (bad && u == 0 && slot == 0) atomicOr(&g_device_error, kErrBadArgument);
    }
    const bool turns = u * 2 * V < a.rotary;  // a unit past the rotated columns is copied
    // the unit's two vectors: first and second elements of its pairs (half layout), or one run of pairs
    const int c0 = !turns ? u * 2 * V : HALF ? u * V : u * 2 * V;
    const int c1 = turns && HALF ? a.rotary / 2 + u * V : c0 + V;
    float cs[V], sn[V];
    if (turns) {
      const int64_t at = (bad ? 0 : p) * (a.rotary / 2) + u * V;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        cs[i] = bad ? __int_as_float(0x7fc00000) : __ldg(a.cos + at + i);  // a position outside the table: NaN
        sn[i] = a.sign * __ldg(a.sin + at + i);
      }
    }
    for (int h = slot; h < heads; h += a.hslots) {
      const bool isq = !APPEND || h < a.heads_q;
      const bool isv = APPEND && h >= a.heads_q + a.heads_kv;
      const View& w = isq ? a.q : isv ? a.v : a.k;
      const int hh = isq ? h : isv ? h - a.heads_q - a.heads_kv : h - a.heads_q;
      if (!isq && row < 0) continue;
      const T* src = reinterpret_cast<const T*>(w.src) + b * w.sb + hh * w.sh + t * w.sn;
      T* dst = reinterpret_cast<T*>(w.dst) + b * w.db + hh * w.dh + (isq ? t : row) * w.dn;
      Vec<T, V> x = *reinterpret_cast<const Vec<T, V>*>(src + c0), y = *reinterpret_cast<const Vec<T, V>*>(src + c1);
      if (turns && !isv) {
        if constexpr (HALF || V == 1) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float f = to_f32(x.e[i]), g = to_f32(y.e[i]);
            x.e[i] = from_f32<T>(turn_a(f, g, cs[i], sn[i]));
            y.e[i] = from_f32<T>(turn_b(f, g, cs[i], sn[i]));
          }
        } else {
#pragma unroll
          for (int i = 0; i < V / 2; ++i) {
            float f = to_f32(x.e[2 * i]), g = to_f32(x.e[2 * i + 1]);
            x.e[2 * i] = from_f32<T>(turn_a(f, g, cs[i], sn[i]));
            x.e[2 * i + 1] = from_f32<T>(turn_b(f, g, cs[i], sn[i]));
            f = to_f32(y.e[2 * i]), g = to_f32(y.e[2 * i + 1]);
            y.e[2 * i] = from_f32<T>(turn_a(f, g, cs[V / 2 + i], sn[V / 2 + i]));
            y.e[2 * i + 1] = from_f32<T>(turn_b(f, g, cs[V / 2 + i], sn[V / 2 + i]));
          }
        }
      }
      *reinterpret_cast<Vec<T, V>*>(dst + c0) = x;
      *reinterpret_cast<Vec<T, V>*>(dst + c1) = y;
    }
  }
}

// Elements per vector: 16 bytes where every row, stride and the rotated part
// allow it, else 8 bytes, else single elements.
inline bool fits(const View& w, int64_t elems, int64_t size) {
  return w.src == nullptr || (aligned_n(w.src, elems * size) && aligned_n(w.dst, elems * size) && w.sb % elems == 0 &&
                              w.sh % elems == 0 && w.sn % elems == 0 && w.db % elems == 0 && w.dh % elems == 0 &&
                              w.dn % elems == 0);
}

template <typename T, int V, bool APPEND>
int launch_v(Params& a, bool half, cudaStream_t st) {
  a.units = a.head_dim / (2 * V);
  const int heads = a.heads_q + 2 * a.heads_kv;
  a.hslots = heads;
  a.tokens_per_block = THREADS / (a.units * a.hslots);
  if (a.tokens_per_block < 1) a.tokens_per_block = 1;
  const int64_t blocks = (a.tokens + a.tokens_per_block - 1) / a.tokens_per_block;
  if (half)
    rope_kernel<T, V, true, APPEND><<<static_cast<unsigned>(blocks), THREADS, 0, st>>>(a);
  else
    rope_kernel<T, V, false, APPEND><<<static_cast<unsigned>(blocks), THREADS, 0, st>>>(a);
  IRIS_CUDA(cudaGetLastError());
  return IRIS_OK;
}

template <typename T, bool APPEND>
int launch(Params& a, bool half, cudaStream_t st) {
  constexpr int S = sizeof(T), W = 16 / S;
  auto ok = [&](int v) {
    return a.rotary % (2 * v) == 0 && a.head_dim % (2 * v) == 0 && fits(a.q, v, S) && fits(a.k, v, S) && fits(a.v, v, S);
  };
  if (ok(W)) return launch_v<T, W, APPEND>(a, half, st);
  if (ok(W / 2)) return launch_v<T, W / 2, APPEND>(a, half, st);
  return launch_v<T, 1, APPEND>(a, half, st);
}

template <bool APPEND>
int dispatch(Params& a, int64_t dtype, bool half, void* stream) {
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == IRIS_F32) return launch<float, APPEND>(a, half, st);
  if (dtype == IRIS_BF16) return launch<__nv_bfloat16, APPEND>(a, half, st);
  return launch<__half, APPEND>(a, half, st);
}

inline int check(int64_t dtype, int64_t batch, int64_t heads, int64_t n, int64_t head_dim, int64_t rotary,
                 int64_t table_rows, int64_t layout) {
  IRIS_REQUIRE(dtype >= IRIS_F32 && dtype <= IRIS_F16, "rope: bad dtype");
  IRIS_REQUIRE(batch >= 0 && n >= 0 && heads > 0 && batch < (1ll << 31) && n < (1ll << 31) && batch * n < (1ll << 31),
               "rope: bad row counts");
  IRIS_REQUIRE(heads <= 65536 && head_dim > 0 && head_dim <= 4096 && head_dim % 2 == 0, "rope: head_dim must be even, at most 4096");
  IRIS_REQUIRE(rotary > 0 && rotary % 2 == 0 && rotary <= head_dim, "rope: the rotated columns must be even, at most head_dim");
  IRIS_REQUIRE(table_rows > 0, "rope: empty table");
  IRIS_REQUIRE(layout == IRIS_ROPE_INTERLEAVED || layout == IRIS_ROPE_HALF, "rope: bad layout");
  return IRIS_OK;
}

}  // namespace rope
}  // namespace iris

using namespace iris;

namespace {
iris::rope::View view(const iris_head_rows& from, const iris_head_rows& to) {
  return iris::rope::View{from.data, from.stride_b, from.stride_h, from.stride_n, to.data, to.stride_b, to.stride_h, to.stride_n};
}
}  // namespace

extern "C" int iris_rope(const iris_rope_problem* q, void* stream) {
  using namespace iris::rope;
  IRIS_REQUIRE(q != nullptr, "rope: null pointer");
  IRIS_CHECK_STATUS(check(q->dtype, q->batch, q->heads, q->n, q->head_dim, q->rotary, q->table_rows, q->layout));
  if (q->batch * q->n == 0) return IRIS_OK;
  IRIS_REQUIRE(q->x.data && q->out.data && q->cos && q->sin, "rope: null pointer");
  Params a = {};
  a.q = view(q->x, q->out);
  a.heads_q = static_cast<int>(q->heads);
  a.n = static_cast<int>(q->n);
  a.head_dim = static_cast<int>(q->head_dim);
  a.rotary = static_cast<int>(q->rotary);
  a.tokens = q->batch * q->n;
  a.cos = q->cos;
  a.sin = q->sin;
  a.table_rows = q->table_rows;
  a.positions = q->positions;
  a.pos_stride = q->positions_stride;
  a.pos64 = q->positions_64 != 0;
  a.sign = q->inverse ? -1.f : 1.f;
  return dispatch<false>(a, q->dtype, q->layout == IRIS_ROPE_HALF, stream);
}

extern "C" int iris_rope_append(const iris_append_problem* q, void* stream) {
  using namespace iris::rope;
  IRIS_REQUIRE(q != nullptr, "rope_append: null pointer");
  IRIS_CHECK_STATUS(check(q->dtype, q->batch, q->heads_q, q->n, q->head_dim, q->rotary, q->table_rows, q->layout));
  IRIS_REQUIRE(q->heads_kv > 0 && q->heads_kv <= 65536, "rope_append: bad head counts");
  IRIS_REQUIRE(q->capacity > 0 && q->sinks >= -1 && q->sinks < q->capacity,
               "rope_append: a rolling cache needs more slots than sinks");
  if (q->batch * q->n == 0) return IRIS_OK;
  IRIS_REQUIRE(q->q.data && q->k.data && q->v.data && q->out.data && q->k_cache.data && q->v_cache.data && q->cos &&
                   q->sin && q->starts,
               "rope_append: null pointer");
  Params a = {};
  a.q = view(q->q, q->out);
  a.k = view(q->k, q->k_cache);
  a.v = view(q->v, q->v_cache);
  a.heads_q = static_cast<int>(q->heads_q);
  a.heads_kv = static_cast<int>(q->heads_kv);
  a.n = static_cast<int>(q->n);
  a.head_dim = static_cast<int>(q->head_dim);
  a.rotary = static_cast<int>(q->rotary);
  a.tokens = q->batch * q->n;
  a.cos = q->cos;
  a.sin = q->sin;
  a.table_rows = q->table_rows;
  a.sign = 1.f;
  a.starts = q->starts;
  a.counts = q->counts;
  a.capacity = q->capacity;
  a.sinks = q->sinks;
  a.zero_rest = q->zero_rest != 0;
  return dispatch<true>(a, q->dtype, q->layout == IRIS_ROPE_HALF, stream);
}
