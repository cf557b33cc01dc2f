// Rotary positions on head rows in any strides, and the same with the append
// to a key / value cache (text side: the denoiser's own heads go through
// qk_norm_rope, heads.cu). A pair (a, b) of a head row at position p becomes
// (a c - b s, a s + b c) with c, s = cos / sin[p] of that pair; pairs are
// (2 i, 2 i + 1) or (i, i + R / 2), the columns from R on are copied.
// Arithmetic in fp32, one rounding to the row's type.
//
// HBM-bound (3 flops per element read and written once), as long as few instructions
// are spent on finding the element. A thread owns one unit of a token's rows, two
// vectors of V elements: V neighbouring pairs (interleaved) or V columns and their
// partners R / 2 further (half), so both layouts read and write whole vectors. Where
// there are threads to spare it takes that unit in EACH = 4 heads of one tensor, their
// loads in flight together and the token's table entries read once for them. Slots
// are the heads of a tensor that its threads begin at: `step` of them.
//
// Measured: 25 fp32 heads of 16384 tokens 67 us (6.3 TB/s, 0.97 of a plain copy); 8 x
// 300 bf16 tokens, rows in L2, 7.7 us (4.0 TB/s); one token appended 2.3 us on the
// device. Four heads a thread against one: 67 / 69 us, the append of 8 x 301 f16
// tokens 5.4 / 6.0 us where there are threads to spare.
#include "common.cuh"
#include "iris_abi_internal.h"

namespace iris {
namespace rope {

constexpr int THREADS = 256;
constexpr int64_t SPARE_THREADS = 4096;  // per SM, from which a thread takes four heads

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
  int units;           // of a row
  int step_q, step_kv;  // slots of q; of k and of v
  int items;           // units * slots of a token
  int tokens_per_block;
  unsigned by_units, by_items;  // ceil(2^20 / d): exact quotients of numbers below 1024
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
template <typename T>
IRIS_DEVICE void turn(T& a, T& b, float c, float s) {
  const float f = to_f32(a), g = to_f32(b);
  a = from_f32<T>(fmaf(f, c, -__fmul_rn(g, s)));
  b = from_f32<T>(fmaf(f, s, __fmul_rn(g, c)));
}

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T e[V];
};

// Slot of position p, or -1 where it is not kept. `last`: the sample's last position
// that the call appends (none behind the tables); a rolling cache skips tokens whose slot
// a later one of the call takes.
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

template <int V>
IRIS_DEVICE void load_floats(const float* p, float (&v)[V]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 f = *reinterpret_cast<const float4*>(p + i);
      v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = p[i];
  }
}

template <typename T, int V, bool HALF, bool APPEND, int EACH>
__global__ void __launch_bounds__(THREADS) rope_kernel(const __grid_constant__ Params a) {
  grid_wait();
  grid_trigger();
  // rows wider than the block's threads take several turns
  for (unsigned item = threadIdx.x; item < static_cast<unsigned>(a.tokens_per_block * a.items); item += THREADS) {
    const unsigned local = a.items <= THREADS ? (item * a.by_items) >> 20 : 0u;
    const unsigned rest = item - local * a.items;
    const int slot0 = a.items <= THREADS ? static_cast<int>((rest * a.by_units) >> 20) : static_cast<int>(rest / a.units);
    const int u = static_cast<int>(rest) - slot0 * a.units;
    const unsigned token = blockIdx.x * static_cast<unsigned>(a.tokens_per_block) + local;
    if (token >= a.tokens) return;
    const int b = static_cast<int>(token / static_cast<unsigned>(a.n)), t = static_cast<int>(token) - b * a.n;
    // the tensor of this slot, and its first head
    const bool isq = !APPEND || slot0 < a.step_q, isv = APPEND && slot0 >= a.step_q + a.step_kv;
    const View& w = isq ? a.q : isv ? a.v : a.k;
    const int heads = isq ? a.heads_q : a.heads_kv, step = isq ? a.step_q : a.step_kv;
    const int head = isq ? slot0 : isv ? slot0 - a.step_q - a.step_kv : slot0 - a.step_q;
    int64_t p = t, row = t;  // position; row of the target
    bool bad = false;
    if constexpr (APPEND) {
      const int64_t first = a.starts[b];
      const int64_t count = a.counts ? min(a.counts[b], a.n) : a.n;
      if (t >= count) {
        if (isq && a.zero_rest) {
          const Vec<T, V> none = {};
          T* dst = reinterpret_cast<T*>(w.dst) + b * w.db + t * w.dn + u * 2 * V;
          for (int h = head; h < heads; h += step) {
            *reinterpret_cast<Vec<T, V>*>(dst + h * w.dh) = none;
            *reinterpret_cast<Vec<T, V>*>(dst + h * w.dh + V) = none;
          }
        }
        continue;
      }
      p = first + t;
      bad = p < 0 || p >= a.table_rows;
      bool full = false;
      const int64_t kept = bad ? -1 : cache_slot(a, p, min(first + count, a.table_rows) - 1, &full);
      if ((bad || full) && u == 0 && slot0 == 0) atomicOr(&g_device_error, kErrBadArgument);
      if (!isq) {
        if (kept < 0) continue;
        row = kept;
      }
    } else {
      if (a.positions) {
        const int64_t at = b * a.pos_stride + t;
        p = a.pos64 ? reinterpret_cast<const int64_t*>(a.positions)[at] : reinterpret_cast<const int*>(a.positions)[at];
      }
      bad = p < 0 || p >= a.table_rows;
      if (bad && u == 0 && slot0 == 0) atomicOr(&g_device_error, kErrBadArgument);
    }
    const bool turns = u * 2 * V < a.rotary && !isv;  // a unit past the rotated columns is copied, and so is v
    // the unit's two vectors: first and second elements of its pairs (half layout), or one run of pairs
    const int c0 = turns && HALF ? u * V : u * 2 * V;
    const int c1 = turns && HALF ? a.rotary / 2 + u * V : c0 + V;
    const T* src = reinterpret_cast<const T*>(w.src) + b * w.sb + t * w.sn + head * w.sh;
    T* dst = reinterpret_cast<T*>(w.dst) + b * w.db + row * w.dn + head * w.dh;
    Vec<T, V> x[EACH], y[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      if (j > 0 && head + j * step >= heads) break;
      const T* from = src + j * step * w.sh;
      x[j] = *reinterpret_cast<const Vec<T, V>*>(from + c0);
      y[j] = *reinterpret_cast<const Vec<T, V>*>(from + c1);
    }
    float cs[V], sn[V];
    if (turns) {
      const int64_t at = (bad ? 0 : p) * (a.rotary / 2) + u * V;
      load_floats<V>(a.cos + at, cs);
      load_floats<V>(a.sin + at, sn);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        sn[i] *= a.sign;
        if (bad) cs[i] = __int_as_float(0x7fc00000);  // a position outside the table: NaN
      }
    }
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      if (j > 0 && head + j * step >= heads) break;
      if (turns) {
        if constexpr (HALF || V == 1) {
#pragma unroll
          for (int i = 0; i < V; ++i) turn(x[j].e[i], y[j].e[i], cs[i], sn[i]);
        } else {
#pragma unroll
          for (int i = 0; i < V / 2; ++i) {
            turn(x[j].e[2 * i], x[j].e[2 * i + 1], cs[i], sn[i]);
            turn(y[j].e[2 * i], y[j].e[2 * i + 1], cs[V / 2 + i], sn[V / 2 + i]);
          }
        }
      } else if (bad) {  // the whole row is NaN, its copied columns too
#pragma unroll
        for (int i = 0; i < V; ++i) x[j].e[i] = y[j].e[i] = from_f32<T>(__int_as_float(0x7fc00000));
      }
      T* to = dst + j * step * w.dh;
      *reinterpret_cast<Vec<T, V>*>(to + c0) = x[j];
      *reinterpret_cast<Vec<T, V>*>(to + c1) = y[j];
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

template <typename T, int V, bool APPEND, int EACH>
int launch_each(Params& a, bool half, cudaStream_t st) {
  a.units = a.head_dim / (2 * V);
  a.step_q = (a.heads_q + EACH - 1) / EACH;
  a.step_kv = (a.heads_kv + EACH - 1) / EACH;
  a.items = a.units * (a.step_q + 2 * a.step_kv);
  a.tokens_per_block = a.items <= THREADS ? THREADS / a.items : 1;
  a.by_units = ((1u << 20) + a.units - 1) / a.units;
  a.by_items = ((1u << 20) + a.items - 1) / a.items;
  const int64_t blocks = (a.tokens + a.tokens_per_block - 1) / a.tokens_per_block;
  auto kernel = half ? rope_kernel<T, V, true, APPEND, EACH> : rope_kernel<T, V, false, APPEND, EACH>;
  IRIS_CUDA(launch_early(kernel, dim3(static_cast<unsigned>(blocks)), THREADS, 0, st, 1, a));
  return IRIS_OK;
}

template <typename T, int V, bool APPEND>
int launch_v(Params& a, bool half, cudaStream_t st) {
  const int64_t threads = a.tokens * (a.head_dim / (2 * V)) * (a.heads_q + 2 * a.heads_kv);
  if (threads >= static_cast<int64_t>(num_sms()) * SPARE_THREADS) return launch_each<T, V, APPEND, 4>(a, half, st);
  return launch_each<T, V, APPEND, 1>(a, half, st);
}

template <typename T, bool APPEND>
int launch(Params& a, bool half, cudaStream_t st) {
  constexpr int S = sizeof(T), W = 16 / S;
  auto ok = [&](int v) {
    return a.rotary % (2 * v) == 0 && a.head_dim % (2 * v) == 0 && fits(a.q, v, S) && fits(a.k, v, S) && fits(a.v, v, S) &&
           aligned16(a.cos) && aligned16(a.sin);
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
