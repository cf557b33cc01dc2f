// CPython module of the text side's calls: argument checks, outputs and the launch.
// They run once per token, and a single token's kernels take a few microseconds; the
// same checks in Python with a ctypes call took 10 to 16 us of host time per call, here
// they take about 5 (torch's own x + x: 4.5). The kernels stay behind the C ABI, whose
// addresses iris_b200._lib binds here; every failed check raises ValueError before any
// launch.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <optional>
#include <stdexcept>
#include <string>

#include "../../include/iris_b200.h"

namespace {

struct Refused : std::runtime_error {  // becomes ValueError
  using std::runtime_error::runtime_error;
};
struct Raised {};  // a Python exception is set

inline void require(bool ok, const char* message) {
  if (!ok) throw Refused(message);
}

struct Entries {
  decltype(&iris_rope) rope;
  decltype(&iris_rope_append) rope_append;
  decltype(&iris_window_attn_fwd) window_attn_fwd;
  decltype(&iris_window_attn_workspace) window_attn_workspace;
  decltype(&iris_gemv_q4) gemv_q4;
  decltype(&iris_last_error) last_error;
} entries = {};
long long launches = 0;

const at::Tensor& tensor(PyObject* o, const char* message) {
  if (!THPVariable_Check(o)) throw Refused(message);
  return THPVariable_Unpack(o);
}
// None: no tensor
const at::Tensor* maybe(PyObject* o, const char* message) { return o == Py_None ? nullptr : &tensor(o, message); }

int64_t whole(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised{};
  return v != 0;
}

int64_t type_code(at::ScalarType t) {
  if (t == at::kFloat) return IRIS_F32;
  if (t == at::kBFloat16) return IRIS_BF16;
  if (t == at::kHalf) return IRIS_F16;
  throw Refused(std::string("unsupported dtype ") + c10::toString(t));
}

int64_t rope_layout(PyObject* o) {
  if (PyUnicode_Check(o)) {
    if (PyUnicode_CompareWithASCIIString(o, "interleaved") == 0) return IRIS_ROPE_INTERLEAVED;
    if (PyUnicode_CompareWithASCIIString(o, "half") == 0) return IRIS_ROPE_HALF;
  }
  throw Refused("layout must be \"half\" or \"interleaved\"");
}

// Address and strides (0 for a lone row: its stride says nothing) of head rows
// [batch, heads, n, dim] that are contiguous along dim.
iris_head_rows head_rows(const at::Tensor& t, int64_t batch, int64_t heads, int64_t n, int64_t dim, const char* message) {
  const auto size = t.sizes();
  if (size.size() != 4 || size[0] != batch || size[1] != heads || size[2] != n || size[3] != dim) throw Refused(message);
  const auto stride = t.strides();
  require(stride[3] == 1 || dim == 1, "head rows must be contiguous");
  return iris_head_rows{t.data_ptr(), batch > 1 ? stride[0] : 0, heads > 1 ? stride[1] : 0, n > 1 ? stride[2] : 0};
}

// Outputs take every element once: two writes to one place would be a race, as would
// a write to what other threads of the call still read.
void writable(const at::Tensor& t) {
  const int64_t dims = t.dim();
  for (int64_t d = 0; d < dims; ++d) {
    if (t.size(d) <= 1) continue;
    require(t.stride(d) != 0, "an output must not be an expanded view");
    // rows apart: each stride steps over all that the dimensions of smaller strides span
    int64_t span = 1;
    for (int64_t e = 0; e < dims; ++e)
      if (t.stride(e) < t.stride(d)) span += (t.size(e) - 1) * t.stride(e);
      else require(e == d || t.size(e) <= 1 || t.stride(e) != t.stride(d), "an output's rows must not overlap");
    require(t.numel() == 0 || t.stride(d) >= span, "an output's rows must not overlap");
  }
}

// Whether both hold an element for certain: the same first one, or dense tensors whose
// ranges meet (views of one buffer that interleave are the caller's to keep apart).
bool share(const at::Tensor& a, const at::Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const char *x = static_cast<const char*>(a.data_ptr()), *y = static_cast<const char*>(b.data_ptr());
  if (x == y) return true;
  return a.is_non_overlapping_and_dense() && b.is_non_overlapping_and_dense() && x < y + b.nbytes() && y < x + a.nbytes();
}

bool same_rows(const at::Tensor& a, const at::Tensor& b) {
  if (a.data_ptr() != b.data_ptr() || a.sizes() != b.sizes()) return false;
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}

const int* int32_rows(const at::Tensor* t, int64_t batch, const char* message) {
  if (t == nullptr) return nullptr;
  if (t->scalar_type() != at::kInt || t->dim() != 1 || t->size(0) != batch || !t->is_contiguous()) throw Refused(message);
  return static_cast<const int*>(t->data_ptr());
}

// The tables of rotary positions: rows, and the columns that turn.
void tables(const at::Tensor& cos, const at::Tensor& sin, int64_t dim, int64_t* rows, int64_t* rotary) {
  require(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat && cos.is_contiguous() && sin.is_contiguous(),
          "rotary tables must be contiguous FP32");
  require(cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.size(0) > 0 && cos.size(1) > 0 && 2 * cos.size(1) <= dim,
          "rotary tables must be [positions, rotary / 2] with rotary <= head_dim");
  *rows = cos.size(0);
  *rotary = 2 * cos.size(1);
}

// The CUDA device of all the tensors, made current for the launch, and its current stream.
class On {
 public:
  On(const at::Tensor& first, std::initializer_list<const at::Tensor*> others) : device_(first.device()) {
    require(device_.is_cuda(), "the B200 kernels need CUDA tensors (there is no CPU path)");
    for (const at::Tensor* t : others) require(t == nullptr || t->device() == device_, "tensors must be on one CUDA device");
    if (c10::cuda::current_device() != device_.index()) guard_.emplace(device_);
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(device_.index()).stream(); }
  void check(const char* name, int status, int kernels) const {
    if (status == IRIS_OK) {
      launches += kernels;
      return;
    }
    const std::string message = entries.last_error();
    if (status == IRIS_EINVAL) throw Refused(message);
    throw std::runtime_error(std::string(name) + ": " + message);
  }

 private:
  c10::Device device_;
  std::optional<c10::cuda::CUDAGuard> guard_;
};

PyObject* rope(PyObject* const* a) {
  const at::Tensor& x = tensor(a[0], "rope needs [B, H, N, D] head rows");
  const at::Tensor &cos = tensor(a[1], "rope needs cos and sin"), &sin = tensor(a[2], "rope needs cos and sin");
  const at::Tensor* positions = maybe(a[3], "positions must be int32 or int64 [N] or [B, N]");
  const at::Tensor* given = maybe(a[6], "rope: out must be a tensor");
  require(x.dim() == 4, "rope needs [B, H, N, D] head rows");
  iris_rope_problem q = {};
  q.batch = x.size(0), q.heads = x.size(1), q.n = x.size(2), q.head_dim = x.size(3);
  q.dtype = type_code(x.scalar_type());
  tables(cos, sin, q.head_dim, &q.table_rows, &q.rotary);
  q.x = head_rows(x, q.batch, q.heads, q.n, q.head_dim, "");
  if (positions == nullptr) {
    require(q.n <= q.table_rows, "rope: the tables do not cover the rows");
  } else {
    q.positions_64 = positions->scalar_type() == at::kLong;
    const bool flat = positions->dim() == 1 && positions->size(0) == q.n;
    require((q.positions_64 || positions->scalar_type() == at::kInt) &&
                (flat || (positions->dim() == 2 && positions->size(0) == q.batch && positions->size(1) == q.n)),
            "positions must be int32 or int64 [N] or [B, N]");
    require(q.n <= 1 || positions->stride(-1) == 1, "positions must be contiguous along the rows");
    q.positions_stride = flat ? 0 : positions->stride(0);
    q.positions = positions->data_ptr();
  }
  q.layout = rope_layout(a[4]);
  q.inverse = truth(a[5]);
  require(given == nullptr || !share(*given, x) || same_rows(*given, x), "rope: out must be x itself or share no memory with it");
  const On on(x, {&cos, &sin, positions, given});
  if (given) {
    require(given->scalar_type() == x.scalar_type(), "rope: out must have the input's type");
    writable(*given);
  }
  at::Tensor out = given ? *given : at::empty(x.sizes(), x.options());
  q.out = head_rows(out, q.batch, q.heads, q.n, q.head_dim, "rope: out must have the input's shape");
  q.cos = static_cast<const float*>(cos.data_ptr()), q.sin = static_cast<const float*>(sin.data_ptr());
  on.check("iris_rope", entries.rope(&q, on.stream()), q.batch * q.n > 0);
  return THPVariable_Wrap(std::move(out));
}

PyObject* rope_append(PyObject* const* a) {
  const char* need = "rope_append needs [B, H, N, D] head rows";
  const at::Tensor &qt = tensor(a[0], need), &k = tensor(a[1], need), &v = tensor(a[2], need);
  const at::Tensor &cos = tensor(a[3], "rope_append needs cos and sin"), &sin = tensor(a[4], "rope_append needs cos and sin");
  const at::Tensor& starts = tensor(a[5], "starts must be contiguous int32 [B]");
  const at::Tensor &k_cache = tensor(a[6], need), &v_cache = tensor(a[7], need);
  const at::Tensor* counts = maybe(a[9], "counts must be contiguous int32 [B]");
  const at::Tensor* given = maybe(a[11], "rope_append: out must be a tensor");
  require(qt.dim() == 4 && k.dim() == 4 && k_cache.dim() == 4, need);
  iris_append_problem q = {};
  q.batch = qt.size(0), q.heads_q = qt.size(1), q.n = qt.size(2), q.head_dim = qt.size(3);
  q.heads_kv = k.size(1), q.capacity = k_cache.size(2);
  const at::ScalarType type = qt.scalar_type();
  q.dtype = type_code(type);
  tables(cos, sin, q.head_dim, &q.table_rows, &q.rotary);
  require(k.scalar_type() == type && v.scalar_type() == type && k_cache.scalar_type() == type && v_cache.scalar_type() == type,
          "rope_append: one type for rows and cache");
  q.q = head_rows(qt, q.batch, q.heads_q, q.n, q.head_dim, need);
  q.k = head_rows(k, q.batch, q.heads_kv, q.n, q.head_dim, "rope_append: k must be [B, H_kv, N, D]");
  q.v = head_rows(v, q.batch, q.heads_kv, q.n, q.head_dim, "rope_append: v must be [B, H_kv, N, D]");
  q.k_cache = head_rows(k_cache, q.batch, q.heads_kv, q.capacity, q.head_dim, "rope_append: k_cache must be [B, H_kv, C, D]");
  q.v_cache = head_rows(v_cache, q.batch, q.heads_kv, q.capacity, q.head_dim, "rope_append: v_cache must be [B, H_kv, C, D]");
  writable(k_cache);
  writable(v_cache);
  require(!share(k_cache, v_cache), "rope_append: the caches must not share memory");
  for (const at::Tensor* rows : {&qt, &k, &v})
    require(!share(*rows, k_cache) && !share(*rows, v_cache), "rope_append: the rows must not share memory with a cache");
  if (given) {
    require(!share(*given, qt) || same_rows(*given, qt), "rope_append: out must be q itself or share no memory with it");
    for (const at::Tensor* other : {&k, &v, &k_cache, &v_cache})
      require(!share(*given, *other), "rope_append: out must not share memory with k, v or a cache");
  }
  q.sinks = -1;
  if (a[8] != Py_None) {
    q.sinks = whole(a[8]);
    require(0 <= q.sinks && q.sinks < q.capacity, "rope_append: a rolling cache needs more slots than sinks");
  }
  q.starts = int32_rows(&starts, q.batch, "starts must be contiguous int32 [B]");
  q.counts = int32_rows(counts, q.batch, "counts must be contiguous int32 [B]");
  q.layout = rope_layout(a[10]);
  const On on(qt, {&k, &v, &cos, &sin, &starts, &k_cache, &v_cache, counts, given});
  if (given) {
    require(given->scalar_type() == type, "rope_append: out must have the input's type");
    writable(*given);
  }
  at::Tensor out = given ? *given : at::empty(qt.sizes(), qt.options());
  q.zero_rest = given == nullptr;  // rows from counts[b] on of a new output
  q.out = head_rows(out, q.batch, q.heads_q, q.n, q.head_dim, "rope_append: out must have q's shape");
  q.cos = static_cast<const float*>(cos.data_ptr()), q.sin = static_cast<const float*>(sin.data_ptr());
  on.check("iris_rope_append", entries.rope_append(&q, on.stream()), q.batch * q.n > 0);
  return THPVariable_Wrap(std::move(out));
}

PyObject* window_attention(PyObject* const* a) {
  const char* need = "window_attention: q [B, H, N, D], k/v [B, H_kv, N_kv, D]";
  const at::Tensor &qt = tensor(a[0], need), &k = tensor(a[1], need), &v = tensor(a[2], need);
  const at::Tensor* starts = maybe(a[6], "starts must be contiguous int32 [B]");
  const at::Tensor* lengths = maybe(a[7], "lengths must be contiguous int32 [B]");
  const at::Tensor* given = maybe(a[9], "window_attention: out must be a tensor");
  require(qt.dim() == 4 && k.dim() == 4, need);
  iris_window_problem q = {};
  q.batch = qt.size(0), q.heads_q = qt.size(1), q.n = qt.size(2), q.head_dim = qt.size(3);
  q.heads_kv = k.size(1), q.n_kv = k.size(2);
  const at::ScalarType type = qt.scalar_type();
  require((type == at::kBFloat16 || type == at::kHalf) && k.scalar_type() == type && v.scalar_type() == type,
          "window_attention: q, k and v in one of bf16, f16");
  q.dtype = type_code(type);
  require(q.head_dim == 128 || q.head_dim == 64, "window_attention: head_dim must be 64 or 128");
  q.q = head_rows(qt, q.batch, q.heads_q, q.n, q.head_dim, need);
  q.k = head_rows(k, q.batch, q.heads_kv, q.n_kv, q.head_dim, "window_attention: k must be [B, H_kv, N_kv, D]");
  q.v = head_rows(v, q.batch, q.heads_kv, q.n_kv, q.head_dim, "window_attention: v must be [B, H_kv, N_kv, D]");
  q.left = a[3] == Py_None ? -1 : whole(a[3]);
  q.right = a[4] == Py_None ? -1 : whole(a[4]);
  q.sinks = whole(a[5]);
  require((q.left >= 0 || a[3] == Py_None) && (q.right >= 0 || a[4] == Py_None) && q.sinks >= 0,
          "window_attention: left, right and sinks must not be negative");
  q.starts = int32_rows(starts, q.batch, "starts must be contiguous int32 [B]");
  q.lengths = int32_rows(lengths, q.batch, "lengths must be contiguous int32 [B]");
  q.scale = 1.0 / std::sqrt(static_cast<double>(q.head_dim));
  if (a[8] != Py_None) {
    q.scale = PyFloat_AsDouble(a[8]);
    if (q.scale == -1.0 && PyErr_Occurred()) throw Raised{};
  }
  const int64_t width = q.heads_q * q.head_dim;
  if (given) {
    // onto q's own rows: a row is read by the CTAs that write it, before they do
    const bool own = given->dim() == 3 && given->data_ptr() == qt.data_ptr() && given->size(0) == q.batch &&
                     given->size(1) == q.n && given->size(2) == width && given->stride(2) == 1 &&
                     (q.batch <= 1 || given->stride(0) == qt.stride(0)) && (q.n <= 1 || given->stride(1) == qt.stride(2)) &&
                     (q.heads_q <= 1 || qt.stride(1) == q.head_dim);
    require(own || !share(*given, qt), "window_attention: out must be q's own rows or share no memory with q");
    require(!share(*given, k) && !share(*given, v), "window_attention: out must not share memory with k or v");
  }
  const On on(qt, {&k, &v, starts, lengths, given});
  if (given) {
    require(given->dim() == 3 && given->size(0) == q.batch && given->size(1) == q.n && given->size(2) == width &&
                given->scalar_type() == type && given->stride(2) == 1,
            "window_attention: out must be [B, N, H * D] rows of the input's type");
    writable(*given);
  }
  at::Tensor out = given ? *given : at::empty({q.batch, q.n, width}, qt.options());
  q.out = out.data_ptr();
  q.out_stride_b = q.batch > 1 ? out.stride(0) : 0;
  q.out_stride_n = q.n > 1 ? out.stride(1) : 0;
  on.check("iris_window_attn_workspace", entries.window_attn_workspace(&q, &q.workspace_bytes), 0);
  // a workspace of this call's own: two graphs or streams never share one
  at::Tensor workspace;
  if (q.workspace_bytes > 0) {
    workspace = at::empty({q.workspace_bytes}, qt.options().dtype(at::kByte));
    q.workspace = workspace.data_ptr();
  }
  on.check("iris_window_attn_fwd", entries.window_attn_fwd(&q, on.stream()), q.batch * q.n == 0 ? 0 : q.workspace ? 2 : 1);
  return THPVariable_Wrap(std::move(out));
}

PyObject* gemv_q4(PyObject* const* a) {
  const char* need = "gemv_q4 needs x [M, K], packed [N, K / 2], scale [N, K / group]";
  const at::Tensor &x = tensor(a[0], need), &packed = tensor(a[1], need), &scale = tensor(a[2], need);
  const at::Tensor* zero = maybe(a[3], "gemv_q4: zero must be contiguous uint8 [N, K / group]");
  const at::Tensor* bias = maybe(a[4], "gemv_q4: bias must be a tensor");
  require(x.dim() == 2 && packed.dim() == 2 && scale.dim() == 2, need);
  iris_q4_problem q = {};
  q.M = x.size(0), q.K = x.size(1), q.N = packed.size(0);
  require(packed.scalar_type() == at::kByte && packed.is_contiguous() && packed.size(1) * 2 == q.K,
          "gemv_q4: packed must be contiguous uint8 [N, K / 2]");
  const int64_t groups = scale.size(1);
  require(scale.scalar_type() == at::kBFloat16 && scale.is_contiguous() && scale.size(0) == q.N && groups > 0 && q.K % groups == 0,
          "gemv_q4: scale must be contiguous bf16 [N, K / group]");
  require(zero == nullptr || (zero->scalar_type() == at::kByte && zero->is_contiguous() && zero->sizes() == scale.sizes()),
          "gemv_q4: zero must be contiguous uint8 [N, K / group]");
  require(x.stride(1) == 1 || q.K == 1, "gemv_q4: x rows must be contiguous");
  require(bias == nullptr || (bias->scalar_type() == at::kFloat && bias->is_contiguous()), "bias must be contiguous FP32");
  require(bias == nullptr || (bias->dim() == 1 && bias->size(0) == q.N), "gemv_q4: bias width");
  q.group = q.K / groups;
  q.x_dtype = q.out_dtype = type_code(x.scalar_type());
  at::ScalarType out_type = x.scalar_type();
  if (a[7] != Py_None) {
    require(THPDtype_Check(a[7]), "gemv_q4: out_dtype must be a dtype");
    out_type = reinterpret_cast<THPDtype*>(a[7])->scalar_type;
    q.out_dtype = type_code(out_type);
  }
  q.silu_in = truth(a[5]), q.silu_out = truth(a[6]);
  q.ldx = q.M > 1 ? x.stride(0) : q.K;
  const On on(x, {&packed, &scale, zero, bias});
  at::Tensor out = at::empty({q.M, q.N}, x.options().dtype(out_type));
  q.x = x.data_ptr(), q.packed = packed.data_ptr(), q.scale = scale.data_ptr(), q.out = out.data_ptr();
  q.zero = zero ? zero->data_ptr() : nullptr;
  q.bias = bias ? static_cast<const float*>(bias->data_ptr()) : nullptr;
  on.check("iris_gemv_q4", entries.gemv_q4(&q, on.stream()), 1);
  return THPVariable_Wrap(std::move(out));
}

// No C++ exception leaves the module.
template <PyObject* (*Call)(PyObject* const*), int Args>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t n) {
  try {
    if (n != Args) throw Refused("wrong number of arguments");
    if (entries.last_error == nullptr) throw std::runtime_error("the library is not bound");
    return Call(args);
  } catch (const Raised&) {
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (...) {  // torch's own (out of memory, among others) keep their Python types
    torch::translate_exception_to_python(std::current_exception());
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

// Addresses of the entry points, in the order of Entries.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  void* at[6] = {};
  if (n != 6) {
    PyErr_SetString(PyExc_ValueError, "bind takes six addresses");
    return nullptr;
  }
  for (int i = 0; i < 6; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (at[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: null address");
      return nullptr;
    }
  }
  entries.rope = reinterpret_cast<decltype(entries.rope)>(at[0]);
  entries.rope_append = reinterpret_cast<decltype(entries.rope_append)>(at[1]);
  entries.window_attn_fwd = reinterpret_cast<decltype(entries.window_attn_fwd)>(at[2]);
  entries.window_attn_workspace = reinterpret_cast<decltype(entries.window_attn_workspace)>(at[3]);
  entries.gemv_q4 = reinterpret_cast<decltype(entries.gemv_q4)>(at[4]);
  entries.last_error = reinterpret_cast<decltype(entries.last_error)>(at[5]);
  Py_RETURN_NONE;
}

PyObject* launched(PyObject*, PyObject*) { return PyLong_FromLongLong(launches); }

template <PyObject* (*Call)(PyObject* const*), int Args>
PyMethodDef method(const char* name) {
  return PyMethodDef{name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(guarded<Call, Args>)), METH_FASTCALL, ""};
}

PyMethodDef methods[] = {
    method<rope, 7>("rope"),
    method<rope_append, 12>("rope_append"),
    method<window_attention, 10>("window_attention"),
    method<gemv_q4, 8>("gemv_q4"),
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(bind)), METH_FASTCALL, ""},
    {"launched", launched, METH_NOARGS, "Kernels that these calls enqueued."},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_text_side", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__text_side(void) { return PyModule_Create(&module); }
