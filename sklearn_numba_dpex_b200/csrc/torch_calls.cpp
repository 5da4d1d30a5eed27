// The expert and 8-bit calls of kmb200.h on torch tensors: checks of arguments, allocation of results, launch
// on the device's current stream.  A decoding step makes these calls at a few microseconds each, and the same
// work in Python and ctypes costs 12 to 18 us a call; here it costs 4 to 6.  Nothing is computed in this file.
//
// Every entry takes its arguments by position from the Python functions of sklearn_numba_dpex_b200.common, and
// turns a C++ exception into a Python one: bad arguments into ValueError, failures of the library into the
// exception that its status stands for (_cabi.check).
#include <stdarg.h>
#include <string.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include "kmb200.h"

namespace {

PyObject* g_kmb_error = nullptr;      // _cabi.KmbError

struct Raised {};                     // a Python exception is set

[[noreturn]] void bad(const char* format, ...) {
  va_list ap;
  va_start(ap, format);
  PyErr_FormatV(PyExc_ValueError, format, ap);
  va_end(ap);
  throw Raised();
}

void check(int status, const char* call) {
  if (status >= 0) return;
  PyObject* type = status == KMB_ERR_INVALID       ? PyExc_ValueError
                   : status == KMB_ERR_UNSUPPORTED ? PyExc_NotImplementedError
                                                   : g_kmb_error;
  PyErr_Format(type, "%s: %s", call, kmb_last_error());
  throw Raised();
}

// Runs a body that may throw, as a Python call.
template <typename F>
PyObject* guarded(F body) {
  try {
    return body();
  } catch (const Raised&) {
    return nullptr;
  } catch (...) {
    torch::translate_exception_to_python(std::current_exception());   // torch's own, out of memory among them
  }
  return nullptr;
}

[[noreturn]] void unsupported(const char* format, const char* name) {
  PyErr_Format(PyExc_NotImplementedError, format, name);
  throw Raised();
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o) || !THPVariable_Unpack(o).is_cuda()) bad("%s must be a CUDA tensor", name);
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.layout() != at::kStrided) bad("%s must be a dense tensor", name);
  // what stands for other tensors (those of torch.func and vmap) has no memory of its own
  if (!t.has_storage()) unsupported("%s is a tensor of a torch.func transform, which this call does not support", name);
  // (asked of the tensor itself: the dispatched Tensor::_fw_grad costs 0.8 us of host time)
  if (t.unsafeGetTensorImpl()->_fw_grad(0, t).defined())
    unsupported("%s carries a forward-mode tangent, which this call does not support", name);
  return t;
}
const char* type_name(at::ScalarType t) { return c10::toString(t); }

at::Tensor matrix(PyObject* o, const char* name) {
  const at::Tensor& t = tensor(o, name);
  if (t.dim() != 2) bad("%s must have two dimensions, got %lld", name, (long long)t.dim());
  const at::Tensor plain = t.is_neg() ? t.resolve_neg() : t;       // a view whose memory holds the negated values
  return plain.is_contiguous() ? plain : plain.contiguous();
}
at::Tensor matrix(PyObject* o, const char* name, at::ScalarType type) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != type) bad("%s must have dtype %s, got %s", name, type_name(type), type_name(t.scalar_type()));
  return matrix(o, name);
}
void same_device(const at::Tensor& t, const char* name, const at::Tensor& other) {
  if (t.device() != other.device())
    bad("%s must be on %s, got %s", name, other.device().str().c_str(), t.device().str().c_str());
}
// A contiguous tensor of a type on the device of `other`.
const at::Tensor& dense(PyObject* o, const char* name, at::ScalarType type, const at::Tensor& other) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != type) bad("%s must have dtype %s, got %s", name, type_name(type), type_name(t.scalar_type()));
  if (!t.is_contiguous() || t.is_neg()) bad("%s must be contiguous", name);
  same_device(t, name, other);
  return t;
}
int row_code(at::ScalarType t, const char* name) {
  if (t == at::kFloat) return KMB_F32;
  if (t == at::kHalf) return KMB_F16;
  if (t == at::kBFloat16) return KMB_BF16;
  bad("%s must have dtype float32, float16 or bfloat16, got %s", name, type_name(t));
}
int64_t whole(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised();
  return v;
}
// A count that the library takes as an int: whatever does not fit is refused there all the same.
int small(PyObject* o) {
  const int64_t v = whole(o);
  return v > INT32_MAX ? INT32_MAX : v < INT32_MIN ? INT32_MIN : (int)v;
}
int width(int64_t v, const char* name) {
  if (v > INT32_MAX) bad("%s is too long: %lld", name, (long long)v);
  return (int)v;
}
float real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1 && PyErr_Occurred()) throw Raised();
  return (float)v;
}
template <typename T = void>
T* ptr(const at::Tensor& t) { return static_cast<T*>(t.data_ptr()); }

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
  return at::empty(sizes, at::TensorOptions().dtype(type).device(like.device()));
}
void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

PyObject* wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }
PyObject* wrap(at::Tensor a, at::Tensor b) {
  PyObject* x = wrap(std::move(a));
  PyObject* y = x ? wrap(std::move(b)) : nullptr;
  PyObject* r = y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  return r;
}
PyObject* wrap(at::Tensor a, at::Tensor b, at::Tensor c) {
  PyObject* x = wrap(std::move(a));
  PyObject* y = x ? wrap(std::move(b)) : nullptr;
  PyObject* z = y ? wrap(std::move(c)) : nullptr;
  PyObject* r = z ? PyTuple_Pack(3, x, y, z) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  Py_XDECREF(z);
  return r;
}

#define CALL(NAME, COUNT)                                                                             \
  static PyObject* NAME##_body(PyObject* const* a);                                                   \
  static PyObject* NAME(PyObject*, PyObject* const* a, Py_ssize_t n) {                                \
    if (n != COUNT) {                                                                                 \
      PyErr_Format(PyExc_TypeError, #NAME " takes %d arguments, got %zd", COUNT, n);                  \
      return nullptr;                                                                                 \
    }                                                                                                 \
    return guarded([&] { return NAME##_body(a); });                                                   \
  }                                                                                                   \
  static PyObject* NAME##_body(PyObject* const* a)

// (logits, k, bias, flags, n_groups, topk_groups, group_best, scale)
CALL(route_topk, 8) {
  const at::Tensor logits = matrix(a[0], "logits");
  const int code = row_code(logits.scalar_type(), "logits");
  const int64_t n = logits.size(0);
  const int e = width(logits.size(1), "logits"), k = small(a[1]);
  const float* bias = nullptr;
  if (a[2] != Py_None) {
    const at::Tensor& b = dense(a[2], "bias", at::kFloat, logits);
    if (b.dim() != 1 || b.size(0) != e) bad("bias must have shape (%d,)", e);
    bias = ptr<float>(b);
  }
  if (k < 1) bad("k must be at least 1, got %d", k);
  if (k > e) bad("Expected k to be greater than or equal to the number of items in the search space, but got k=%d and %d items in the search space.", k, e);
  c10::cuda::CUDAGuard guard(logits.device());
  at::Tensor weights = empty({n, k}, at::kFloat, logits), experts = empty({n, k}, at::kInt, logits);
  check(kmb_route_topk(code, ptr(logits), bias, n, e, k, small(a[3]), small(a[4]), small(a[5]), small(a[6]),
                       real(a[7]), ptr<float>(weights), ptr<int32_t>(experts), stream_of(logits)),
        "kmb_route_topk");
  return wrap(std::move(weights), std::move(experts));
}

// (logits, experts, grad_weights, flags, scale)
CALL(route_topk_grad, 5) {
  const at::Tensor logits = matrix(a[0], "logits");
  const int code = row_code(logits.scalar_type(), "logits");
  const at::Tensor experts = matrix(a[1], "experts", at::kInt), grad = matrix(a[2], "grad_weights", at::kFloat);
  const int64_t n = logits.size(0);
  if (experts.size(0) != n || grad.sizes() != experts.sizes())
    bad("experts and grad_weights must both have shape (%lld, k)", (long long)n);
  same_device(experts, "experts", logits);
  same_device(grad, "grad_weights", logits);
  c10::cuda::CUDAGuard guard(logits.device());
  at::Tensor out = empty(logits.sizes(), logits.scalar_type(), logits);
  check(kmb_route_topk_grad(code, ptr(logits), ptr<int32_t>(experts), ptr<float>(grad), n,
                            width(logits.size(1), "logits"), width(experts.size(1), "experts"), small(a[3]),
                            real(a[4]), ptr(out), stream_of(logits)),
        "kmb_route_topk_grad");
  return wrap(std::move(out));
}

// (experts, n_experts)
CALL(expert_slots, 2) {
  const at::Tensor experts = matrix(a[0], "experts", at::kInt);
  const int64_t n = experts.size(0);
  const int k = width(experts.size(1), "experts"), e = small(a[1]);
  if (k < 1) bad("experts must have at least one column");
  if (e < 1 || e > 1024) bad("the number of experts must be in [1, 1024], got %d", e);
  c10::cuda::CUDAGuard guard(experts.device());
  at::Tensor slots = empty({n, k}, at::kInt, experts), rows = empty({n * k}, at::kInt, experts),
             offsets = empty({e + 1}, at::kInt, experts), ws;
  const size_t bytes = kmb_expert_slots_workspace_bytes(n, k, e);
  if (bytes) ws = empty({(int64_t)bytes}, at::kByte, experts);
  check(kmb_expert_slots(ptr<int32_t>(experts), n, k, e, ptr<int32_t>(slots), ptr<int32_t>(rows),
                         ptr<int32_t>(offsets), bytes ? ptr(ws) : nullptr, bytes, stream_of(experts)),
        "kmb_expert_slots");
  return wrap(std::move(slots), std::move(rows), std::move(offsets));
}

struct CombineArgs {
  at::Tensor values, slots, weights;
  int code, k, d;
  int64_t n;
  explicit CombineArgs(PyObject* const* a)
      : values(matrix(a[0], "values")), slots(matrix(a[1], "slots", at::kInt)),
        weights(matrix(a[2], "weights", at::kFloat)) {
    code = row_code(values.scalar_type(), "values");
    if (weights.sizes() != slots.sizes())
      bad("weights must have the shape of slots (%lld, %lld)", (long long)slots.size(0), (long long)slots.size(1));
    same_device(slots, "slots", values);
    same_device(weights, "weights", values);
    n = slots.size(0);
    k = width(slots.size(1), "slots");
    d = width(values.size(1), "values");
  }
};

// (values, slots, weights)
CALL(combine_experts, 3) {
  const CombineArgs c(a);
  c10::cuda::CUDAGuard guard(c.values.device());
  at::Tensor out = empty({c.n, c.d}, c.values.scalar_type(), c.values);
  check(kmb_combine_experts(c.code, ptr(c.values), c.values.size(0), ptr<int32_t>(c.slots), ptr<float>(c.weights),
                            c.n, c.k, c.d, ptr(out), stream_of(c.values)),
        "kmb_combine_experts");
  return wrap(std::move(out));
}

// (values, slots, weights, grad_out)
CALL(combine_experts_grad, 4) {
  const CombineArgs c(a);
  const at::Tensor grad = matrix(a[3], "grad_out", c.values.scalar_type());
  if (grad.size(0) != c.n || grad.size(1) != c.d) bad("grad_out must have shape (%lld, %d)", (long long)c.n, c.d);
  same_device(grad, "grad_out", c.values);
  c10::cuda::CUDAGuard guard(c.values.device());
  at::Tensor gv = empty(c.values.sizes(), c.values.scalar_type(), c.values), gw = empty({c.n, c.k}, at::kFloat, c.values);
  const size_t bytes = kmb_combine_experts_grad_workspace_bytes_for(c.values.size(0), c.n, c.k);
  at::Tensor ws = empty({(int64_t)bytes}, at::kByte, c.values);
  check(kmb_combine_experts_grad(c.code, ptr(c.values), c.values.size(0), ptr<int32_t>(c.slots), ptr<float>(c.weights),
                                 ptr(grad), c.n, c.k, c.d, ptr(gv), ptr<float>(gw), ptr(ws), bytes,
                                 stream_of(c.values)),
        "kmb_combine_experts_grad");
  return wrap(std::move(gv), std::move(gw));
}

// For calls that have no gradient: what asks for one would not get it.
void no_gradient(const at::Tensor& t, const char* name, const char* call) {
  if (t.requires_grad() && c10::GradMode::is_enabled())
    bad("%s requires a gradient, but %s has none: detach it, or call under torch.no_grad()", name, call);
}

int64_t round16(int64_t d) { return (d + 15) / 16 * 16; }

// Row pitch of 8-bit rows of our own: whole lines of 128 bytes where that costs an eighth at most.  The product
// reads rows in pieces of 128 bytes, and pieces that straddle lines cost it (32 groups, 16 396 rows, 1408
// outputs: 57 us with 2048 features, 71 us with 2056 at a pitch of 2064).
int64_t pitch_of(int64_t d) {
  for (int64_t line = 128; line > 16; line /= 2) {
    const int64_t pitch = (d + line - 1) / line * line;
    if (pitch - d <= d / 8) return pitch;
  }
  return round16(d);
}

// (x, rows)
CALL(quantize_rows, 2) {
  const at::Tensor& x0 = tensor(a[0], "x");
  if (x0.dim() != 2 || x0.size(1) < 1) bad("x must have shape (n, d) with d >= 1");
  const int code = row_code(x0.scalar_type(), "x");
  no_gradient(x0, "x", "quantize_rows");
  const at::Tensor x = matrix(a[0], "x");
  const int64_t n = x.size(0);
  const int d = width(x.size(1), "x");
  int64_t m = n;
  const int32_t* rows = nullptr;
  if (a[1] != Py_None) {
    const at::Tensor& r = dense(a[1], "rows", at::kInt, x);
    if (r.dim() != 1) bad("rows must have one dimension");
    m = r.size(0);
    rows = ptr<int32_t>(r);
  }
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t pitch = pitch_of(d);
  at::Tensor q = empty({m, pitch}, at::kChar, x), scales = empty({m}, at::kFloat, x);
  check(kmb_quantize_rows(code, ptr(x), n, d, rows, m, ptr<int8_t>(q), pitch, ptr<float>(scales), stream_of(x)),
        "kmb_quantize_rows");
  // the rows without what pads them to the pitch (a view would cost as much as the launch)
  const int64_t sizes[2] = {m, d}, strides[2] = {pitch, 1};
  q.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef(sizes, 2), at::IntArrayRef(strides, 2));
  return wrap(std::move(q), std::move(scales));
}

// `t` with rows at a pitch of a multiple of 16 bytes, as the kernel's loads need them: itself if it is laid
// out so (as quantize_rows returns it), else a copy.
at::Tensor pitched(const at::Tensor& t, int64_t* pitch) {
  const int64_t d = t.size(-1), dims = t.dim();
  if (t.numel() && !t.is_neg() && ((uintptr_t)t.data_ptr() & 15) == 0 && (d == 1 || t.stride(-1) == 1)) {
    *pitch = t.size(-2) == 1 && (dims == 2 || t.size(0) == 1) ? round16(t.stride(-2) > d ? t.stride(-2) : d) : t.stride(-2);
    if (*pitch % 16 == 0 && *pitch >= d && (dims == 2 || t.size(0) == 1 || t.stride(0) == t.size(1) * *pitch)) return t;
  }
  *pitch = pitch_of(d);
  std::vector<int64_t> sizes(t.sizes().begin(), t.sizes().end());
  sizes.back() = *pitch;
  at::Tensor copy = empty(sizes, at::kChar, t).narrow(-1, 0, d);
  copy.copy_(t);
  return copy;
}

// (a, a_scales, b, b_scales, bias, offsets, out_dtype)
CALL(int8_matmul, 7) {
  const at::Tensor &x = tensor(a[0], "a"), &w = tensor(a[2], "b");
  for (const at::Tensor* t : {&x, &w})
    if (t->scalar_type() != at::kChar)
      bad("%s must have dtype torch.int8, got %s", t == &x ? "a" : "b", type_name(t->scalar_type()));
  if (!THPDtype_Check(a[6])) bad("out_dtype must be a torch.dtype");
  const at::ScalarType out_type = reinterpret_cast<THPDtype*>(a[6])->scalar_type;
  const int code = row_code(out_type, "out_dtype");
  const bool grouped = a[5] != Py_None;
  if (x.dim() != 2 || w.dim() != (grouped ? 3 : 2)) bad("a must be (m, d) and b (n, d), or (g, n, d) with offsets");
  const int64_t m = x.size(0), d = x.size(1), g = grouped ? w.size(0) : 1, n = w.size(-2);
  if (w.size(-1) != d) bad("a and b disagree on the number of features: %lld and %lld", (long long)d, (long long)w.size(-1));
  same_device(w, "b", x);
  const at::Tensor &xs = dense(a[1], "a_scales", at::kFloat, x), &ws = dense(a[3], "b_scales", at::kFloat, x);
  if (xs.dim() != 1 || xs.size(0) != m) bad("a_scales must have shape (%lld,)", (long long)m);
  const auto per_feature = w.sizes().slice(0, w.dim() - 1);
  if (ws.sizes() != per_feature) bad("b_scales must have a scale for each row of b");
  no_gradient(xs, "a_scales", "int8_matmul");
  no_gradient(ws, "b_scales", "int8_matmul");
  const float* bias = nullptr;
  if (a[4] != Py_None) {
    const at::Tensor& b = dense(a[4], "bias", at::kFloat, x);
    if (b.sizes() != per_feature) bad("bias must have the shape of b_scales");
    no_gradient(b, "bias", "int8_matmul");
    bias = ptr<float>(b);
  }
  const int32_t* offsets = nullptr;
  if (grouped) {
    const at::Tensor& o = dense(a[5], "offsets", at::kInt, x);
    if (o.dim() != 1 || o.size(0) != g + 1) bad("offsets must have shape (%lld,)", (long long)(g + 1));
    offsets = ptr<int32_t>(o);
  }
  if (d > 131071) bad("at most 131071 features (sums are held in 32 bits), got %lld", (long long)d);
  c10::cuda::CUDAGuard guard(x.device());
  at::Tensor out = empty({m, n}, out_type, x);
  if (m == 0 || n == 0) return wrap(std::move(out));
  if (d == 0 || g == 0) bad("d and the number of groups must be at least 1");
  int64_t lda, ldb;
  const at::Tensor xp = pitched(x, &lda), wp = pitched(w, &ldb);
  check(kmb_int8_matmul(code, ptr<int8_t>(xp), lda, ptr<float>(xs), ptr<int8_t>(wp), ldb, ptr<float>(ws), bias,
                        offsets, width(g, "b"), ptr(out), m, width(n, "b"), (int)d, stream_of(x)),
        "kmb_int8_matmul");
  return wrap(std::move(out));
}

#define ENTRY(NAME) {#NAME, (PyCFunction)(void (*)(void))NAME, METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {ENTRY(route_topk),      ENTRY(route_topk_grad),      ENTRY(expert_slots),
                           ENTRY(combine_experts), ENTRY(combine_experts_grad), ENTRY(quantize_rows),
                           ENTRY(int8_matmul),     {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_torch_calls", nullptr, -1, g_methods};

}  // namespace

// The file's name does not tell what it was built for, so the module does, before it touches anything whose layout
// hangs on it.
static bool built_for_this_process() {
  const char* built = PY_VERSION;
  const char* runs = Py_GetVersion();
  size_t minor = strchr(strchr(built, '.') + 1, '.') - built + 1;      // "3.12."
  if (strncmp(built, runs, minor) != 0) {
    PyErr_Format(PyExc_ImportError, "_torch_calls was built for Python %s, this is %s", built, runs);
    return false;
  }
  PyObject* torch = PyImport_ImportModule("torch");
  PyObject* version = torch ? PyObject_GetAttrString(torch, "__version__") : nullptr;
  const char* have = version ? PyUnicode_AsUTF8(version) : nullptr;
  const bool same = have && strcmp(have, KMB_TORCH_VERSION) == 0;
  if (have && !same)
    PyErr_Format(PyExc_ImportError, "_torch_calls was built for torch %s, this is %s", KMB_TORCH_VERSION, have);
  Py_XDECREF(version);
  Py_XDECREF(torch);
  return same;
}

PyMODINIT_FUNC PyInit__torch_calls() {
  if (!built_for_this_process()) return nullptr;
  PyObject* cabi = PyImport_ImportModule("sklearn_numba_dpex_b200._cabi");
  if (!cabi) return nullptr;
  Py_XDECREF(g_kmb_error);
  g_kmb_error = PyObject_GetAttrString(cabi, "KmbError");
  Py_DECREF(cabi);
  if (!g_kmb_error) return nullptr;
  return PyModule_Create(&g_module);
}
