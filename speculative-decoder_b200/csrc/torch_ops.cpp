// The torch-tensor side of the 8-bit operators as a Python extension module: argument checks,
// output allocation and the call of the C ABI. The kernels of small calls take 2-7 us, and the same
// steps through Python and ctypes took 11-16 us of host time per call.
//
// specb200/ops.py documents the functions; they take positional arguments only. Errors are those of
// specb200/_ffi.py: ValueError for bad arguments, NotImplementedError for types and sizes the
// kernels do not handle, RuntimeError for tensors that are not on a CUDA device and for CUDA errors.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <optional>
#include <sstream>
#include <string>

#include "specb200.h"

namespace {

constexpr int64_t kGroup = 128;

struct Refusal {
  PyObject* type;
  std::string text;
};

template <typename... T>
std::string text(const T&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  return s.str();
}
std::string shape(const at::Tensor& t) { return text(t.sizes()); }
[[noreturn]] void bad(const std::string& s) { throw Refusal{PyExc_ValueError, s}; }

const at::Tensor& tensor(PyObject* o, const char* where) {
  if (!THPVariable_Check(o)) throw Refusal{PyExc_TypeError, text(where, ": expected a tensor, got ", Py_TYPE(o)->tp_name)};
  const at::Tensor& t = THPVariable_Unpack(o);
  // such a view's memory holds the values with the other sign
  if (t.is_neg()) bad(text(where, ": a view that is negated on reading (call resolve_neg() first)"));
  return t;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Refusal{nullptr, ""};  // the error is set
  return v != 0;
}

void check_device(const char* where, const at::Tensor& first, std::initializer_list<const at::Tensor*> others) {
  if (!first.is_cuda())
    throw Refusal{PyExc_RuntimeError, text(where, ": the B200 engine runs on CUDA tensors only (got ", first.device(), ")")};
  for (const at::Tensor* t : others)
    if (t && t->device() != first.device()) bad(text(where, ": tensors on ", first.device(), " and ", t->device()));
}
int dtype_code(const at::Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return SPECB200_BF16;
  if (t.scalar_type() == at::kFloat) return SPECB200_F32;
  throw Refusal{PyExc_NotImplementedError,
                text("the B200 engine runs float32 and bfloat16, not ", t.scalar_type())};
}
int as_int(const char* where, int64_t v) {
  if (v > 0x7fffffff) bad(text(where, ": a size of ", v, " is out of range"));
  return static_cast<int>(v);
}
int64_t groups_of(int64_t k) { return (k + kGroup - 1) / kGroup; }
int64_t padded(int64_t k) { return (k + 15) / 16 * 16; }

// torch.empty on x's device without the dispatcher (0.25 us of host time less per tensor).
at::Tensor empty_beside(const at::Tensor& x, at::IntArrayRef sizes, at::ScalarType type) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, x.device(), std::nullopt));
}

// [..., K] as M rows of K consecutive elements, `pitch` elements apart (any pitch that fits a
// single row); copied only if the tensor does not lie like that.
struct Rows {
  at::Tensor held;  // keeps a copy alive until the launch
  const void* ptr;
  int64_t m, k, pitch;
};
Rows rows_of(const char* where, const at::Tensor& x) {
  if (x.dim() == 0) bad(text(where, ": expected rows, got a scalar"));
  Rows r;
  r.k = x.size(-1);
  r.m = 1;
  for (int64_t d = 0; d + 1 < x.dim(); ++d) r.m *= x.size(d);
  auto lies = [&](const at::Tensor& t) {  // a matrix with consecutive columns and rows that do not overlap
    return t.dim() == 2 && (r.k <= 1 || t.stride(1) == 1) && (r.m <= 1 || t.stride(0) >= r.k);
  };
  if (lies(x)) {
    r.held = x;
    r.pitch = x.stride(0);
  } else if (x.is_contiguous()) {
    r.held = x;
    r.pitch = r.k;
  } else {
    r.held = x.detach().reshape({r.m, r.k});
    if (!lies(r.held)) r.held = r.held.contiguous();
    r.pitch = r.held.stride(0);
  }
  if (r.m <= 1) r.pitch = padded(r.k);
  r.ptr = r.held.data_ptr();
  return r;
}

// Room for outputs [..., n] with x's leading dimensions, whose rows start on 16-byte boundaries: linear_fp8
// loads e4m3 rows by TMA, and every kernel reads and writes such rows in whole units (linear 4096 x 8191 x 64:
// 19 us into such rows, 46 into dense ones). Rows that are padded at all are padded to whole 32-byte sectors.
struct Output {
  at::Tensor t;
  int64_t pitch;
};
Output rows_beside(const at::Tensor& x, int64_t n, at::ScalarType type) {
  const int64_t unit = 16 / static_cast<int64_t>(at::elementSize(type));
  Output out;
  out.pitch = n % unit ? (n + 2 * unit - 1) / (2 * unit) * (2 * unit) : n;
  c10::SmallVector<int64_t, 6> sizes(x.sizes().begin(), x.sizes().end());
  sizes.back() = n;
  if (out.pitch == n) {
    out.t = empty_beside(x, sizes, type);
  } else {
    c10::SmallVector<int64_t, 6> strides(sizes.size(), 1);
    int64_t stride = out.pitch;
    for (size_t d = sizes.size() - 1; d-- > 0; stride *= sizes[d]) strides[d] = stride;
    out.t = at::Tensor(at::detail::empty_strided_cuda(sizes, strides, type, x.device()));
  }
  return out;
}
struct Quantized {
  at::Tensor q, scales;
  int64_t pitch;
};
Quantized quantized_like(const at::Tensor& x, int64_t k, at::IntArrayRef scale_sizes = {}) {
  const Output q = rows_beside(x, k, at::kFloat8_e4m3fn);
  c10::SmallVector<int64_t, 6> sizes(x.sizes().begin(), x.sizes().end());
  sizes.back() = groups_of(k);
  return {q.t, empty_beside(x, scale_sizes.empty() ? at::IntArrayRef(sizes) : scale_sizes, at::kFloat), q.pitch};
}

// The current stream of the tensors' device, which is made current for the launch.
struct Here {
  c10::cuda::OptionalCUDAGuard guard;
  void* stream;
  explicit Here(const at::Tensor& x) {
    guard.set_index(x.get_device());
    stream = c10::cuda::getCurrentCUDAStream(x.get_device()).stream();
  }
};

void check_rc(const char* where, int rc) {
  if (rc == SPECB200_OK) return;
  PyObject* type = rc == SPECB200_ERR_ARG           ? PyExc_ValueError
                   : rc == SPECB200_ERR_RANGE       ? PyExc_IndexError
                   : rc == SPECB200_ERR_UNSUPPORTED ? PyExc_NotImplementedError
                                                    : PyExc_RuntimeError;
  throw Refusal{type, text(where, ": ", specb200_last_error(), type == PyExc_RuntimeError ? text(" (status ", rc, ")") : "")};
}

PyObject* tuple_of(std::initializer_list<at::Tensor> parts) {
  PyObject* t = PyTuple_New(static_cast<Py_ssize_t>(parts.size()));
  if (!t) throw Refusal{nullptr, ""};
  Py_ssize_t i = 0;
  for (const at::Tensor& p : parts) PyTuple_SET_ITEM(t, i++, THPVariable_Wrap(p));
  return t;
}

// ------------------------------------------------------------------------------ the operators
PyObject* quantize(PyObject* const* args) {
  const char* where = "quantize_fp8";
  const at::Tensor& x = tensor(args[0], where);
  check_device(where, x, {});
  const long block_rows = PyLong_AsLong(args[1]);
  if (block_rows == -1 && PyErr_Occurred()) throw Refusal{nullptr, ""};
  if (block_rows != 1 && block_rows != kGroup) bad(text(where, ": block_rows is 1 or 128, not ", block_rows));
  if (block_rows != 1 && x.dim() != 2) bad(text(where, ": blocks of 128 rows need a matrix, got shape ", shape(x)));
  const int code = dtype_code(x);
  const Rows r = rows_of(where, x);
  const Quantized out = block_rows == 1 ? quantized_like(x, r.k) : quantized_like(x, r.k, {groups_of(r.m), groups_of(r.k)});
  const Here here(x);
  check_rc(where, specb200_quantize_fp8(code, r.ptr, r.pitch, as_int(where, r.m), as_int(where, r.k),
                                        static_cast<int>(block_rows), out.q.data_ptr(), out.pitch,
                                        static_cast<float*>(out.scales.data_ptr()), here.stream));
  return tuple_of({out.q, out.scales});
}

PyObject* rmsnorm(PyObject* const* args) {
  const char* where = "rmsnorm_fp8";
  const at::Tensor& x = tensor(args[0], where);
  const at::Tensor& weight = tensor(args[1], where);
  const double eps = PyFloat_AsDouble(args[2]);
  if (eps == -1.0 && PyErr_Occurred()) throw Refusal{nullptr, ""};
  const at::Tensor* delta = args[3] == Py_None ? nullptr : &tensor(args[3], where);
  check_device(where, x, {&weight, delta});
  const int code = dtype_code(x);
  const Rows r = rows_of(where, x);
  if (weight.dim() != 1 || weight.size(0) != r.k || weight.scalar_type() != x.scalar_type())
    bad(text(where, ": weight is ", weight.scalar_type(), " ", shape(weight), " for x ", x.scalar_type(), " ", shape(x)));
  if (delta && (delta->sizes() != x.sizes() || delta->scalar_type() != x.scalar_type()))
    bad(text(where, ": delta is ", delta->scalar_type(), " ", shape(*delta), " for x ", x.scalar_type(), " ", shape(x)));
  const at::Tensor w = weight.is_contiguous() ? weight : weight.detach().contiguous();
  const Quantized out = quantized_like(x, r.k);
  Rows d = {};
  Output h = {};
  if (delta) {
    d = rows_of(where, *delta);
    h = rows_beside(x, r.k, x.scalar_type());
  }
  const Here here(x);
  check_rc(where, specb200_rmsnorm_fp8(code, r.ptr, r.pitch, d.ptr, d.pitch, w.data_ptr(), as_int(where, r.m),
                                       as_int(where, r.k), static_cast<float>(eps), delta ? h.t.data_ptr() : nullptr, h.pitch,
                                       out.q.data_ptr(), out.pitch, static_cast<float*>(out.scales.data_ptr()), here.stream));
  return delta ? tuple_of({out.q, out.scales, h.t}) : tuple_of({out.q, out.scales});
}

PyObject* silu_mul(PyObject* const* args) {
  const char* where = "silu_mul_fp8";
  const at::Tensor& x = tensor(args[0], where);
  check_device(where, x, {});
  const bool packed = truth(args[1]);
  const int code = dtype_code(x);
  const Rows r = rows_of(where, x);
  if (r.k % (packed ? 128 : 2))
    bad(text(where, ": ", r.k, " columns are not gate and up", packed ? " in groups of 64" : ""));
  const int64_t inter = r.k / 2;
  const Quantized out = quantized_like(x, inter);
  const Here here(x);
  check_rc(where, specb200_silu_mul_fp8(code, r.ptr, r.pitch, as_int(where, r.m), as_int(where, inter), packed,
                                        out.q.data_ptr(), out.pitch, static_cast<float*>(out.scales.data_ptr()), here.stream));
  return tuple_of({out.q, out.scales});
}

// e4m3 rows that TMA can load: on 16-byte boundaries, copied there if need be.
Rows operand_of(const at::Tensor& x, const char* what) {
  const char* where = "linear_fp8";
  if (x.scalar_type() != at::kFloat8_e4m3fn) bad(text(where, ": ", what, " is ", x.scalar_type(), ", not Float8_e4m3fn"));
  Rows r = rows_of(where, x);
  if (r.pitch % 16 || reinterpret_cast<uintptr_t>(r.ptr) % 16) {
    const at::Tensor bytes = empty_beside(x, {r.m, padded(r.k)}, at::kByte);
    bytes.narrow(1, 0, r.k).copy_(r.held.detach().reshape({r.m, r.k}).view(at::kByte));
    r.held = bytes;
    r.ptr = bytes.data_ptr();
    r.pitch = padded(r.k);
  }
  return r;
}

// The status word, with the interpreter free for other threads while the stream runs.
int wait_for(const at::Tensor& status) {
  struct Released {
    PyThreadState* state = PyEval_SaveThread();
    ~Released() { PyEval_RestoreThread(state); }
  } released;
  return status.item<int>();
}

PyObject* linear(PyObject* const* args) {
  const char* where = "linear_fp8";
  const at::Tensor& x = tensor(args[0], where);
  const at::Tensor& x_scales = tensor(args[1], where);
  const at::Tensor& w = tensor(args[2], where);
  const at::Tensor& w_scales = tensor(args[3], where);
  const bool out_f32 = truth(args[4]), check = truth(args[5]);
  check_device(where, x, {&x_scales, &w, &w_scales});
  if (x.dim() == 0 || w.dim() != 2 || x.size(-1) != w.size(1)) bad(text(where, ": x ", shape(x), " and w ", shape(w), " do not multiply"));
  const Rows rx = operand_of(x, "x"), rw = operand_of(w, "w");
  const int64_t n = rw.m, groups = groups_of(rx.k);
  bool fits = x_scales.dim() == x.dim() && x_scales.size(-1) == groups && w_scales.dim() == 2 &&
              w_scales.size(0) == groups_of(n) && w_scales.size(1) == groups;
  for (int64_t d = 0; fits && d + 1 < x.dim(); ++d) fits = x_scales.size(d) == x.size(d);
  if (!fits)
    bad(text(where, ": scales ", shape(x_scales), " and ", shape(w_scales), " for x ", shape(x), ", w ", shape(w),
             ": one per 128 of K and 128 x 128"));
  if (x_scales.scalar_type() != at::kFloat || w_scales.scalar_type() != at::kFloat)
    bad(text(where, ": scales are float32, not ", x_scales.scalar_type(), " and ", w_scales.scalar_type()));
  const at::Tensor xs = x_scales.is_contiguous() ? x_scales : x_scales.detach().contiguous();
  const at::Tensor ws = w_scales.is_contiguous() ? w_scales : w_scales.detach().contiguous();
  const Output y = rows_beside(x, n, out_f32 ? at::kFloat : at::kBFloat16);
  at::Tensor status;
  if (check) status = empty_beside(x, {1}, at::kInt);
  {
    const Here here(x);
    check_rc(where, specb200_linear_fp8(rx.ptr, rx.pitch, static_cast<const float*>(xs.data_ptr()), rw.ptr, rw.pitch,
                                        static_cast<const float*>(ws.data_ptr()), as_int(where, rx.m), as_int(where, n),
                                        as_int(where, rx.k), out_f32, y.t.data_ptr(), y.pitch,
                                        check ? static_cast<int32_t*>(status.data_ptr()) : nullptr, here.stream));
  }
  if (check) {
    const int code = wait_for(status);
    if (code == SPECB200_ERR_TIMEOUT) throw Refusal{PyExc_RuntimeError, text(where, ": a device-side wait gave up (timeout)")};
    if (code != SPECB200_OK) throw Refusal{PyExc_RuntimeError, text(where, ": device status ", code)};
  }
  return THPVariable_Wrap(y.t);
}

// ------------------------------------------------------------------------------ the module
template <PyObject* (*kFn)(PyObject* const*), Py_ssize_t kArgs>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != kArgs) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", kArgs, n);
    return nullptr;
  }
  try {
    return kFn(args);
  } catch (const Refusal& r) {
    if (r.type) PyErr_SetString(r.type, r.text.c_str());
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    PyErr_SetString(type ? type : PyExc_RuntimeError, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

template <PyObject* (*kFn)(PyObject* const*), Py_ssize_t kArgs>
constexpr PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<kFn, kArgs>)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<quantize, 2>("quantize_fp8"), method<rmsnorm, 4>("rmsnorm_fp8"),
                         method<silu_mul, 2>("silu_mul_fp8"), method<linear, 6>("linear_fp8"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, methods};

}  // namespace

// `target`: what the module was compiled for, which specb200/_ffi.py compares with what runs.
PyMODINIT_FUNC PyInit__torch_ops() {
  PyObject* m = PyModule_Create(&module_def);
  if (m && PyModule_AddStringConstant(m, "target", SPECB200_TARGET) < 0) Py_CLEAR(m);
  return m;
}
