// Python module _rows: the operators of powersparse_b200/rows.py on torch tensors.
//
// Checks the tensors, allocates outputs and scratch from torch's allocator on the
// stream of the call, and calls the C entry points (include/powersparse_b200.h) by the
// addresses that bind() was given, so that it serves whichever library the package has
// loaded.  Native because at a serving step's sizes the kernels take a few
// microseconds, and the same checks in Python with a ctypes call took 14 (24 for
// dispatch, with its four outputs) against the kernels' 2 to 5; these take 4 (6).
//
// Every function takes positional arguments only, checked for their number; rows.py
// holds the signatures.  ValueError for refused arguments, RuntimeError for CUDA errors.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <optional>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "powersparse_b200.h"

namespace {

struct Api {
  decltype(&ps_last_error) last_error;
  decltype(&ps_embedding) embedding;
  decltype(&ps_embedding_grad_workspace) embedding_grad_workspace;
  decltype(&ps_embedding_grad) embedding_grad;
  decltype(&ps_route) route;
  decltype(&ps_route_grad) route_grad;
  decltype(&ps_dispatch_rows) dispatch_rows;
  decltype(&ps_dispatch) dispatch;
  decltype(&ps_combine) combine;
  decltype(&ps_combine_grad) combine_grad;
} api = {};

struct Refused : std::invalid_argument {
  using std::invalid_argument::invalid_argument;
};

[[noreturn]] void refuse(const std::string& text) { throw Refused(text); }

void check(int status) {
  if (status == PS_OK) return;
  if (status == PS_ERR_INVALID_ARGUMENT) refuse(api.last_error());
  throw std::runtime_error(api.last_error());
}

constexpr int64_t kMaxWidth = 1 << 24, kMaxRows = (1LL << 31) - 1;  // what the C entry points take
constexpr int64_t kMaxExperts = 1024, kMaxTopK = 32, kMaxAlign = 65536;

std::string text(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kHalf: return "torch.float16";
    case at::kInt: return "torch.int32";
    case at::kLong: return "torch.int64";
    default: return c10::toString(t);
  }
}
std::string text(at::IntArrayRef shape) {
  std::string s = "(";
  for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
  return s + ")";
}

int type_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return PS_F32;
    case at::kBFloat16: return PS_BF16;
    case at::kHalf: return PS_F16;
    default: return -1;
  }
}

// A tensor argument; the reference lives as long as the caller's arguments.
const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a CUDA tensor");
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda()) refuse(std::string(name) + " must be a CUDA tensor");
  // A view whose elements stand in memory with the other sign.
  if (t.is_neg()) refuse(std::string(name) + " is a negated view: resolve it first (Tensor.resolve_neg)");
  return t;
}

struct Matrix {
  at::Tensor t;
  int64_t rows = 0, width = 0, stride = 0;
  int type = -1;
  void* ptr = nullptr;
};

// A matrix whose rows are contiguous and do not overlap.
Matrix matrix_of(const at::Tensor& t, const char* name) {
  const int type = type_of(t.scalar_type());
  if (t.dim() != 2 || type < 0) refuse(std::string(name) + " must be a matrix of float32, bfloat16 or float16");
  const int64_t rows = t.size(0), width = t.size(1);
  if (width < 1 || width > kMaxWidth || rows > kMaxRows)
    refuse(std::string(name) + " must have rows of 1 to 2^24 elements, and below 2^31 of them");
  if (width > 1 && t.stride(1) != 1) refuse(std::string(name) + " must have contiguous rows");
  int64_t stride = width;
  if (rows > 1) {
    stride = t.stride(0);
    if (stride < width) refuse(std::string(name) + " has rows that overlap");
  }
  return {t, rows, width, stride, type, t.data_ptr()};
}

Matrix matrix(PyObject* o, const char* name) { return matrix_of(tensor(o, name), name); }

void require_device(const at::Tensor& t, const char* name, c10::Device device) {
  if (t.device() != device) refuse(std::string(name) + " is on " + t.device().str() + ", the other tensors on " + device.str());
}

// A matrix like `as`: its device and type; rows < 0: any number of rows.
Matrix matrix_like(PyObject* o, const char* name, c10::Device device, at::ScalarType type, int64_t rows, int64_t width) {
  const at::Tensor& t = tensor(o, name);
  require_device(t, name, device);
  Matrix m = matrix_of(t, name);
  if (t.scalar_type() != type) refuse(std::string(name) + " must be " + text(type) + ", not " + text(t.scalar_type()));
  if (rows < 0 && m.width != width) refuse(std::string(name) + " must have rows of " + std::to_string(width) + " elements");
  if ((rows >= 0 && m.rows != rows) || m.width != width)
    refuse(std::string(name) + " must have the shape " + text({rows, width}) + ", not " + text(t.sizes()));
  return m;
}

// torch.empty without the dispatcher, which took longer than the allocation.
at::Tensor new_tensor(at::IntArrayRef shape, at::ScalarType type, c10::Device device) {
  return at::detail::empty_cuda(shape, type, device, std::nullopt);
}

Matrix new_matrix(int64_t rows, int64_t width, const at::Tensor& like, at::ScalarType type) {
  at::Tensor t = new_tensor({rows, width}, type, like.device());
  void* p = t.data_ptr();
  return {std::move(t), rows, width, width, type_of(type), p};
}

const at::Tensor& packed(PyObject* o, const char* name, c10::Device device, at::ScalarType type) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != type) refuse(std::string(name) + " must be " + text(type) + ", not " + text(t.scalar_type()));
  require_device(t, name, device);
  if (!t.is_contiguous()) refuse(std::string(name) + " must be contiguous");
  return t;
}

const at::Tensor& packed(PyObject* o, const char* name, c10::Device device, at::ScalarType type, at::IntArrayRef shape) {
  const at::Tensor& t = packed(o, name, device, type);
  if (t.sizes() != shape) refuse(std::string(name) + " must have the shape " + text(shape) + ", not " + text(t.sizes()));
  return t;
}

const at::Tensor& indices(PyObject* o, const char* name, c10::Device device, int& index_type) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong)
    refuse(std::string(name) + " must be torch.int32 or torch.int64, not " + text(t.scalar_type()));
  index_type = t.scalar_type() == at::kLong ? PS_I64 : PS_I32;
  return packed(o, name, device, t.scalar_type());
}

int64_t integer(PyObject* o, const char* name) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    if (!PyErr_ExceptionMatches(PyExc_OverflowError)) throw python_error();
    PyErr_Clear();
    refuse(std::string(name) + " is out of range");
  }
  return v;
}

float real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return float(v);
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}

// The device and stream of a call: the tensors' device, and PyTorch's current stream
// there or the one given (None, or a stream's handle), which then also owns what the
// call allocates.
class Place {
 public:
  Place(c10::Device device, PyObject* stream) : device_(device) {
    if (stream == Py_None) {
      handle_ = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    } else {
      const int64_t value = integer(stream, "stream");
      // 0 and cudaStreamLegacy are the default stream; torch takes other odd values for streams of its own.
      if (value != 0 && value != 1 && value % 2) refuse("stream is not a stream's handle");
      const auto s = value == 0 || value == 1 ? c10::cuda::getDefaultCUDAStream(device.index())
                                              : c10::cuda::getStreamFromExternal(reinterpret_cast<cudaStream_t>(value), device.index());
      handle_ = s.stream();
      stream_.emplace(s);
    }
  }
  void* handle() const { return handle_; }

 private:
  c10::cuda::CUDAGuard device_;
  std::optional<c10::cuda::CUDAStreamGuard> stream_;
  cudaStream_t handle_ = nullptr;
};

class WithoutGil {
 public:
  WithoutGil() : state_(PyEval_SaveThread()) {}
  ~WithoutGil() { PyEval_RestoreThread(state_); }

 private:
  PyThreadState* state_;
};

PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }

// An output: the tensor that the caller gave, as the same object and counted as changed
// (autograd refuses a backward pass that needs what stood there), or a new one.
PyObject* result(PyObject* given, const Matrix& m) {
  if (given == Py_None) return wrap(m.t);
  if (!m.t.is_inference()) m.t.unsafeGetTensorImpl()->bump_version();
  Py_INCREF(given);
  return given;
}

template <typename... P>
PyObject* tuple(P*... items) {
  PyObject* all[] = {items...};
  PyObject* out = PyTuple_New(sizeof...(P));
  if (!out) {
    for (PyObject* o : all) Py_XDECREF(o);
    throw python_error();
  }
  for (size_t i = 0; i < sizeof...(P); ++i) PyTuple_SET_ITEM(out, i, all[i]);
  return out;
}

PyObject* embedding(PyObject* const* a) {  // table, tokens, scale, out, stream
  const Matrix table = matrix(a[0], "table");
  const c10::Device device = table.t.device();
  int index_type = 0;
  const at::Tensor& tokens = indices(a[1], "tokens", device, index_type);
  const float scale = real(a[2]);
  const int64_t n = tokens.numel();
  if (table.rows < 1) refuse("the table has no rows");
  if (n > kMaxRows) refuse("the number of tokens must be below 2^31");
  Matrix out;
  const bool fresh = a[3] == Py_None;
  if (!fresh) out = matrix_like(a[3], "out", device, table.t.scalar_type(), n, table.width);
  const Place place(device, a[4]);
  {
    WithoutGil nogil;
    if (fresh) out = new_matrix(n, table.width, table.t, table.t.scalar_type());
    check(api.embedding(table.ptr, table.type, table.rows, int(table.width), table.stride, tokens.data_ptr(), index_type, n, scale,
                        out.ptr, out.stride, place.handle()));
    if (fresh && tokens.dim() != 1) {
      std::vector<int64_t> shape(tokens.sizes().vec());
      shape.push_back(table.width);
      out.t = out.t.view(shape);
    }
  }
  return result(a[3], out);
}

PyObject* embedding_grad(PyObject* const* a) {  // grad, tokens, rows, scale, padding, dtype (-1: grad's or out's), out, accumulate, stream
  const at::Tensor& given = tensor(a[0], "grad");
  const c10::Device device = given.device();
  int index_type = 0;
  const at::Tensor& tokens = indices(a[1], "tokens", device, index_type);
  const int64_t n = tokens.numel(), rows = integer(a[2], "rows");
  const float scale = real(a[3]);
  at::Tensor flat = given;
  if (given.dim() != 2 && given.dim() == tokens.dim() + 1 && given.sizes().slice(0, tokens.dim()) == tokens.sizes()) {
    if (!given.is_contiguous()) refuse("grad must be a matrix with contiguous rows, or contiguous");
    flat = given.view({n, given.size(-1)});
  }
  const Matrix grad = matrix_of(flat, "grad");
  if (grad.rows != n) refuse("grad has " + std::to_string(grad.rows) + " rows for " + std::to_string(n) + " tokens");
  if (rows < 1 || rows >= kMaxRows) refuse("the table's rows must be in [1, 2^31 - 2]");
  int64_t padding = -1;
  if (a[4] != Py_None) {
    padding = integer(a[4], "padding");
    if (padding < 0 || padding >= rows) refuse("padding must be a row of the table");
  }
  const bool fresh = a[6] == Py_None, accumulate = truth(a[7]);
  if (accumulate && fresh) refuse("accumulate needs the gradient to add to (out)");
  const int64_t asked = integer(a[5], "dtype");
  at::ScalarType type = asked == PS_F32 ? at::kFloat : asked == PS_BF16 ? at::kBFloat16 : asked == PS_F16 ? at::kHalf
                                                                                          : fresh ? grad.t.scalar_type()
                                                                                                  : tensor(a[6], "out").scalar_type();
  if (type != grad.t.scalar_type() && type != at::kFloat)
    refuse("the gradient of the table is " + text(grad.t.scalar_type()) + " or torch.float32, not " + text(type));
  Matrix out;
  if (!fresh) out = matrix_like(a[6], "out", device, type, rows, grad.width);
  const int64_t need = api.embedding_grad_workspace(n, rows, int(grad.width));
  if (need < 0) refuse("the number of tokens must be below 2^31");
  const Place place(device, a[8]);
  {
    WithoutGil nogil;
    if (fresh) out = new_matrix(rows, grad.width, grad.t, type);
    const at::Tensor workspace = new_tensor({need}, at::kByte, device);
    check(api.embedding_grad(grad.ptr, grad.type, grad.stride, tokens.data_ptr(), index_type, n, scale, padding, accumulate, out.ptr,
                             out.type, out.stride, rows, int(grad.width), workspace.data_ptr(), need, place.handle()));
  }
  return result(a[6], out);
}

PyObject* route(PyObject* const* a) {  // logits, top_k, normalize, stream
  const Matrix logits = matrix(a[0], "logits");
  const int64_t top_k = integer(a[1], "top_k");
  const bool normalize = truth(a[2]);
  if (logits.width > kMaxExperts) refuse("the number of experts must be in [1, 1024]");
  if (top_k < 1 || top_k > std::min(logits.width, kMaxTopK))
    refuse("top_k must be in [1, min(" + std::to_string(logits.width) + ", 32)]");
  const Place place(logits.t.device(), a[3]);
  at::Tensor weights, chosen;
  {
    WithoutGil nogil;
    weights = new_tensor({logits.rows, top_k}, at::kFloat, logits.t.device());
    chosen = new_tensor({logits.rows, top_k}, at::kInt, logits.t.device());
    check(api.route(logits.ptr, logits.type, logits.stride, int(logits.rows), int(logits.width), int(top_k), normalize,
                    static_cast<float*>(weights.data_ptr()), static_cast<int*>(chosen.data_ptr()), place.handle()));
  }
  return tuple(wrap(weights), wrap(chosen));
}

PyObject* route_grad(PyObject* const* a) {  // grad, logits, weights, chosen, normalize, out, stream
  const Matrix logits = matrix(a[1], "logits");
  const c10::Device device = logits.t.device();
  const at::Tensor& chosen = packed(a[3], "chosen", device, at::kInt);
  if (chosen.dim() != 2 || chosen.size(0) != logits.rows) refuse("chosen must be [" + std::to_string(logits.rows) + ", top_k]");
  if (chosen.size(1) < 1 || chosen.size(1) > std::min(logits.width, kMaxTopK))
    refuse("top_k must be in [1, min(" + std::to_string(logits.width) + ", 32)]");
  const at::Tensor& weights = packed(a[2], "weights", device, at::kFloat, chosen.sizes());
  const at::Tensor& grad = packed(a[0], "grad", device, at::kFloat, chosen.sizes());
  const bool normalize = truth(a[4]), fresh = a[5] == Py_None;
  Matrix out;
  if (!fresh) out = matrix_like(a[5], "out", device, logits.t.scalar_type(), logits.rows, logits.width);
  const Place place(device, a[6]);
  {
    WithoutGil nogil;
    if (fresh) out = new_matrix(logits.rows, logits.width, logits.t, logits.t.scalar_type());
    check(api.route_grad(static_cast<const float*>(grad.data_ptr()), logits.ptr, logits.type, logits.stride,
                         static_cast<const float*>(weights.data_ptr()), static_cast<const int*>(chosen.data_ptr()), int(logits.rows),
                         int(logits.width), int(chosen.size(1)), normalize, out.ptr, out.stride, place.handle()));
  }
  return result(a[5], out);
}

int64_t rows_needed(int64_t slots, int64_t experts, int64_t align) {
  if (slots < 0 || slots > kMaxRows || experts < 1 || experts > kMaxExperts || align < 1 || align > kMaxAlign)
    refuse("slots must be in [0, 2^31), the number of experts in [1, 1024] and align in [1, 65536]");
  return api.dispatch_rows(slots, int(experts), int(align));
}

PyObject* dispatch_rows(PyObject* const* a) {  // slots, num_experts, align
  return PyLong_FromLongLong(rows_needed(integer(a[0], "slots"), integer(a[1], "num_experts"), integer(a[2], "align")));
}

PyObject* dispatch(PyObject* const* a) {  // x, chosen, num_experts, align, out, stream
  const Matrix x = matrix(a[0], "x");
  const c10::Device device = x.t.device();
  int index_type = 0;
  const at::Tensor& chosen = indices(a[1], "chosen", device, index_type);
  if (chosen.dim() != 2 || chosen.size(0) != x.rows || chosen.size(1) < 1 || chosen.size(1) > kMaxTopK)
    refuse("chosen must be [" + std::to_string(x.rows) + ", top_k] with top_k in [1, 32]");
  const int64_t top_k = chosen.size(1), experts = integer(a[2], "num_experts"), align = integer(a[3], "align");
  const int64_t need = rows_needed(x.rows * top_k, experts, align);
  const bool fresh = a[4] == Py_None;
  Matrix out;
  if (!fresh) {
    out = matrix_like(a[4], "out", device, x.t.scalar_type(), -1, x.width);
    if (out.rows < need) refuse("out must have at least " + std::to_string(need) + " rows");
  }
  const Place place(device, a[5]);
  at::Tensor position, offsets, counts;
  {
    WithoutGil nogil;
    if (fresh) out = new_matrix(need, x.width, x.t, x.t.scalar_type());
    position = new_tensor({x.rows, top_k}, at::kInt, device);
    offsets = new_tensor({experts + 1}, at::kInt, device);
    counts = new_tensor({experts}, at::kInt, device);
    check(api.dispatch(x.ptr, x.type, x.stride, chosen.data_ptr(), index_type, int(x.rows), int(top_k), int(experts), int(align),
                       int(x.width), out.ptr, out.stride, out.rows, fresh, static_cast<int*>(position.data_ptr()),
                       static_cast<int*>(offsets.data_ptr()), static_cast<int*>(counts.data_ptr()), place.handle()));
  }
  return tuple(result(a[4], out), wrap(position), wrap(offsets), wrap(counts));
}

struct Plan {
  at::Tensor position, offsets, counts;
  int64_t tokens, top_k, experts;
};

Plan plan_of(PyObject* position_o, PyObject* offsets_o, PyObject* counts_o, c10::Device device) {
  const at::Tensor& position = packed(position_o, "plan.position", device, at::kInt);
  if (position.dim() != 2 || position.size(0) > kMaxRows || position.size(1) < 1 || position.size(1) > kMaxTopK)
    refuse("plan.position must be [tokens, top_k] with top_k in [1, 32]");
  const at::Tensor& counts = packed(counts_o, "plan.counts", device, at::kInt);
  if (counts.dim() != 1 || counts.size(0) < 1 || counts.size(0) > kMaxExperts)
    refuse("plan.counts must be [experts] with 1 to 1024 experts");
  const at::Tensor& offsets = packed(offsets_o, "plan.offsets", device, at::kInt, {counts.size(0) + 1});
  return {position, offsets, counts, position.size(0), position.size(1), counts.size(0)};
}

PyObject* combine(PyObject* const* a) {  // y, position, offsets, counts, weights, add, out, stream
  const Matrix y = matrix(a[0], "y");
  const c10::Device device = y.t.device();
  const Plan plan = plan_of(a[1], a[2], a[3], device);
  const float* weights = nullptr;
  if (a[4] != Py_None) weights = static_cast<const float*>(packed(a[4], "weights", device, at::kFloat, plan.position.sizes()).data_ptr());
  Matrix add;
  if (a[5] != Py_None) add = matrix_like(a[5], "add", device, y.t.scalar_type(), plan.tokens, y.width);
  const bool fresh = a[6] == Py_None;
  Matrix out;
  if (!fresh) out = matrix_like(a[6], "out", device, y.t.scalar_type(), plan.tokens, y.width);
  const Place place(device, a[7]);
  {
    WithoutGil nogil;
    if (fresh) out = new_matrix(plan.tokens, y.width, y.t, y.t.scalar_type());
    check(api.combine(y.ptr, y.type, y.stride, y.rows, static_cast<const int*>(plan.position.data_ptr()), weights, add.ptr, add.stride,
                      int(plan.tokens), int(plan.top_k), int(y.width), out.ptr, out.stride, place.handle()));
  }
  return result(a[6], out);
}

PyObject* combine_grad(PyObject* const* a) {  // grad, y, position, offsets, counts, weights, out, stream
  const Matrix y = matrix(a[1], "y");
  const c10::Device device = y.t.device();
  const Plan plan = plan_of(a[2], a[3], a[4], device);
  const Matrix grad = matrix_like(a[0], "grad", device, y.t.scalar_type(), plan.tokens, y.width);
  const at::Tensor& weights = packed(a[5], "weights", device, at::kFloat, plan.position.sizes());
  const bool fresh = a[6] == Py_None;
  Matrix out;
  if (!fresh) out = matrix_like(a[6], "out", device, y.t.scalar_type(), y.rows, y.width);
  const Place place(device, a[7]);
  at::Tensor grad_weights;
  {
    WithoutGil nogil;
    if (fresh) out = new_matrix(y.rows, y.width, y.t, y.t.scalar_type());
    grad_weights = new_tensor({plan.tokens, plan.top_k}, at::kFloat, device);
    check(api.combine_grad(grad.ptr, y.type, grad.stride, y.ptr, y.stride, y.rows, static_cast<const int*>(plan.position.data_ptr()),
                           static_cast<const int*>(plan.offsets.data_ptr()), static_cast<const int*>(plan.counts.data_ptr()),
                           int(plan.experts), static_cast<const float*>(weights.data_ptr()), int(plan.tokens), int(plan.top_k),
                           int(y.width), out.ptr, out.stride, fresh, static_cast<float*>(grad_weights.data_ptr()), place.handle()));
  }
  return tuple(result(a[6], out), wrap(grad_weights));
}

// The addresses of the C entry points, in the order of Api's members.
PyObject* bind(PyObject* const* a) {
  void** to = reinterpret_cast<void**>(&api);
  for (size_t i = 0; i < sizeof(Api) / sizeof(void*); ++i) to[i] = reinterpret_cast<void*>(integer(a[i], "address"));
  Py_RETURN_NONE;
}

template <PyObject* (*kFunction)(PyObject* const*), int kArguments>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != kArguments) {
    PyErr_Format(PyExc_TypeError, "%d arguments wanted, %zd given", kArguments, count);
    return nullptr;
  }
  try {
    return kFunction(args);
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

#define PSB_METHOD(name, arguments) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<name, arguments>)), METH_FASTCALL, nullptr}

PyMethodDef methods[] = {PSB_METHOD(bind, int(sizeof(Api) / sizeof(void*))),
                         PSB_METHOD(embedding, 5),
                         PSB_METHOD(embedding_grad, 9),
                         PSB_METHOD(route, 4),
                         PSB_METHOD(route_grad, 7),
                         PSB_METHOD(dispatch_rows, 3),
                         PSB_METHOD(dispatch, 6),
                         PSB_METHOD(combine, 8),
                         PSB_METHOD(combine_grad, 8),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_rows", "Native part of powersparse_b200.rows.", -1, methods, nullptr, nullptr, nullptr,
                      nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__rows(void) { return PyModule_Create(&module); }
