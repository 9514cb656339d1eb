// Short way from Python to the entry points whose calls are often so small that the way is what they
// cost: the FP8 products and their quantiser, the router's balance loss and gradient.
//
// Each function here checks its arguments as the Python function of the same name in ops.py does, allocates
// the outputs and calls the C ABI on torch's current stream of the tensors' device. Where anything is
// not as the usual call has it - a wrong type, shape, device or alignment, no rows - it does nothing and
// returns None; the Python function then goes its own, complete way, which says what is wrong. One call of
// fp8_gemm for one row costs 4.9 us of host time this way, 10.5 through ctypes.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "b200_nvfp4.h"

namespace {

using at::ScalarType;
using at::Tensor;

constexpr int64_t kMost = 0x7fffff00, kMostTokens = 1 << 30, kMostGroups = 1024;

int64_t blocks_128(int64_t n) { return (n + 127) / 128; }

// The tensor of an argument; nullptr for None; *bad where it is neither.
const Tensor* tensor_arg(PyObject* o, bool* bad) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) {
    *bad = true;
    return nullptr;
  }
  return &THPVariable_Unpack(o);
}

bool on(const Tensor* t, int index) { return t != nullptr && t->is_cuda() && t->get_device() == index && t->is_contiguous(); }

bool is_fp8(const Tensor* t) { return t->scalar_type() == ScalarType::Float8_e4m3fn || t->scalar_type() == ScalarType::Byte; }

bool aligned16(const Tensor* t) { return (reinterpret_cast<uintptr_t>(t->data_ptr()) & 15u) == 0; }

bool is_shape(const Tensor* t, std::initializer_list<int64_t> shape) {
  return t->sizes() == at::IntArrayRef(shape.begin(), shape.size());
}

// Codes of the C ABI; -1: none.
int input_code(ScalarType t) {
  return t == ScalarType::Half ? 0 : t == ScalarType::BFloat16 ? 1 : t == ScalarType::Float ? 2 : -1;
}
int output_code(ScalarType t) {
  return t == ScalarType::Half ? 0 : t == ScalarType::Float ? 1 : t == ScalarType::BFloat16 ? 2 : -1;
}

Tensor empty(at::IntArrayRef size, ScalarType type, int index) {
  return at::detail::empty_cuda(size, type, at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(index)), std::nullopt);
}

PyObject* refuse(const char* what, int status) {
  PyErr_Format(PyExc_RuntimeError, "%s failed: %s", what, b200_nvfp4_status_string(status));
  return nullptr;
}

void* stream_of(int index) { return at::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream(); }

// The interpreter is free for other threads from here to the end of the scope: an allocation or a launch can wait for
// the GPU (a launch does while the queue is full), and what the GPU waits for may be another thread's to do.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  Unlocked() = default;
  Unlocked(const Unlocked&) = delete;
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// A C++ exception (an allocation that failed) becomes the Python one torch has for it.
template <typename Body>
PyObject* guarded(Body body) {
  HANDLE_TH_ERRORS
  return body();
  END_HANDLE_TH_ERRORS
}

// The output of a product: the given one, or a new one of the wanted type. Undefined where something is off.
Tensor product_output(PyObject* dtype, const Tensor* given, bool bad, int64_t rows, int64_t n, int index) {
  if (bad) return Tensor();
  ScalarType wanted = ScalarType::Half;
  if (dtype != Py_None) {
    if (!THPDtype_Check(dtype)) return Tensor();
    wanted = reinterpret_cast<THPDtype*>(dtype)->scalar_type;
  }
  if (given == nullptr) return output_code(wanted) < 0 ? Tensor() : empty({rows, n}, wanted, index);
  if (!on(given, index) || output_code(given->scalar_type()) < 0 || !is_shape(given, {rows, n}) || !aligned16(given) ||
      (dtype != Py_None && given->scalar_type() != wanted))
    return Tensor();
  return *given;
}

bool product_operands(const Tensor* x, const Tensor* w, const Tensor* xs, const Tensor* ws, int index) {
  if (!on(x, index) || !on(w, index) || !on(xs, index) || !on(ws, index) || x->dim() != 2 || !is_fp8(x) || !is_fp8(w) ||
      xs->scalar_type() != ScalarType::Float || ws->scalar_type() != ScalarType::Float || !aligned16(x) || !aligned16(w))
    return false;
  const int64_t rows = x->size(0), k = x->size(1), n = w->size(-2);
  return rows > 0 && rows <= kMost && k > 0 && k <= kMost && k % 16 == 0 && n > 0 && n <= kMost && n % 8 == 0 &&
         w->size(-1) == k && is_shape(xs, {rows, blocks_128(k)});
}

// fp8_gemm(a, b, a_scale, b_scale, out_dtype, output)
PyObject* fp8_gemm(PyObject*, PyObject* const* args, Py_ssize_t count) {
  return guarded([&]() -> PyObject* {
    if (count != 6) Py_RETURN_NONE;
    bool bad = false;
    const Tensor *a = tensor_arg(args[0], &bad), *b = tensor_arg(args[1], &bad), *sa = tensor_arg(args[2], &bad),
                 *sb = tensor_arg(args[3], &bad), *given = tensor_arg(args[5], &bad);
    if (bad || a == nullptr || !a->is_cuda() || b == nullptr || b->dim() != 2) Py_RETURN_NONE;
    const int index = a->get_device();
    if (!product_operands(a, b, sa, sb, index)) Py_RETURN_NONE;
    const int64_t m = a->size(0), k = a->size(1), n = b->size(0);
    if (!is_shape(sb, {blocks_128(n), blocks_128(k)})) Py_RETURN_NONE;
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index));
    Tensor out;
    int status = 0;
    {
      const Unlocked unlocked;
      out = product_output(args[4], given, bad, m, n, index);
      if (out.defined())
        status = b200_nvfp4_fp8_gemm(static_cast<int>(m), static_cast<int>(n), static_cast<int>(k), a->data_ptr(), b->data_ptr(),
                                     sa->data_ptr(), sb->data_ptr(), out.data_ptr(), output_code(out.scalar_type()), stream_of(index));
    }
    if (!out.defined()) Py_RETURN_NONE;
    if (status != 0) return refuse("b200_nvfp4_fp8_gemm", status);
    return THPVariable_Wrap(out);
  });
}

// fp8_grouped_gemm(x, weight, seqlens, cu_seqlens, x_scale, weight_scale, out_dtype, output)
PyObject* fp8_grouped_gemm(PyObject*, PyObject* const* args, Py_ssize_t count) {
  return guarded([&]() -> PyObject* {
    if (count != 8) Py_RETURN_NONE;
    bool bad = false;
    const Tensor *x = tensor_arg(args[0], &bad), *w = tensor_arg(args[1], &bad), *seqlens = tensor_arg(args[2], &bad),
                 *cu = tensor_arg(args[3], &bad), *xs = tensor_arg(args[4], &bad), *ws = tensor_arg(args[5], &bad),
                 *given = tensor_arg(args[7], &bad);
    if (bad || x == nullptr || !x->is_cuda() || w == nullptr || w->dim() != 3) Py_RETURN_NONE;
    const int index = x->get_device();
    if (!product_operands(x, w, xs, ws, index) || !on(seqlens, index) || !on(cu, index) ||
        seqlens->scalar_type() != ScalarType::Int || cu->scalar_type() != ScalarType::Int)
      Py_RETURN_NONE;
    const int64_t groups = w->size(0), m = x->size(0), k = x->size(1), n = w->size(1);
    if (groups <= 0 || groups > kMostGroups || groups * n > kMost || !is_shape(ws, {groups, blocks_128(n), blocks_128(k)}) ||
        seqlens->numel() != groups || cu->numel() != groups + 1)
      Py_RETURN_NONE;
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index));
    Tensor out;
    int status = 0;
    {
      const Unlocked unlocked;
      out = product_output(args[6], given, bad, m, n, index);
      if (out.defined())
        status = b200_nvfp4_fp8_grouped_gemm(out.data_ptr(), x->data_ptr(), w->data_ptr(), seqlens->data_ptr(), cu->data_ptr(),
                                             xs->data_ptr(), ws->data_ptr(), static_cast<int>(groups), static_cast<int>(m),
                                             static_cast<int>(n), static_cast<int>(k), 0, output_code(out.scalar_type()), stream_of(index));
    }
    if (!out.defined()) Py_RETURN_NONE;
    if (status != 0) return refuse("b200_nvfp4_fp8_grouped_gemm", status);
    return THPVariable_Wrap(out);
  });
}

// quantize_fp8(x, swiglu, output, output_scale)
PyObject* quantize_fp8(PyObject*, PyObject* const* args, Py_ssize_t count) {
  return guarded([&]() -> PyObject* {
    if (count != 4) Py_RETURN_NONE;
    bool bad = false;
    const Tensor *x = tensor_arg(args[0], &bad), *given = tensor_arg(args[2], &bad), *given_scale = tensor_arg(args[3], &bad);
    const int swiglu = PyObject_IsTrue(args[1]);
    if (swiglu < 0) return nullptr;
    if (bad || x == nullptr || !x->is_cuda() || !x->is_contiguous() || x->dim() != 2) Py_RETURN_NONE;
    const int index = x->get_device(), code = input_code(x->scalar_type());
    const int64_t rows = x->size(0), wide = x->size(1), k = swiglu ? wide / 2 : wide, kb = blocks_128(k);
    if (code < 0 || rows <= 0 || rows > kMost || k <= 0 || k > kMost || k % 16 != 0 || (swiglu && wide % 2 != 0) || !aligned16(x) ||
        rows * kb > 0x7fffffffLL)
      Py_RETURN_NONE;
    if (given != nullptr && (!on(given, index) || !is_fp8(given) || !is_shape(given, {rows, k}) || !aligned16(given))) Py_RETURN_NONE;
    if (given_scale != nullptr &&
        (!on(given_scale, index) || given_scale->scalar_type() != ScalarType::Float || !is_shape(given_scale, {rows, kb})))
      Py_RETURN_NONE;
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index));
    Tensor q, s;
    int status = 0;
    {
      const Unlocked unlocked;
      q = given != nullptr ? *given : empty({rows, k}, ScalarType::Float8_e4m3fn, index);
      s = given_scale != nullptr ? *given_scale : empty({rows, kb}, ScalarType::Float, index);
      status = b200_nvfp4_fp8_quantize_rows(q.data_ptr(), s.data_ptr(), x->data_ptr(), static_cast<int>(rows), static_cast<int>(k),
                                            code, swiglu, stream_of(index));
    }
    if (status != 0) return refuse("b200_nvfp4_fp8_quantize_rows", status);
    return Py_BuildValue("(NN)", THPVariable_Wrap(q), THPVariable_Wrap(s));
  });
}

struct RouterArgs {
  const Tensor *logits, *ids, *cu;
  int index, code;
  int64_t tokens, experts, topk, sequences;
};

bool router_args(PyObject* logits, PyObject* ids, PyObject* cu, RouterArgs* r) {
  bool bad = false;
  r->logits = tensor_arg(logits, &bad);
  r->ids = tensor_arg(ids, &bad);
  r->cu = tensor_arg(cu, &bad);
  if (bad || r->logits == nullptr || r->ids == nullptr || !r->logits->is_cuda() || !r->logits->is_contiguous() || r->logits->dim() != 2)
    return false;
  r->index = r->logits->get_device();
  r->code = input_code(r->logits->scalar_type());
  r->tokens = r->logits->size(0);
  r->experts = r->logits->size(1);
  if (r->code < 0 || r->tokens <= 0 || r->tokens > kMostTokens || r->experts > 4096 || !on(r->ids, r->index) ||
      r->ids->scalar_type() != ScalarType::Int || r->ids->dim() != 2 || r->ids->size(0) != r->tokens)
    return false;
  r->topk = r->ids->size(1);
  r->sequences = 1;
  if (r->cu != nullptr) {
    if (!on(r->cu, r->index) || r->cu->scalar_type() != ScalarType::Int || r->cu->dim() != 1) return false;
    r->sequences = r->cu->numel() - 1;
  }
  return r->topk > 0 && r->topk <= r->experts && r->tokens * r->topk <= 0x7fffffff && r->sequences > 0 && r->sequences <= 65536;
}

void* data_or_null(const Tensor* t) { return t == nullptr ? nullptr : t->data_ptr(); }

// balance_loss(logits, topk_ids, cu_seqlens, scoring code, alpha)
PyObject* balance_loss(PyObject*, PyObject* const* args, Py_ssize_t count) {
  return guarded([&]() -> PyObject* {
    RouterArgs r;
    if (count != 5 || !router_args(args[0], args[1], args[2], &r)) Py_RETURN_NONE;
    const long scoring = PyLong_AsLong(args[3]);
    const double alpha = PyFloat_AsDouble(args[4]);
    if (PyErr_Occurred()) return nullptr;
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(r.index));
    const int tokens = static_cast<int>(r.tokens), experts = static_cast<int>(r.experts), sequences = static_cast<int>(r.sequences);
    Tensor loss, counts, slope;
    int status = 0;
    {
      const Unlocked unlocked;
      const size_t need = b200_nvfp4_moe_balance_loss_workspace_bytes(tokens, experts, sequences);
      loss = empty({}, ScalarType::Float, r.index);
      counts = empty({r.sequences, r.experts}, ScalarType::Int, r.index);
      slope = empty({r.sequences, r.experts}, ScalarType::Float, r.index);
      const Tensor workspace = empty({static_cast<int64_t>(need)}, ScalarType::Byte, r.index);
      status = b200_nvfp4_moe_balance_loss(loss.data_ptr(), counts.data_ptr(), slope.data_ptr(), r.logits->data_ptr(), r.ids->data_ptr(),
                                           data_or_null(r.cu), tokens, experts, static_cast<int>(r.topk), sequences, r.code,
                                           static_cast<int>(scoring), static_cast<float>(alpha), workspace.data_ptr(), need,
                                           stream_of(r.index));
    }
    if (status != 0) return refuse("b200_nvfp4_moe_balance_loss", status);
    return Py_BuildValue("(NNN)", THPVariable_Wrap(loss), THPVariable_Wrap(counts), THPVariable_Wrap(slope));
  });
}

// router_backward(logits, topk_ids, topk_weights, grad_weights, slope, grad_loss, cu_seqlens, scoring code)
PyObject* router_backward(PyObject*, PyObject* const* args, Py_ssize_t count) {
  return guarded([&]() -> PyObject* {
    RouterArgs r;
    if (count != 8 || !router_args(args[0], args[1], args[6], &r)) Py_RETURN_NONE;
    bool bad = false;
    const Tensor *weights = tensor_arg(args[2], &bad), *grad_weights = tensor_arg(args[3], &bad), *slope = tensor_arg(args[4], &bad),
                 *grad_loss = tensor_arg(args[5], &bad);
    const long scoring = PyLong_AsLong(args[7]);
    if (PyErr_Occurred()) return nullptr;
    auto slots = [&](const Tensor* t) {
      return on(t, r.index) && t->scalar_type() == ScalarType::Float && is_shape(t, {r.tokens, r.topk});
    };
    if (bad || (grad_weights == nullptr && slope == nullptr) || (grad_weights != nullptr && (!slots(grad_weights) || !slots(weights))))
      Py_RETURN_NONE;
    if (slope != nullptr &&
        (!on(slope, r.index) || slope->scalar_type() != ScalarType::Float || !is_shape(slope, {r.sequences, r.experts}) ||
         grad_loss == nullptr || !grad_loss->is_cuda() || grad_loss->get_device() != r.index ||
         grad_loss->scalar_type() != ScalarType::Float || grad_loss->numel() != 1))
      Py_RETURN_NONE;
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(r.index));
    Tensor grad;
    int status = 0;
    {
      const Unlocked unlocked;
      grad = empty({r.tokens, r.experts}, r.logits->scalar_type(), r.index);
      status = b200_nvfp4_moe_router_backward(
          grad.data_ptr(), r.logits->data_ptr(), r.ids->data_ptr(), grad_weights != nullptr ? weights->data_ptr() : nullptr,
          data_or_null(grad_weights), data_or_null(slope), slope != nullptr ? grad_loss->data_ptr() : nullptr, data_or_null(r.cu),
          static_cast<int>(r.tokens), static_cast<int>(r.experts), static_cast<int>(r.topk), static_cast<int>(r.sequences), r.code,
          static_cast<int>(scoring), stream_of(r.index));
    }
    if (status != 0) return refuse("b200_nvfp4_moe_router_backward", status);
    return THPVariable_Wrap(grad);
  });
}

PyMethodDef kMethods[] = {
    {"fp8_gemm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fp8_gemm)), METH_FASTCALL, nullptr},
    {"fp8_grouped_gemm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fp8_grouped_gemm)), METH_FASTCALL, nullptr},
    {"quantize_fp8", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(quantize_fp8)), METH_FASTCALL, nullptr},
    {"balance_loss", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(balance_loss)), METH_FASTCALL, nullptr},
    {"router_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(router_backward)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls(void) { return PyModule_Create(&kModule); }
