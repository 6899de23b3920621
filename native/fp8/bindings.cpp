// Calls of the 8-bit operators (native/hip/fp8_blocks.hip, fp8_matmul.hip) on torch tensors: checks, outputs and
// the launch in one step. From Python the same took 8 to 17 us a call (3 of them the launch), more than the
// kernels of a decoded token.
//
// A call that is not wanted gets None and is refused in words by ops/fp8.py; a status that is not 0 comes back
// as a number. The C entries of libyoda_hip.so are bound by address, so this module links to torch alone.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "build_id.h"

namespace {

using NormFn = int (*)(int, void*, int, int, int, const void*, int64_t, const void*, int64_t, const void*, void*, void*,
                       void*, int64_t, int, double);
using QuantizeFn = int (*)(int, void*, int, int, int, const void*, int64_t, void*, void*, int64_t, int);
using MatmulFn = int (*)(int, void*, int, int, const void*, const void*, const void*, const void*, const void*, void*,
                         int64_t, int64_t, int, int64_t, int64_t, void*, int64_t);
using WorkspaceFn = int64_t (*)(int64_t, int64_t, int, int);
NormFn norm_entry = nullptr;
QuantizeFn quantize_entry = nullptr;
MatmulFn matmul_entry = nullptr;
WorkspaceFn workspace_entry = nullptr;

constexpr int64_t kBlock = 128;

int type_of(at::ScalarType t) {
  return t == at::kBFloat16 ? 0 : t == at::kHalf ? 1 : t == at::kFloat ? 2 : -1;
}

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// whether a derivative of t is recorded (reverse mode) or goes along with it (forward mode, which no_grad leaves on)
bool recorded(const at::Tensor& t) {
  return (at::GradMode::is_enabled() && t.requires_grad()) ||
         (t._fw_grad(/*level=*/0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode());
}

// a matrix on a GPU whose columns are neighbours, of a type the operators take, and no part of a graph (a view that
// negates its values holds others than it shows)
bool matrix(const at::Tensor& t) {
  return t.is_cuda() && t.layout() == at::kStrided && t.dim() == 2 && t.size(1) >= 1 &&
         (t.stride(1) == 1 || t.size(1) == 1) && type_of(t.scalar_type()) >= 0 && !t.is_neg() && !recorded(t);
}

bool neighbours(const at::Tensor& t, int64_t n, const at::Device& device) {
  return t.device() == device && t.layout() == at::kStrided && t.dim() == 1 && t.size(0) == n && (n == 1 || t.stride(0) == 1) &&
         !t.is_neg() && !recorded(t);
}

// a new tensor next to x, straight from the device's allocator (the dispatcher's way to it takes longer)
at::Tensor room(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& x) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, x.device(), std::nullopt));
}

at::Tensor values_for(const at::Tensor& x) {
  return room({x.size(0), (x.size(1) + kBlock - 1) / kBlock * kBlock}, at::kFloat8_e4m3fn, x);
}

// the scales' layout: 1 x 128 blocks [blocks of K][rows to a multiple of 8], as [rows, blocks]; 128 x 128 [rows' blocks][blocks of K to one of 4]
at::Tensor scales_for(const at::Tensor& x, bool tiles, bool pow2) {
  const auto type = pow2 ? at::kFloat8_e8m0fnu : at::kFloat;
  const int64_t kb = (x.size(1) + kBlock - 1) / kBlock;
  if (tiles) return room({(x.size(0) + kBlock - 1) / kBlock, (kb + 3) / 4 * 4}, type, x);
  const int64_t pitch = (x.size(0) + 7) / 8 * 8;
  return at::Tensor(at::detail::empty_strided_cuda({pitch, kb}, {1, pitch}, type, x.device()));
}

// whether values and scales are those of a block matrix of these sizes
bool laid_out(const at::Tensor& v, const at::Tensor& s, const at::Device& device, int64_t rows, int64_t kb, bool tiles) {
  if (v.device() != device || s.device() != device || v.scalar_type() != at::kFloat8_e4m3fn || v.dim() != 2 || s.dim() != 2 ||
      v.size(0) != rows || v.size(1) != kb * kBlock || !v.is_contiguous() ||
      (s.scalar_type() != at::kFloat && s.scalar_type() != at::kFloat8_e8m0fnu) ||
      s.is_neg() || recorded(v) || recorded(s) || ((uintptr_t)v.data_ptr() | (uintptr_t)s.data_ptr()) % 16)
    return false;
  if (tiles) return s.size(0) == (rows + kBlock - 1) / kBlock && s.size(1) == (kb + 3) / 4 * 4 && s.is_contiguous();
  const int64_t pitch = (rows + 7) / 8 * 8;
  return s.size(0) == pitch && s.size(1) == kb && (pitch == 0 || kb == 1 || s.stride(1) == pitch) && (pitch <= 1 || s.stride(0) == 1);
}

// the current stream of a tensor's device
void* stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

PyObject* refused() { Py_RETURN_NONE; }

// norm(x, weight, residual or None, eps, pow2) -> (values, scales, sum or None)
PyObject* norm(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 5) return refused();
  const at::Tensor *x = tensor(args[0]), *w = tensor(args[1]), *r = tensor(args[2]);
  if (!x || !w || (!r && args[2] != Py_None) || !matrix(*x)) return refused();
  const int64_t rows = x->size(0), cols = x->size(1);
  const bool wide = w->scalar_type() == at::kFloat;
  if (!neighbours(*w, cols, x->device()) || (!wide && w->scalar_type() != x->scalar_type())) return refused();
  if (r && (!matrix(*r) || r->scalar_type() != x->scalar_type() || r->size(0) != rows || r->size(1) != cols ||
            r->device() != x->device()))
    return refused();
  const double eps = PyFloat_AsDouble(args[3]);
  const long pow2 = PyLong_AsLong(args[4]);
  if (PyErr_Occurred()) return nullptr;
  if (!(eps >= 0) || cols > (1 << 30)) return refused();
  at::Tensor q = values_for(*x), s = scales_for(*x, false, pow2), h;
  if (r) h = room({rows, cols}, x->scalar_type(), *x);
  // (what may throw comes before the lock is given up)
  const int device = x->get_device(), type = type_of(x->scalar_type());
  const int64_t pitch = x->stride(0), r_pitch = r ? r->stride(0) : 0;
  const void *from = x->data_ptr(), *add = r ? r->data_ptr() : nullptr, *by = w->data_ptr();
  void *stream = stream_of(*x), *sum = r ? h.data_ptr() : nullptr, *values = q.data_ptr(), *scales = s.data_ptr();
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS
  rc = norm_entry(device, stream, type, wide, pow2 != 0, from, pitch, add, r_pitch, by, sum, values, scales, rows, (int)cols, eps);
  Py_END_ALLOW_THREADS
  if (rc) return PyLong_FromLong(rc);
  PyObject* out = PyTuple_New(3);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(q)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(s)));
  if (r) {
    PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(std::move(h)));
  } else {
    Py_INCREF(Py_None);
    PyTuple_SET_ITEM(out, 2, Py_None);
  }
  return out;
  END_HANDLE_TH_ERRORS
}

// quantize(x, tiles, pow2) -> (values, scales)
PyObject* quantize(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  const at::Tensor* x = count == 3 ? tensor(args[0]) : nullptr;
  if (!x || !matrix(*x) || x->size(1) > (1 << 30)) return refused();
  const long tiles = PyLong_AsLong(args[1]), pow2 = PyLong_AsLong(args[2]);
  if (PyErr_Occurred()) return nullptr;
  at::Tensor q = values_for(*x), s = scales_for(*x, tiles, pow2);
  const int device = x->get_device(), type = type_of(x->scalar_type());
  const int64_t pitch = x->stride(0), rows = x->size(0), cols = x->size(1);
  const void* from = x->data_ptr();
  void *stream = stream_of(*x), *values = q.data_ptr(), *scales = s.data_ptr();
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS
  rc = quantize_entry(device, stream, type, tiles != 0, pow2 != 0, from, pitch, values, scales, rows, (int)cols);
  Py_END_ALLOW_THREADS
  if (rc) return PyLong_FromLong(rc);
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(q)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(s)));
  return out;
  END_HANDLE_TH_ERRORS
}

// matmul(a's values, a's scales, b's values, b's scales, rows, columns, K, type of out, bias or None, out or None) -> out
// (values and scales are a BlockMatrix's own, laid out by it)
PyObject* matmul(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 10) return refused();
  const at::Tensor *a = tensor(args[0]), *sa = tensor(args[1]), *b = tensor(args[2]), *sb = tensor(args[3]),
                   *bias = tensor(args[8]), *given = tensor(args[9]);
  if (!a || !sa || !b || !sb || (!bias && args[8] != Py_None) || (!given && args[9] != Py_None)) return refused();
  const int64_t m = PyLong_AsLongLong(args[4]), n = PyLong_AsLongLong(args[5]), k = PyLong_AsLongLong(args[6]);
  const long type = PyLong_AsLong(args[7]);
  if (PyErr_Occurred()) return nullptr;
  const at::Device device = a->device();
  const at::ScalarType out_type = type == 0 ? at::kBFloat16 : at::kHalf;
  if (!a->is_cuda() || sa->scalar_type() != sb->scalar_type() || k < 1 || type < 0 || type > 1) return refused();
  const int kb = (int)((k + kBlock - 1) / kBlock);
  if (!laid_out(*a, *sa, device, m, kb, false) || !laid_out(*b, *sb, device, n, kb, true)) return refused();
  if (bias && (bias->scalar_type() != out_type || !neighbours(*bias, n, device))) return refused();
  at::Tensor out;
  if (given) {
    out = *given;
    if (!out.is_cuda() || out.layout() != at::kStrided || out.dim() != 2 || out.scalar_type() != out_type ||
        out.device() != device || out.size(0) != m || out.size(1) != n || (n > 1 && out.stride(1) != 1) ||
        (m > 1 && out.stride(0) < n) || out.is_neg() || recorded(out))
      return refused();
    if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();        // written in place
  } else {
    out = room({m, n}, out_type, *a);
  }
  const int pow2 = sa->scalar_type() != at::kFloat;
  const int64_t bytes = workspace_entry(m, n, kb, pow2);
  at::Tensor workspace;
  if (bytes) workspace = room({bytes}, at::kByte, *a);
  const int64_t pitch = m > 1 ? out.stride(0) : std::max<int64_t>(n, 1);
  const void *pa = a->data_ptr(), *psa = sa->data_ptr(), *pb = b->data_ptr(), *psb = sb->data_ptr(),
             *add = bias ? bias->data_ptr() : nullptr;
  void *stream = stream_of(*a), *to = out.data_ptr(), *space = bytes ? workspace.data_ptr() : nullptr;
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS
  rc = matmul_entry(device.index(), stream, (int)type, pow2, pa, psa, pb, psb, add, to, m, n, kb, pitch, (m + 7) / 8 * 8, space, bytes);
  Py_END_ALLOW_THREADS
  if (rc) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// corner(t, rows, columns) -> a view of t's first rows and columns, or None where torch has to make it (of a tensor
// that is part of a graph or has a tangent). A slice in Python takes 2 us, and every call's result is asked for its values and scales.
PyObject* corner(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  const at::Tensor* t = count == 3 ? tensor(args[0]) : nullptr;
  if (!t || !t->is_cuda() || t->layout() != at::kStrided || t->dim() != 2 || t->requires_grad() || t->_fw_grad(0).defined() ||
      t->is_inference() || t->is_neg())
    return refused();
  const int64_t rows = PyLong_AsLongLong(args[1]), cols = PyLong_AsLongLong(args[2]);
  if (PyErr_Occurred()) return nullptr;
  if (rows < 0 || cols < 0 || rows > t->size(0) || cols > t->size(1)) return refused();
  const c10::TensorImpl* from = t->unsafeGetTensorImpl();
  at::Tensor view(from->shallow_copy_and_detach(from->version_counter(), /*allow_tensor_metadata_change=*/true));
  view.unsafeGetTensorImpl()->set_sizes_and_strides({rows, cols}, t->strides(), t->storage_offset());
  return THPVariable_Wrap(std::move(view));
  END_HANDLE_TH_ERRORS
}

// bind(norm, quantize, matmul, workspace): addresses of the C entries
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long n = 0, q = 0, m = 0, w = 0;
  if (!PyArg_ParseTuple(args, "KKKK", &n, &q, &m, &w)) return nullptr;
  norm_entry = (NormFn)(uintptr_t)n;
  quantize_entry = (QuantizeFn)(uintptr_t)q;
  matmul_entry = (MatmulFn)(uintptr_t)m;
  workspace_entry = (WorkspaceFn)(uintptr_t)w;
  Py_RETURN_NONE;
}

PyObject* build_id(PyObject*, PyObject*) { return PyUnicode_FromString(YODA_BUILD_ID); }

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"build_id", build_id, METH_NOARGS, nullptr},
    {"norm", (PyCFunction)(void (*)())norm, METH_FASTCALL, nullptr},
    {"quantize", (PyCFunction)(void (*)())quantize, METH_FASTCALL, nullptr},
    {"matmul", (PyCFunction)(void (*)())matmul, METH_FASTCALL, nullptr},
    {"corner", (PyCFunction)(void (*)())corner, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_yoda_fp8", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__yoda_fp8() { return PyModule_Create(&module); }
