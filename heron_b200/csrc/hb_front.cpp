// The checks, allocations and calls of the grouped and 4-bit operators in one step (a CPython extension
// over torch's C++ tensors).  heron_b200/kernels.py holds the same checks in Python: a call that this
// file finds anything unusual about (another type, layout, shape or device, knobs) returns None and
// takes that path, which names the fault.  Why it exists: a token's product keeps the GPU busy for a
// few microseconds, and the Python path costs 10.9 us a call (3.6 us of it for one fresh output, 2.4 us
// for the checks, 1.2 us for ctypes; the launch itself 2.5 us).
//
// Python's lock is released while an output is allocated and the library called: both may wait (for memory, for room in
// a stream's queue), and other threads, or a host function in that very queue, may need the lock meanwhile.
//
// Every function returns the result, an int (a status of the library that is not HB_OK), or None.
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/heron_b200.h"

namespace {

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return HB_F32;
    case at::kHalf: return HB_F16;
    case at::kBFloat16: return HB_BF16;
    default: return -1;
  }
}

// A dense CUDA tensor of exactly torch's own class, or nullptr.
const at::Tensor* dense(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.layout() == at::kStrided && t.is_contiguous() && !t.is_conj() && !t.is_neg() ? &t : nullptr;
}

bool is_u8(const at::Tensor* t, int dim) { return t && t->dim() == dim && t->scalar_type() == at::kByte; }

// Whether a caller would expect a graph behind the output (the other path refuses that).
bool wants_graph(const at::Tensor* t) { return t && t->requires_grad() && c10::GradMode::is_enabled(); }

// Sizes as the library takes them; false beyond its ints.
bool fits(int64_t v) { return v >= 0 && v <= 0x7fffffff; }

// The device that all tensors share, if it is the current one; -1 otherwise.
int device_of(std::initializer_list<const at::Tensor*> ts) {
  const int dev = (*ts.begin())->get_device();
  for (const at::Tensor* t : ts)
    if (t && t->get_device() != dev) return -1;
  return dev == c10::cuda::current_device() ? dev : -1;
}

void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(dev).stream(); }

// For its lifetime other threads may run Python.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  Unlocked() = default;
  Unlocked(const Unlocked&) = delete;
  Unlocked& operator=(const Unlocked&) = delete;
  ~Unlocked() { PyEval_RestoreThread(state); }
};

void allocate(at::Tensor* t, at::IntArrayRef shape, const at::Tensor& like, at::ScalarType type) {
  if (!t->defined()) *t = at::empty(shape, like.options().dtype(type).requires_grad(false));
}

// The output: the caller's (if it is what the operator writes), or none yet and the type of a fresh one; false: not for
// this path.
bool output(PyObject* out, PyObject* dtype, at::IntArrayRef shape, int dev, at::Tensor* result, at::ScalarType* type) {
  *type = at::kFloat;
  if (dtype != Py_None) {
    if (!THPDtype_Check(dtype)) return false;
    *type = reinterpret_cast<THPDtype*>(dtype)->scalar_type;
  }
  if (out != Py_None) {
    const at::Tensor* t = dense(out);
    if (!t || t->sizes() != shape || t->get_device() != dev || (dtype != Py_None && t->scalar_type() != *type)) return false;
    *result = *t;
    *type = t->scalar_type();
  }
  return code_of(*type) >= 0;
}

PyObject* answer(int status, PyObject* out, const at::Tensor& result) {
  if (status != HB_OK) return PyLong_FromLong(status);
  if (out == Py_None) return THPVariable_Wrap(result);
  Py_INCREF(out);
  return out;
}

const int* offsets_ptr(const at::Tensor* t) { return static_cast<const int*>(t->const_data_ptr()); }

// grouped(mode, first, second, offsets, out, out_dtype); mode 0: grouped_gemm, 1: _dx, 2: _dw
PyObject* grouped(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) Py_RETURN_NONE;
  const long mode = PyLong_AsLong(a[0]);
  const at::Tensor *x = dense(a[1]), *w = dense(a[2]), *off = dense(a[3]);
  if (!x || !w || !off || x->dim() != 2 || w->dim() != (mode == 2 ? 2 : 3) || x->scalar_type() != w->scalar_type() ||
      off->dim() != 1 || off->scalar_type() != at::kInt || off->numel() < 2 || wants_graph(x) || wants_graph(w))
    Py_RETURN_NONE;
  const int in = code_of(x->scalar_type());
  if (in < 0) Py_RETURN_NONE;
  const int64_t T = x->size(0), E = off->numel() - 1;
  int64_t N, K;
  if (mode == 2) {
    N = x->size(1);
    K = w->size(1);
    if (w->size(0) != T) Py_RETURN_NONE;
  } else {
    N = w->size(1);
    K = w->size(2);
    if (w->size(0) != E || x->size(1) != (mode == 0 ? K : N)) Py_RETURN_NONE;
  }
  if (!fits(T) || !fits(E) || !fits(N) || !fits(K)) Py_RETURN_NONE;
  const int dev = device_of({x, w, off});
  if (dev < 0) Py_RETURN_NONE;
  at::Tensor out;
  at::ScalarType type;
  const int64_t sizes[3] = {mode == 2 ? E : T, mode == 1 ? K : N, K};
  const at::IntArrayRef shape(sizes, mode == 2 ? 3 : 2);
  if (!output(a[4], a[5], shape, dev, &out, &type) || (out.defined() && wants_graph(&out))) Py_RETURN_NONE;
  const auto fn = mode == 0 ? hb_grouped_gemm : (mode == 1 ? hb_grouped_gemm_dx : hb_grouped_gemm_dw);
  int rc;
  {
    Unlocked unlocked;
    allocate(&out, shape, *x, type);
    rc = fn(x->const_data_ptr(), w->const_data_ptr(), out.mutable_data_ptr(), offsets_ptr(off), static_cast<int>(T),
            static_cast<int>(K), static_cast<int>(N), static_cast<int>(E), static_cast<hb_dtype>(in),
            static_cast<hb_dtype>(code_of(type)), nullptr, stream_of(dev));
  }
  return answer(rc, a[4], out);
  END_HANDLE_TH_ERRORS
}

// Shape of a quantised matrix or batch; K elements a row.
struct Mx {
  int64_t batch, rows, K, groups;
  size_t bytes;  // scales of one matrix
};
bool mx_shape(const at::Tensor& t, int64_t K, const at::Tensor* off, Mx* m) {
  const int64_t dim = t.dim();
  if ((dim != 2 && dim != 3) || (off && (dim != 2 || off->dim() != 1 || off->scalar_type() != at::kInt || off->numel() < 2)))
    return false;
  m->batch = dim == 3 ? t.size(0) : 1;
  m->rows = t.size(dim - 2);
  m->K = K;
  m->groups = off ? off->numel() - 1 : 0;
  if (!fits(m->batch) || !fits(m->rows) || !fits(K) || !fits(m->groups)) return false;
  m->bytes = hb_mxfp4_scale_bytes(1, static_cast<int>(m->rows), static_cast<int>(K), static_cast<int>(m->groups));
  return m->bytes > 0;  // (no rows, or sizes that are refused: the other path)
}
bool scales_fit(const at::Tensor& s, const Mx& m, int64_t dim) {
  if (s.scalar_type() != at::kByte) return false;
  const int64_t bytes = static_cast<int64_t>(m.bytes);
  return dim == 2 ? s.dim() == 1 && s.size(0) == bytes : s.dim() == 2 && s.size(0) == m.batch && s.size(1) == bytes;
}

// quantize(x, offsets, codes, scales) -> (codes, scales)
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) Py_RETURN_NONE;
  const at::Tensor *x = dense(a[0]), *off = a[1] == Py_None ? nullptr : dense(a[1]);
  if (!x || (a[1] != Py_None && !off) || x->dim() < 2) Py_RETURN_NONE;
  const int in = code_of(x->scalar_type());
  const int64_t dim = x->dim(), K = x->size(dim - 1);
  Mx m;
  if (in < 0 || !mx_shape(*x, K, off, &m)) Py_RETURN_NONE;
  const int dev = device_of({x, off ? off : x});
  if (dev < 0) Py_RETURN_NONE;
  const int64_t code_sizes[3] = {x->size(0), dim == 3 ? x->size(1) : K / 2, K / 2};
  const int64_t scale_sizes[2] = {dim == 3 ? m.batch : static_cast<int64_t>(m.bytes), static_cast<int64_t>(m.bytes)};
  const at::IntArrayRef code_shape(code_sizes, dim), scale_shape(scale_sizes, dim - 1);
  at::Tensor codes, scales;
  if (a[2] != Py_None) {
    const at::Tensor* t = dense(a[2]);
    if (!is_u8(t, dim) || t->sizes() != code_shape || t->get_device() != dev) Py_RETURN_NONE;
    codes = *t;
  }
  if (a[3] != Py_None) {
    const at::Tensor* t = dense(a[3]);
    if (!t || !scales_fit(*t, m, dim) || t->get_device() != dev) Py_RETURN_NONE;
    scales = *t;
  }
  int rc;
  {
    Unlocked unlocked;
    allocate(&codes, code_shape, *x, at::kByte);
    allocate(&scales, scale_shape, *x, at::kByte);
    rc = hb_quantize_mxfp4(x->const_data_ptr(), codes.mutable_data_ptr(), scales.mutable_data_ptr(),
                           off ? offsets_ptr(off) : nullptr, static_cast<int>(m.batch), static_cast<int>(m.rows),
                           static_cast<int>(K), static_cast<int>(m.groups), static_cast<hb_dtype>(in), stream_of(dev));
  }
  if (rc != HB_OK) return PyLong_FromLong(rc);
  PyObject* pair = PyTuple_New(2);
  if (!pair) return nullptr;
  for (int i = 0; i < 2; ++i) {
    PyObject* o = a[2 + i];
    if (o == Py_None) o = THPVariable_Wrap(i == 0 ? codes : scales); else Py_INCREF(o);
    PyTuple_SET_ITEM(pair, i, o);
  }
  return pair;
  END_HANDLE_TH_ERRORS
}

// dequantize(codes, scales, offsets, out, out_dtype)
PyObject* dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5) Py_RETURN_NONE;
  const at::Tensor *codes = dense(a[0]), *scales = dense(a[1]), *off = a[2] == Py_None ? nullptr : dense(a[2]);
  if (!codes || !scales || (a[2] != Py_None && !off) || codes->dim() < 2 || codes->scalar_type() != at::kByte)
    Py_RETURN_NONE;
  const int64_t dim = codes->dim(), K = 2 * codes->size(dim - 1);
  Mx m;
  if (!mx_shape(*codes, K, off, &m) || !scales_fit(*scales, m, dim)) Py_RETURN_NONE;
  const int dev = device_of({codes, scales, off ? off : codes});
  if (dev < 0) Py_RETURN_NONE;
  const int64_t sizes[3] = {codes->size(0), dim == 3 ? codes->size(1) : K, K};
  const at::IntArrayRef shape(sizes, dim);
  at::Tensor out;
  at::ScalarType type;
  if (!output(a[3], a[4], shape, dev, &out, &type)) Py_RETURN_NONE;
  int rc;
  {
    Unlocked unlocked;
    allocate(&out, shape, *codes, type);
    rc = hb_dequantize_mxfp4(codes->const_data_ptr(), scales->const_data_ptr(), out.mutable_data_ptr(),
                             off ? offsets_ptr(off) : nullptr, static_cast<int>(m.batch), static_cast<int>(m.rows),
                             static_cast<int>(K), static_cast<int>(m.groups), static_cast<hb_dtype>(code_of(type)),
                             stream_of(dev));
  }
  return answer(rc, a[3], out);
  END_HANDLE_TH_ERRORS
}

// mx(a, a_scales, b, b_scales, offsets, out, out_dtype): gemm_mxfp4, with offsets grouped_gemm_mxfp4
PyObject* mx(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) Py_RETURN_NONE;
  const at::Tensor *x = dense(a[0]), *xs = dense(a[1]), *w = dense(a[2]), *ws = dense(a[3]);
  const at::Tensor* off = a[4] == Py_None ? nullptr : dense(a[4]);
  const int64_t wdim = a[4] == Py_None ? 2 : 3;
  if (!is_u8(x, 2) || !xs || !is_u8(w, static_cast<int>(wdim)) || !ws || (a[4] != Py_None && !off)) Py_RETURN_NONE;
  const int64_t K = 2 * x->size(1);
  Mx mx_, mw;
  if (w->size(wdim - 1) * 2 != K || !mx_shape(*x, K, off, &mx_) || !mx_shape(*w, K, nullptr, &mw)) Py_RETURN_NONE;
  if ((off && mx_.groups != mw.batch) || !scales_fit(*xs, mx_, 2) || !scales_fit(*ws, mw, wdim)) Py_RETURN_NONE;
  const int dev = device_of({x, xs, w, ws, off ? off : x});
  if (dev < 0) Py_RETURN_NONE;
  const int64_t shape[2] = {mx_.rows, mw.rows};
  at::Tensor out;
  at::ScalarType type;
  if (!output(a[5], a[6], shape, dev, &out, &type)) Py_RETURN_NONE;
  const hb_dtype ot = static_cast<hb_dtype>(code_of(type));
  const int T = static_cast<int>(mx_.rows), N = static_cast<int>(mw.rows), k = static_cast<int>(K);
  int rc;
  {
    Unlocked unlocked;
    allocate(&out, shape, *x, type);
    rc = off ? hb_grouped_gemm_mxfp4(x->const_data_ptr(), xs->const_data_ptr(), w->const_data_ptr(), ws->const_data_ptr(),
                                     out.mutable_data_ptr(), offsets_ptr(off), T, k, N, static_cast<int>(mw.batch), ot,
                                     nullptr, stream_of(dev))
             : hb_gemm_mxfp4(x->const_data_ptr(), xs->const_data_ptr(), w->const_data_ptr(), ws->const_data_ptr(),
                             out.mutable_data_ptr(), T, k, N, ot, nullptr, stream_of(dev));
  }
  return answer(rc, a[5], out);
  END_HANDLE_TH_ERRORS
}

#define HB_FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {HB_FAST(grouped), HB_FAST(quantize), HB_FAST(dequantize), HB_FAST(mx), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_front", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__front(void) {
  PyObject* m = PyModule_Create(&module);
  // (the torch that this is built for, see build.py)
  if (m && PyModule_AddStringConstant(m, "built_for", HB_FRONT_KEY) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
