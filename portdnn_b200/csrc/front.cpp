// Native half of portdnn_b200/api.py: one function per operator that checks the tensors, allocates the
// result where the caller gave none and calls the C ABI on torch's current stream.  The checks are a
// handful of field reads in here; as Python they took 6-10 us per call, two to three times what the
// launch itself costs the host (api.conv2d 14.0 us against 4.0 us inside the library), and a network of
// short layers is bound by that: its host issues 55 calls before the device has run the first few.
//
// Every function takes exactly the arguments of the api.py function it stands behind, by position and
// in that order; names, defaults and documentation live there.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/portdnn_b200.h"

namespace {

// Thrown after a Python exception has been set.
struct PyFailure {};

[[noreturn]] void raise(PyObject* type, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  PyErr_FormatV(type, fmt, ap);
  va_end(ap);
  throw PyFailure();
}

// Runs f without the interpreter lock, as torch allocates and ctypes calls: a launch waits when the launch queue
// is full, an allocation when memory has to be found, and neither may keep the process's other threads from
// running (they may be what the queue waits for).  Costs the call 0.1 us.
template <typename F>
auto unlocked(F&& f) {
  struct Release {
    PyThreadState* state = PyEval_SaveThread();
    ~Release() { PyEval_RestoreThread(state); }
  } release;
  return f();
}

// A tensor argument; undefined for None.  (By value: the lock is released while it is in use.)
at::Tensor tensor(PyObject* o) {
  if (o == Py_None) return at::Tensor();
  if (!THPVariable_Check(o)) raise(PyExc_TypeError, "expected a torch.Tensor, got %.100s", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}

template <typename... T>
void require_cuda(const T&... ts) {
  const bool ok = ((!ts.defined() || (ts.is_cuda() && ts.is_contiguous())) && ...);
  if (!ok) raise(PyExc_ValueError, "tensors must be contiguous CUDA tensors");
}

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return PDNN_F32;
    case at::kHalf: return PDNN_F16;
    case at::kBFloat16: return PDNN_BF16;
    default: raise(PyExc_KeyError, "unsupported dtype %s", c10::toString(t.scalar_type()));
  }
}

// A whole number.  (A text or a fraction is a mistake in the call: neither is turned into one.)
long integer(PyObject* o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) throw PyFailure();
  return v;
}
// Whatever int() takes.
long to_integer(PyObject* o) {
  if (PyLong_CheckExact(o)) return integer(o);
  PyObject* n = PyNumber_Long(o);
  if (n == nullptr) throw PyFailure();
  const long v = PyLong_AsLong(n);
  Py_DECREF(n);
  if (v == -1 && PyErr_Occurred()) throw PyFailure();
  return v;
}
double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PyFailure();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PyFailure();
  return v != 0;
}

// The bytes of a ctypes parameter structure.
template <typename P>
P params(PyObject* o) {
  Py_buffer view;
  if (PyObject_GetBuffer(o, &view, PyBUF_SIMPLE) != 0) throw PyFailure();
  P p;
  const bool fits = (size_t)view.len == sizeof(P);
  if (fits) memcpy(&p, view.buf, sizeof(P));
  PyBuffer_Release(&view);
  if (!fits) raise(PyExc_TypeError, "wrong parameter structure: %.100s", Py_TYPE(o)->tp_name);
  return p;
}

void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

// Calls the library, and reports its status as portdnn_b200.api does.  (The error text is the thread's own.)
template <typename F>
void call(F&& f) {
  const int status = unlocked(f);
  if (status == PDNN_OK) return;
  PyObject* api = PyImport_ImportModule("portdnn_b200.api");
  if (api != nullptr) {
    PyObject* r = PyObject_CallMethod(api, "_check", "i", status);
    Py_XDECREF(r);
    Py_DECREF(api);
  }
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, pdnn_last_error());
  throw PyFailure();
}

at::Tensor flat(int64_t n, const at::TensorOptions& options) { return unlocked([&] { return at::empty({n}, options); }); }
at::Tensor like(const at::Tensor& t) { return unlocked([&] { return at::empty_like(t); }); }

// `out` if the caller gave one, else a tensor of the shape of `like`.
at::Tensor out_or_like(const at::Tensor& out, const at::Tensor& t) { return out.defined() ? out : like(t); }

PyObject* conv2d(PyObject* const* a) {
  const long pass = integer(a[0]);
  const at::Tensor &inp = tensor(a[1]), &fil = tensor(a[2]);
  const PdnnConv2DParams p = params<PdnnConv2DParams>(a[3]);
  const int algorithm = (int)integer(a[4]);
  at::Tensor out = tensor(a[5]);
  const at::Tensor &workspace = tensor(a[6]), &bias = tensor(a[7]);
  const int activation = (int)integer(a[8]);
  const double alpha = real(a[9]), beta = real(a[10]);
  const at::Tensor& relu_out = tensor(a[11]);
  const bool output_f32 = truth(a[12]);
  const bool accumulate = truth(a[13]);
  const at::Tensor& bits = tensor(a[14]);
  const bool constant_filter = truth(a[15]), any_order = truth(a[16]);

  require_cuda(inp, fil, out, workspace, bias);
  const int64_t x = (int64_t)p.batch * p.in_rows * p.in_cols * p.channels;
  const int64_t w = (int64_t)p.window_rows * p.window_cols * (p.channels / (p.groups > 1 ? p.groups : 1)) * p.features;
  const int64_t y = (int64_t)p.batch * p.out_rows * p.out_cols * p.features;
  if (pass < 0 || pass > 2) raise(PyExc_KeyError, "%ld", pass);
  const int64_t n_in = pass == PDNN_INPUT_BACKPROP ? y : x, n_fil = pass == PDNN_FILTER_BACKPROP ? y : w;
  const int64_t n_out = pass == PDNN_FORWARD ? y : pass == PDNN_INPUT_BACKPROP ? x : w;
  if (inp.numel() != n_in || fil.numel() != n_fil)
    raise(PyExc_ValueError, "tensor sizes do not match the parameters: %lld/%lld, %lld/%lld", (long long)inp.numel(),
          (long long)n_in, (long long)fil.numel(), (long long)n_fil);
  require_cuda(bits);
  if (bits.defined()) {
    if (pass == PDNN_FILTER_BACKPROP)
      raise(PyExc_ValueError, "relu_bitmask belongs to the forward pass (output) and the input backprop (input)");
    if (bits.scalar_type() != at::kByte || bits.numel() * 8 != n_out)
      raise(PyExc_ValueError, "relu_bitmask must be a uint8 tensor of one bit per element");
  }
  const bool backprop_fused = relu_out.defined() || output_f32 || accumulate || (bits.defined() && pass != PDNN_FORWARD) ||
                              (constant_filter && pass == PDNN_INPUT_BACKPROP);
  if (backprop_fused && (pass == PDNN_FORWARD || (relu_out.defined() && pass != PDNN_INPUT_BACKPROP) ||
                         (output_f32 && pass != PDNN_FILTER_BACKPROP)))
    raise(PyExc_ValueError, "relu_forward_output belongs to the input backprop, output_f32 to the filter backprop");
  if (accumulate && !out.defined()) raise(PyExc_ValueError, "accumulate needs the tensor to add to as out");
  require_cuda(relu_out);
  const at::ScalarType out_type = output_f32 ? at::kFloat : inp.scalar_type();
  if (!out.defined()) out = flat(n_out, inp.options().dtype(out_type));
  if (out.numel() != n_out || out.scalar_type() != out_type)
    raise(PyExc_ValueError, "output tensor does not match the parameters");
  const size_t ws_elems = workspace.defined() ? (size_t)(workspace.nbytes() / inp.element_size()) : 0;
  const int dtype = dtype_code(inp);
  if (backprop_fused) {
    if (relu_out.defined() && relu_out.numel() != n_out)
      raise(PyExc_ValueError, "relu_forward_output must have the shape of the input gradient");
    PdnnBackpropFusion f = {};
    f.relu_forward_output = ptr(relu_out);
    f.output_f32 = output_f32;
    f.accumulate = (int)to_integer(a[13]);  // False / True, or 2 (dx already carries the mask)
    f.relu_bitmask = ptr(bits);
    f.constant_filter = constant_filter;
    call([&] {
      return pdnn_conv2d_backprop_fused((int)pass, dtype, ptr(inp), ptr(fil), ptr(out), &p, algorithm, &f, ptr(workspace),
                                        ws_elems, stream());
    });
    return THPVariable_Wrap(out);
  }
  const bool fused = bias.defined() || activation != PDNN_ACT_NONE || alpha != 1.0 || beta != 0.0 || bits.defined() ||
                     (constant_filter && pass == PDNN_FORWARD) || any_order;
  if (fused) {
    if (pass != PDNN_FORWARD) raise(PyExc_ValueError, "the fused epilogue exists for the forward pass only");
    PdnnConvEpilogue e = {};
    e.bias = ptr(bias);
    e.activation = activation;
    e.alpha = (float)alpha;
    e.beta = (float)beta;
    e.relu_bitmask = ptr(bits);
    e.constant_filter = constant_filter;
    e.any_order = any_order;
    call([&] {
      return pdnn_conv2d_fused(dtype, ptr(inp), ptr(fil), ptr(out), &p, algorithm, &e, ptr(workspace), ws_elems, stream());
    });
  } else {
    call([&] {
      return pdnn_conv2d((int)pass, dtype, ptr(inp), ptr(fil), ptr(out), &p, algorithm, ptr(workspace), ws_elems, stream());
    });
  }
  return THPVariable_Wrap(out);
}

PyObject* depthwise_conv2d(PyObject* const* a) {
  const long pass = integer(a[0]);
  const at::Tensor &inp = tensor(a[1]), &fil = tensor(a[2]);
  const PdnnDepthwiseConv2DParams p = params<PdnnDepthwiseConv2DParams>(a[3]);
  at::Tensor out = tensor(a[4]);
  const at::Tensor& workspace = tensor(a[5]);
  require_cuda(inp, fil, out, workspace);
  const int64_t x = (int64_t)p.batch * p.in_rows * p.in_cols * p.channels;
  const int64_t w = (int64_t)p.window_rows * p.window_cols * p.channels * p.channel_multiplier;
  const int64_t y = (int64_t)p.batch * p.out_rows * p.out_cols * p.channels * p.channel_multiplier;
  if (pass < 0 || pass > 2) raise(PyExc_KeyError, "%ld", pass);
  const int64_t n_in = pass == PDNN_INPUT_BACKPROP ? y : x, n_fil = pass == PDNN_FILTER_BACKPROP ? y : w;
  const int64_t n_out = pass == PDNN_FORWARD ? y : pass == PDNN_INPUT_BACKPROP ? x : w;
  if (inp.numel() != n_in || fil.numel() != n_fil) raise(PyExc_ValueError, "tensor sizes do not match the parameters");
  if (!out.defined()) out = flat(n_out, inp.options());
  const int dtype = dtype_code(inp);
  call([&] {
    return pdnn_depthwise_conv2d((int)pass, dtype, ptr(inp), ptr(fil), ptr(out), &p, ptr(workspace),
                                 workspace.defined() ? workspace.nbytes() : 0, stream());
  });
  return THPVariable_Wrap(out);
}

PyObject* pooling(PyObject* const* a) {
  const int op = (int)integer(a[0]), direction = (int)integer(a[1]);
  const at::Tensor& inp = tensor(a[2]);
  const PdnnPoolingParams p = params<PdnnPoolingParams>(a[3]);
  at::Tensor out = tensor(a[4]);
  require_cuda(inp, out);
  if (!out.defined()) {
    const int64_t px = direction == 0 ? (int64_t)p.out_rows * p.out_cols : (int64_t)p.in_rows * p.in_cols;
    out = flat(p.batch * px * p.channels, inp.options());
  }
  const int dtype = dtype_code(inp);
  call([&] { return pdnn_pooling(op, direction, dtype, ptr(inp), ptr(out), &p, stream()); });
  return THPVariable_Wrap(out);
}

PyObject* pooling_max_grad(PyObject* const* a) {
  const int op = (int)integer(a[0]);
  const at::Tensor &x = tensor(a[1]), &y = tensor(a[2]), &dy = tensor(a[3]);
  const PdnnPoolingParams p = params<PdnnPoolingParams>(a[4]);
  at::Tensor out = tensor(a[5]);
  const bool relu_input = truth(a[6]);
  require_cuda(x, y, dy, out);
  if (!out.defined()) out = flat(x.numel(), x.options());
  const int dtype = dtype_code(x);
  call([&] {
    return (relu_input ? pdnn_pooling_max_grad_relu : pdnn_pooling_max_grad)(op, dtype, ptr(x), ptr(y), ptr(dy), ptr(out), &p,
                                                                             stream());
  });
  return THPVariable_Wrap(out);
}

PyObject* pointwise(PyObject* const* a) {
  const int op = (int)integer(a[0]);
  const at::Tensor& inp = tensor(a[1]);
  require_cuda(inp, tensor(a[2]));
  const at::Tensor out = out_or_like(tensor(a[2]), inp);
  const int dtype = dtype_code(inp);
  call([&] { return pdnn_pointwise(op, dtype, ptr(inp), ptr(out), (size_t)inp.numel(), stream()); });
  return THPVariable_Wrap(out);
}

PyObject* pointwise_grad(PyObject* const* a) {
  const int op = (int)integer(a[0]);
  const at::Tensor &fwd = tensor(a[1]), &err = tensor(a[2]);
  require_cuda(fwd, err, tensor(a[3]));
  const at::Tensor out = out_or_like(tensor(a[3]), fwd);
  const int dtype = dtype_code(fwd);
  call([&] { return pdnn_pointwise_grad(op, dtype, ptr(fwd), ptr(err), ptr(out), (size_t)fwd.numel(), stream()); });
  return THPVariable_Wrap(out);
}

PyObject* bias_add(PyObject* const* a) {
  const at::Tensor &inp = tensor(a[0]), &bias = tensor(a[1]);
  const long channels = integer(a[2]);
  require_cuda(inp, bias, tensor(a[4]));
  if (channels == 0) raise(PyExc_ZeroDivisionError, "integer division or modulo by zero");
  const at::Tensor out = out_or_like(tensor(a[4]), inp);
  const int dtype = dtype_code(inp), activation = (int)to_integer(a[3]);
  call([&] {
    return pdnn_bias_add(dtype, ptr(inp), ptr(bias), ptr(out), (size_t)(inp.numel() / channels), (int)channels, activation,
                         stream());
  });
  return THPVariable_Wrap(out);
}

PyObject* scale_blend(PyObject* const* a) {
  const at::Tensor &x = tensor(a[0]), &b = tensor(a[2]);
  require_cuda(x, b, tensor(a[4]));
  const at::Tensor out = out_or_like(tensor(a[4]), x);
  const int dtype = dtype_code(x);
  const float alpha = (float)real(a[1]), beta = (float)real(a[3]);
  call([&] { return pdnn_scale_blend(dtype, ptr(x), alpha, ptr(b), beta, ptr(out), (size_t)x.numel(), stream()); });
  return THPVariable_Wrap(out);
}

// A sequence of extents: all are counted, the first kMostDims kept (the library takes no more than four).
constexpr int kMostDims = 16;
int extents(PyObject* o, int (&d)[kMostDims]) {
  PyObject* seq = PySequence_Fast(o, "expected a sequence of extents");
  if (seq == nullptr) throw PyFailure();
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
  for (Py_ssize_t i = 0; i < n && !PyErr_Occurred(); ++i) {
    PyObject* v = PyNumber_Long(PySequence_Fast_GET_ITEM(seq, i));
    const int extent = v != nullptr ? (int)PyLong_AsLong(v) : 0;
    Py_XDECREF(v);
    if (i < kMostDims) d[i] = extent;
  }
  Py_DECREF(seq);
  if (PyErr_Occurred()) throw PyFailure();
  return (int)n;
}

PyObject* binaryop(PyObject* const* a) {
  const int op = (int)to_integer(a[0]);
  const at::Tensor &lhs = tensor(a[1]), &rhs = tensor(a[3]);
  int ld[kMostDims] = {}, rd[kMostDims] = {};
  require_cuda(lhs, rhs, tensor(a[5]));
  const int nl = extents(a[2], ld), nr = extents(a[4], rd);
  at::Tensor out = tensor(a[5]);
  if (!out.defined()) {
    const int n = nl > nr ? nl : nr;
    int64_t numel = n <= kMostDims ? 1 : 0;  // (more than the library takes)
    for (int i = 0; i < n && numel != 0; ++i) {
      const int l = i < n - nl ? 1 : ld[i - (n - nl)], r = i < n - nr ? 1 : rd[i - (n - nr)];
      const int m = l > r ? l : r;
      numel *= m > 0 ? m : 0;
    }
    out = flat(numel, lhs.options());
  }
  const int dtype = dtype_code(lhs);
  call([&] { return pdnn_binaryop(op, dtype, ptr(lhs), ld, nl, ptr(rhs), rd, nr, ptr(out), stream()); });
  return THPVariable_Wrap(out);
}

PyObject* matmul(PyObject* const* a) {
  const at::Tensor &lhs = tensor(a[0]), &rhs = tensor(a[1]);
  auto extent = [](PyObject* o) {  // 8.0 is one, 8.5 is not
    return PyFloat_Check(o) && PyFloat_AS_DOUBLE(o) == (double)(int)PyFloat_AS_DOUBLE(o) ? to_integer(o) : integer(o);
  };
  const long batches = extent(a[2]), m = extent(a[3]), k = extent(a[4]), n = extent(a[5]);
  const bool tl = truth(a[6]), tr = truth(a[7]);
  const double beta = real(a[8]);
  at::Tensor out = tensor(a[9]);
  require_cuda(lhs, rhs, out);
  if (lhs.numel() != (int64_t)batches * m * k || rhs.numel() != (int64_t)batches * k * n)
    raise(PyExc_ValueError, "tensor sizes do not match the parameters");
  if (!out.defined()) {
    if (beta != 0.0) raise(PyExc_ValueError, "beta != 0 needs an output tensor to accumulate into");
    out = flat((int64_t)batches * m * n, lhs.options());
  }
  const int dtype = dtype_code(lhs);
  call([&] {
    return pdnn_matmul(dtype, tl, tr, ptr(lhs), ptr(rhs), ptr(out), (int)batches, (int)m, (int)k, (int)n, (float)beta, stream());
  });
  return THPVariable_Wrap(out);
}

PyObject* softmax(PyObject* const* a) {
  const at::Tensor &inp = tensor(a[0]), &gradient = tensor(a[5]);
  const long batch = integer(a[1]), rows = integer(a[2]), cols = integer(a[3]), channels = integer(a[4]);
  require_cuda(inp, gradient, tensor(a[6]));
  if (inp.numel() != (int64_t)batch * rows * cols * channels)
    raise(PyExc_ValueError, "tensor size does not match the parameters");
  const at::Tensor out = out_or_like(tensor(a[6]), inp);
  PdnnSoftmaxParams p = {};
  p.channels = (int)channels;
  p.batch = (int)batch;
  p.rows = (int)rows;
  p.cols = (int)cols;
  const int dtype = dtype_code(inp);
  call([&] { return pdnn_softmax(gradient.defined() ? 1 : 0, dtype, ptr(inp), ptr(gradient), ptr(out), &p, stream()); });
  return THPVariable_Wrap(out);
}

// (a, b, c) with None for an undefined tensor.
PyObject* triple(const at::Tensor& a, const at::Tensor& b, const at::Tensor& c) {
  PyObject* t = PyTuple_New(3);
  if (t == nullptr) throw PyFailure();
  int i = 0;
  for (const at::Tensor* v : {&a, &b, &c}) {
    PyObject* o = v->defined() ? THPVariable_Wrap(*v) : Py_NewRef(Py_None);
    if (o == nullptr) {
      Py_DECREF(t);
      throw PyFailure();
    }
    PyTuple_SET_ITEM(t, i++, o);
  }
  return t;
}

PyObject* batchnorm_forward(PyObject* const* a) {
  const at::Tensor &inp = tensor(a[0]), &beta = tensor(a[1]), &gamma = tensor(a[2]), &mean = tensor(a[3]),
                   &variance = tensor(a[4]);
  const PdnnBatchNormParams p = params<PdnnBatchNormParams>(a[5]);
  require_cuda(inp, beta, gamma, mean, variance, tensor(a[6]));
  const at::Tensor out = out_or_like(tensor(a[6]), inp);
  at::Tensor rm, rv;
  if (p.is_training) {
    rm = like(mean);
    rv = like(variance);
  }
  const int dtype = dtype_code(inp);
  call([&] {
    return pdnn_batchnorm_forward(dtype, ptr(inp), ptr(beta), ptr(gamma), ptr(mean), ptr(variance), ptr(rm), ptr(rv), ptr(out),
                                  &p, stream());
  });
  return triple(out, rm, rv);
}

PyObject* batchnorm_gradient(PyObject* const* a) {
  const at::Tensor &inp = tensor(a[0]), &gradient = tensor(a[1]), &gamma = tensor(a[2]);
  const PdnnBatchNormParams p = params<PdnnBatchNormParams>(a[3]);
  const at::Tensor &pop_mean = tensor(a[4]), &pop_variance = tensor(a[5]);
  require_cuda(inp, gradient, gamma, pop_mean, pop_variance, tensor(a[6]));
  const at::Tensor out = out_or_like(tensor(a[6]), inp), bg = like(gamma), gg = like(gamma);
  const int dtype = dtype_code(inp);
  call([&] {
    return pdnn_batchnorm_gradient(dtype, ptr(inp), ptr(gradient), ptr(gamma), ptr(pop_mean), ptr(pop_variance), ptr(bg),
                                   ptr(gg), ptr(out), &p, stream());
  });
  return triple(out, bg, gg);
}

// ---- the operators around a block's matrix products -----------------------------------------------------

// A matrix argument: two dimensions, a row's elements next to each other, rows any distance apart.
struct MatrixArg {
  at::Tensor t;
  int64_t rows = 0, cols = 0;
  long long pitch = 0;
};
MatrixArg matrix(PyObject* o, const char* name) {
  MatrixArg m;
  m.t = tensor(o);
  if (!m.t.defined()) return m;
  if (!m.t.is_cuda() || m.t.dim() != 2) raise(PyExc_ValueError, "%s must be a CUDA tensor of two dimensions", name);
  m.rows = m.t.size(0);
  m.cols = m.t.size(1);
  const bool one_row = m.rows <= 1;
  if (m.t.numel() > 0 && ((m.cols > 1 && m.t.stride(1) != 1) || (!one_row && m.t.stride(0) < m.cols)))
    raise(PyExc_ValueError, "the elements of %s's rows must be next to each other, and its rows must not overlap", name);
  m.pitch = one_row || m.t.numel() == 0 ? m.cols : m.t.stride(0);
  return m;
}
void require_shape(const MatrixArg& m, int64_t rows, int64_t cols, const at::Tensor& like, const char* name) {
  if (!m.t.defined()) return;
  if (m.rows != rows || m.cols != cols)
    raise(PyExc_ValueError, "%s must be [%lld, %lld], not [%lld, %lld]", name, (long long)rows, (long long)cols, (long long)m.rows,
          (long long)m.cols);
  if (m.t.scalar_type() != like.scalar_type() || m.t.device() != like.device())
    raise(PyExc_ValueError, "%s must have the other tensors' type and device", name);
}
// A vector, or another dense tensor, of so many elements.
at::Tensor dense(PyObject* o, int64_t numel, const at::Tensor& like, at::ScalarType type, const char* name) {
  const at::Tensor t = tensor(o);
  if (!t.defined()) return t;
  if (!t.is_cuda() || !t.is_contiguous()) raise(PyExc_ValueError, "tensors must be contiguous CUDA tensors");
  if (t.numel() != numel) raise(PyExc_ValueError, "%s must have %lld elements, not %lld", name, (long long)numel, (long long)t.numel());
  if (t.scalar_type() != type || t.device() != like.device())
    raise(PyExc_ValueError, "%s must have the type %s and the other tensors' device", name, c10::toString(type));
  return t;
}
at::Tensor dense(PyObject* o, int64_t numel, const at::Tensor& like, const char* name) {
  return dense(o, numel, like, like.scalar_type(), name);
}
int extent(int64_t v) {
  if (v > 0x7FFFFFFFll) raise(PyExc_ValueError, "an extent of %lld is too large", (long long)v);
  return (int)v;
}
// The current device is the tensors' own while the library runs: a call with tensors of another device goes there, on that
// device's current stream.
struct OnDevice {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit OnDevice(const at::Tensor& t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};
// A new tensor on the device of `like`, past the dispatcher (0.4 us, and a call of these operators makes up to seven).
at::Tensor fresh(at::IntArrayRef sizes, const at::Tensor& like, at::ScalarType type) {
  return unlocked([&] { return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt); });
}
at::Tensor fresh_like(const at::Tensor& t) { return fresh(t.sizes(), t, t.scalar_type()); }
MatrixArg new_matrix(int64_t rows, int64_t cols, const at::Tensor& like) {
  MatrixArg m;
  m.t = fresh({rows, cols}, like, like.scalar_type());
  m.rows = rows;
  m.cols = cols;
  m.pitch = cols;
  return m;
}
PyObject* wrap_or_none(const at::Tensor& t) { return t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None); }
template <size_t N>
PyObject* tuple_of(const at::Tensor (&list)[N]) {
  PyObject* t = PyTuple_New(N);
  if (t == nullptr) throw PyFailure();
  for (size_t i = 0; i < N; ++i) {
    PyObject* o = wrap_or_none(list[i]);
    if (o == nullptr) {
      Py_DECREF(t);
      throw PyFailure();
    }
    PyTuple_SET_ITEM(t, (Py_ssize_t)i, o);
  }
  return t;
}

PyObject* matmul_fused(PyObject* const* a) {
  const MatrixArg lhs = matrix(a[0], "lhs"), rhs = matrix(a[1], "rhs");
  if (!lhs.t.defined() || !rhs.t.defined()) raise(PyExc_ValueError, "lhs and rhs are needed");
  const bool tr = truth(a[2]);
  const int dtype = dtype_code(lhs.t);
  const int64_t m = lhs.rows, k = lhs.cols, n = tr ? rhs.rows : rhs.cols;
  require_shape(rhs, tr ? n : k, tr ? k : n, lhs.t, "rhs");
  const at::Tensor bias = dense(a[3], n, lhs.t, "bias");
  PdnnMatmulEpilogue e = {};
  e.activation = (int)to_integer(a[4]);
  const MatrixArg residual = matrix(a[5], "residual");
  e.scale = (float)real(a[6]);
  const MatrixArg pre = matrix(a[7], "pre_activation");
  MatrixArg out = matrix(a[8], "out");
  require_shape(residual, m, n, lhs.t, "residual");
  require_shape(pre, m, n, lhs.t, "pre_activation");
  require_shape(out, m, n, lhs.t, "out");
  if (!out.t.defined()) out = new_matrix(m, n, lhs.t);
  e.bias = ptr(bias);
  e.residual = ptr(residual.t);
  e.residual_pitch = residual.pitch;
  e.pre_activation = ptr(pre.t);
  e.pre_activation_pitch = pre.pitch;
  const PdnnMatmulParams p = {extent(m), extent(k), extent(n), tr, lhs.pitch, rhs.pitch, out.pitch};
  const OnDevice on(lhs.t);
  call([&] { return pdnn_matmul_fused(dtype, ptr(lhs.t), ptr(rhs.t), ptr(out.t), &p, &e, on.stream); });
  return THPVariable_Wrap(out.t);
}

PyObject* matmul_fused_grad(PyObject* const* a) {
  const MatrixArg grad = matrix(a[0], "grad"), lhs = matrix(a[1], "lhs"), rhs = matrix(a[2], "rhs");
  if (!grad.t.defined() || !lhs.t.defined() || !rhs.t.defined()) raise(PyExc_ValueError, "grad, lhs and rhs are needed");
  const bool tr = truth(a[3]);
  const int dtype = dtype_code(lhs.t);
  const int64_t m = lhs.rows, k = lhs.cols, n = tr ? rhs.rows : rhs.cols;
  require_shape(rhs, tr ? n : k, tr ? k : n, lhs.t, "rhs");
  require_shape(grad, m, n, lhs.t, "grad");
  PdnnMatmulGradient g = {};
  g.activation = (int)to_integer(a[4]);
  const MatrixArg pre = matrix(a[5], "pre_activation");
  g.scale = (float)real(a[6]);
  g.input_activation = (int)to_integer(a[7]);
  const MatrixArg input_pre = matrix(a[8], "input_pre_activation");
  const bool want[3] = {truth(a[9]), truth(a[10]), truth(a[11])};
  MatrixArg dl = matrix(a[12], "lhs_grad"), dr = matrix(a[13], "rhs_grad");
  at::Tensor db = dense(a[14], n, lhs.t, "bias_grad");
  require_shape(pre, m, n, lhs.t, "pre_activation");
  require_shape(input_pre, m, k, lhs.t, "input_pre_activation");
  require_shape(dl, m, k, lhs.t, "lhs_grad");
  require_shape(dr, rhs.rows, rhs.cols, lhs.t, "rhs_grad");
  if (!dl.t.defined() && want[0]) dl = new_matrix(m, k, lhs.t);
  if (!dr.t.defined() && want[1]) dr = new_matrix(rhs.rows, rhs.cols, lhs.t);
  if (!db.defined() && want[2]) db = fresh({n}, lhs.t, lhs.t.scalar_type());
  g.pre_activation = ptr(pre.t);
  g.pre_activation_pitch = pre.pitch;
  g.input_pre_activation = ptr(input_pre.t);
  g.input_pre_activation_pitch = input_pre.pitch;
  g.lhs_grad = ptr(dl.t);
  g.lhs_grad_pitch = dl.pitch;
  g.rhs_grad = ptr(dr.t);
  g.rhs_grad_pitch = dr.pitch;
  g.bias_grad = ptr(db);
  const PdnnMatmulParams p = {extent(m), extent(k), extent(n), tr, lhs.pitch, rhs.pitch, grad.pitch};
  const OnDevice on(lhs.t);
  call([&] { return pdnn_matmul_fused_gradient(dtype, ptr(grad.t), ptr(lhs.t), ptr(rhs.t), &p, &g, on.stream); });
  return tuple_of({dl.t, dr.t, db});
}

// Tensors of the residual norm that both directions read.
struct NormTensors {
  PdnnResidualNormParams p;
  int64_t numel;
  at::Tensor branch, post_gamma, post_beta, gate, pre_gamma, pre_beta;
  NormTensors(PyObject* b, PyObject* params_, PyObject* const* vectors) : p(params<PdnnResidualNormParams>(params_)) {
    branch = tensor(b);
    if (!branch.defined() || !branch.is_cuda() || !branch.is_contiguous())
      raise(PyExc_ValueError, "tensors must be contiguous CUDA tensors");
    if (p.rows < 0 || p.channels < 0 || p.gate_groups < 0) raise(PyExc_ValueError, "negative extents");
    numel = (int64_t)p.rows * p.channels;
    dense(b, numel, branch, "branch");
    post_gamma = dense(vectors[0], p.channels, branch, "post_gamma");
    post_beta = dense(vectors[1], p.channels, branch, "post_beta");
    gate = dense(vectors[2], (int64_t)p.gate_groups * p.channels, branch, "gate");
    pre_gamma = dense(vectors[3], p.channels, branch, "pre_gamma");
    pre_beta = dense(vectors[4], p.channels, branch, "pre_beta");
  }
  PdnnResidualNormTensors tensors() const {
    PdnnResidualNormTensors t = {};
    t.branch = ptr(branch);
    t.post_gamma = ptr(post_gamma);
    t.post_beta = ptr(post_beta);
    t.gate = ptr(gate);
    t.pre_gamma = ptr(pre_gamma);
    t.pre_beta = ptr(pre_beta);
    return t;
  }
};

PyObject* residual_norm(PyObject* const* a) {
  const NormTensors n(a[0], a[2], a + 3);
  const at::Tensor residual = dense(a[1], n.numel, n.branch, "residual");
  at::Tensor sum = dense(a[8], n.numel, n.branch, "sum_out"), out = dense(a[9], n.numel, n.branch, "out");
  const int dtype = dtype_code(n.branch);
  if (!sum.defined()) sum = fresh_like(n.branch);
  if (!out.defined()) out = fresh_like(n.branch);
  const at::Tensor statistics = fresh({4, (int64_t)n.p.rows}, n.branch, at::kFloat);
  PdnnResidualNormTensors t = n.tensors();
  t.residual = ptr(residual);
  t.sum = ptr(sum);
  t.output = ptr(out);
  t.statistics = static_cast<float*>(ptr(statistics));
  const OnDevice on(n.branch);
  call([&] { return pdnn_residual_norm(dtype, &n.p, &t, on.stream); });
  return tuple_of({sum, out, statistics});
}

PyObject* residual_norm_grad(PyObject* const* a) {
  const NormTensors n(a[2], a[5], a + 6);
  const at::Tensor d_sum = dense(a[0], n.numel, n.branch, "sum_grad"), d_out = dense(a[1], n.numel, n.branch, "output_grad");
  const at::Tensor sum = dense(a[3], n.numel, n.branch, "sum");
  const at::Tensor statistics = dense(a[4], 4 * (int64_t)n.p.rows, n.branch, at::kFloat, "statistics");
  if (!d_out.defined() || !sum.defined() || !statistics.defined()) raise(PyExc_ValueError, "output_grad, sum and statistics are needed");
  at::Tensor d_branch = dense(a[11], n.numel, n.branch, "branch_grad"), d_residual = dense(a[12], n.numel, n.branch, "residual_grad");
  const int dtype = dtype_code(n.branch);
  if (!d_branch.defined()) d_branch = fresh_like(n.branch);
  if (!d_residual.defined()) d_residual = fresh_like(n.branch);
  const at::Tensor of[5] = {n.post_gamma, n.post_beta, n.gate, n.pre_gamma, n.pre_beta};
  at::Tensor d[5];
  for (int i = 0; i < 5; ++i)
    if (of[i].defined()) d[i] = fresh_like(of[i]);
  PdnnResidualNormTensors t = n.tensors();
  t.sum = ptr(sum);
  t.statistics = static_cast<float*>(ptr(statistics));
  PdnnResidualNormGradients g = {};
  g.sum_grad = ptr(d_sum);
  g.output_grad = ptr(d_out);
  g.branch_grad = ptr(d_branch);
  g.residual_grad = ptr(d_residual);
  g.post_gamma_grad = ptr(d[0]);
  g.post_beta_grad = ptr(d[1]);
  g.gate_grad = ptr(d[2]);
  g.pre_gamma_grad = ptr(d[3]);
  g.pre_beta_grad = ptr(d[4]);
  const OnDevice on(n.branch);
  call([&] { return pdnn_residual_norm_gradient(dtype, &n.p, &t, &g, on.stream); });
  return tuple_of({d_branch, d_residual, d[0], d[1], d[2], d[3], d[4]});
}

PyObject* policy_loss(PyObject* const* a) {
  const MatrixArg logits = matrix(a[0], "logits");
  if (!logits.t.defined()) raise(PyExc_ValueError, "logits are needed");
  const int dtype = dtype_code(logits.t);
  const int64_t rows = logits.rows;
  const at::Tensor targets = tensor(a[1]);
  if (!targets.defined() || (targets.scalar_type() != at::kLong && targets.scalar_type() != at::kInt))
    raise(PyExc_ValueError, "targets must be a tensor of whole numbers of 32 or 64 bits");
  dense(a[1], rows, logits.t, targets.scalar_type(), "targets");
  const at::Tensor advantages = dense(a[2], rows, logits.t, at::kFloat, "advantages"),
                   old_logp = dense(a[3], rows, logits.t, at::kFloat, "old_logp"),
                   ref_logp = dense(a[4], rows, logits.t, at::kFloat, "ref_logp"),
                   weights = dense(a[5], rows, logits.t, at::kFloat, "weights");
  if (!advantages.defined()) raise(PyExc_ValueError, "advantages are needed");
  PdnnPolicyLossParams p = {};
  p.rows = extent(rows);
  p.vocab = extent(logits.cols);
  p.target_bytes = (int)targets.element_size();
  p.clip_low = (float)real(a[6]);
  p.clip_high = (float)real(a[7]);
  p.kl = (float)real(a[8]);
  p.temperature = (float)real(a[9]);
  p.grad_scale = (float)real(a[10]);
  const bool want_grad = truth(a[11]);
  MatrixArg grad = matrix(a[12], "grad");
  require_shape(grad, rows, logits.cols, logits.t, "grad");
  if (!grad.t.defined() && want_grad) {
    // dense, or in rows of whole packets where the logits' rows lie apart
    const int64_t pitch = logits.pitch == logits.cols ? logits.cols : (logits.cols + 63) / 64 * 64;
    grad = new_matrix(rows, pitch, logits.t);
    grad.t = grad.t.narrow(1, 0, logits.cols);
  }
  p.logits_pitch = logits.pitch;
  p.grad_pitch = grad.pitch;
  const at::Tensor loss = fresh({}, logits.t, at::kFloat), token_loss = fresh({rows}, logits.t, at::kFloat),
                   logp = fresh({rows}, logits.t, at::kFloat);
  PdnnPolicyLossTensors t = {};
  t.logits = ptr(logits.t);
  t.targets = ptr(targets);
  t.advantages = static_cast<const float*>(ptr(advantages));
  t.old_logp = static_cast<const float*>(ptr(old_logp));
  t.ref_logp = static_cast<const float*>(ptr(ref_logp));
  t.weights = static_cast<const float*>(ptr(weights));
  t.loss = static_cast<float*>(ptr(loss));
  t.token_loss = static_cast<float*>(ptr(token_loss));
  t.logp = static_cast<float*>(ptr(logp));
  t.grad = ptr(grad.t);
  const OnDevice on(logits.t);
  call([&] { return pdnn_policy_loss(dtype, &p, &t, on.stream); });
  return tuple_of({loss, token_loss, logp, grad.t});
}

// The CPython face of one of the functions above: argument count, C++ exceptions to Python ones.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
    return nullptr;
  }
  HANDLE_TH_ERRORS
  try {
    return F(args);
  } catch (const PyFailure&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

#define ENTRY(name, n) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<name, n>)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {ENTRY(conv2d, 17),
                          ENTRY(depthwise_conv2d, 6),
                          ENTRY(pooling, 5),
                          ENTRY(pooling_max_grad, 7),
                          ENTRY(pointwise, 3),
                          ENTRY(pointwise_grad, 4),
                          ENTRY(bias_add, 5),
                          ENTRY(scale_blend, 5),
                          ENTRY(binaryop, 6),
                          ENTRY(matmul, 10),
                          ENTRY(softmax, 7),
                          ENTRY(batchnorm_forward, 7),
                          ENTRY(batchnorm_gradient, 7),
                          ENTRY(matmul_fused, 9),
                          ENTRY(matmul_fused_grad, 15),
                          ENTRY(residual_norm, 10),
                          ENTRY(residual_norm_grad, 13),
                          ENTRY(policy_loss, 13),
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_front", "Native half of portdnn_b200.api.", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__front(void) { return PyModule_Create(&kModule); }
