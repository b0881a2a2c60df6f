// Host side of the microscaled calls: argument checks, output allocation and the launch through the C ABI, as a CPython
// extension module (nesgpu_b200._host).
//
// A call of these operators on a few rows takes the device 2 to 8 us; checked, allocated and launched from Python through
// ctypes it took the host 11 us (a torch.empty 2 us, a ctypes call with its arguments 1.2 us beside the launch, the checks the
// rest), from here 3.6 to 5.7.  Functions take positional arguments only and are called by nesgpu_b200/microscaling.py, which documents them.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <optional>
#include <vector>

#include "../../include/nesgpu_b200.h"

namespace {

struct Raised {};                        // a Python exception has been set

[[noreturn]] void refuse(PyObject* type, const char* format, ...) {
  va_list ap;
  va_start(ap, format);
  PyErr_FormatV(type, format, ap);
  va_end(ap);
  throw Raised();
}

PyObject* dtype_object(at::ScalarType t) { return reinterpret_cast<PyObject*>(torch::getTHPDtype(t)); }

const at::Tensor& cuda_tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o) || !THPVariable_Unpack(o).is_cuda())
    refuse(PyExc_RuntimeError, "nesgpu_b200: %s must be a CUDA tensor (there is no CPU path)", name);
  return THPVariable_Unpack(o);
}

at::Tensor contiguous(const at::Tensor& t) { return t.is_contiguous() ? t : t.contiguous(); }

// `t` at an address that is a multiple of 16 bytes (a copy if it starts inside an allocation)
at::Tensor aligned(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 ? t.clone() : t; }

at::Tensor of_type(PyObject* o, const char* name, at::ScalarType type) {
  const at::Tensor& t = cuda_tensor(o, name);
  if (t.scalar_type() != type)
    refuse(PyExc_NotImplementedError, "nesgpu_b200: %s must have dtype %S, got %S", name, dtype_object(type), dtype_object(t.scalar_type()));
  return contiguous(t);
}

int kind_of(at::ScalarType t, const char* name) {
  switch (t) {
    case at::kFloat: return NES_F32;
    case at::kBFloat16: return NES_BF16;
    case at::kHalf: return NES_F16;
    default: refuse(PyExc_NotImplementedError, "nesgpu_b200: %s must have dtype float32, bfloat16 or float16, got %S", name, dtype_object(t));
  }
}

void same_device(const at::Tensor& t, const at::Device& device, const char* name) {
  if (t.device() != device)
    refuse(PyExc_RuntimeError, "nesgpu_b200: %s is on %s, expected %s", name, t.device().str().c_str(), device.str().c_str());
}

int64_t pitch(int64_t cols, int64_t format) { return (cols + 127) / 128 * (format == NES_MXFP4 ? 64 : 128); }
int64_t scale_pitch(int64_t cols) { return (cols + 127) / 128 * 4; }

// A contiguous plain tensor of at least one column as rows.
struct Rows {
  at::Tensor t;
  int64_t rows, cols;
  int kind;
  Rows(PyObject* o, const char* name) {
    const at::Tensor& given = cuda_tensor(o, name);
    kind = kind_of(given.scalar_type(), name);
    if (given.dim() == 0 || given.size(-1) == 0) {
      PyObject* shape = PyObject_GetAttrString(o, "shape");
      PyObject* tuple = shape ? PySequence_Tuple(shape) : nullptr;
      PyErr_Format(PyExc_RuntimeError, "%s needs at least one column, got shape %S", name, tuple ? tuple : Py_None);
      Py_XDECREF(tuple);
      Py_XDECREF(shape);
      throw Raised();
    }
    t = contiguous(given);
    cols = t.size(-1);
    rows = t.numel() / cols;
  }
};

// uninitialised, contiguous, on the device of `like`: the caching allocator without the dispatcher's way to it
at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}
at::Tensor bytes(const at::Tensor& like, int64_t rows, int64_t width) { return empty({rows, width}, at::kByte, like); }

// Makes a tensor's device current for a launch and gives the stream that is current there.
struct Launch {
  c10::cuda::OptionalCUDAGuard guard;
  nes_stream_t stream;
  explicit Launch(const at::Device& d) {
    if (d.index() != c10::cuda::current_device()) guard.set_index(d.index());
    stream = c10::cuda::getCurrentCUDAStream(d.index()).stream();
  }
};

// Calls an entry point without the interpreter's lock, as a ctypes call does (a launch waits while the device's queue is full);
// status -> NotImplementedError or nesgpu_b200._cabi.NesError.
template <typename F>
void run(const char* name, F&& call) {
  PyThreadState* state = PyEval_SaveThread();
  const int status = call();
  PyEval_RestoreThread(state);
  if (status == NES_OK) return;
  PyObject* type = PyExc_NotImplementedError;
  if (status != NES_ERR_UNSUPPORTED) {
    PyObject* module = PyImport_ImportModule("nesgpu_b200._cabi");
    type = module ? PyObject_GetAttrString(module, "NesError") : nullptr;
    Py_XDECREF(module);
    if (!type) throw Raised();
  }
  PyErr_Format(type, "%s: %s (%s)", name, nes_status_string(status), nes_last_error());
  if (status != NES_ERR_UNSUPPORTED) Py_DECREF(type);
  throw Raised();
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised();
  return v == 1;
}

int64_t whole(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised();
  return v;
}

// (lead ..., last); lead: a tuple of whole numbers whose product is `rows`
std::vector<int64_t> sizes_of(PyObject* lead, int64_t last, int64_t rows) {
  std::vector<int64_t> s;
  const Py_ssize_t n = PyTuple_Size(lead);
  if (n < 0) throw Raised();
  int64_t product = 1;
  for (Py_ssize_t i = 0; i < n; ++i) {
    s.push_back(whole(PyTuple_GET_ITEM(lead, i)));
    product *= s.back();
  }
  if (product != rows) refuse(PyExc_RuntimeError, "leading dimensions %R do not match %lld rows", lead, (long long)rows);
  s.push_back(last);
  return s;
}

PyObject* lead_of(const at::Tensor& t) {
  PyObject* lead = PyTuple_New(t.dim() - 1);
  if (!lead) throw Raised();
  for (int64_t i = 0; i + 1 < t.dim(); ++i) PyTuple_SET_ITEM(lead, i, PyLong_FromLongLong(t.size(i)));
  return lead;
}

// (codes, scales, rows, cols, leading dimensions) of new blocks for the rows of `like`
PyObject* blocks_tuple(const at::Tensor& codes, const at::Tensor& scales, const Rows& x) {
  PyObject* lead = lead_of(x.t);
  return Py_BuildValue("(NNLLN)", THPVariable_Wrap(codes), THPVariable_Wrap(scales), (long long)x.rows, (long long)x.cols, lead);
}

// (codes, scales, cols, format) -> (codes, scales, rows): checked, contiguous and aligned as the kernels read them
PyObject* blocks(PyObject* const* a) {
  at::Tensor codes = of_type(a[0], "codes", at::kByte), scales = of_type(a[1], "scales", at::kByte);
  const int64_t cols = whole(a[2]), format = whole(a[3]);
  if (cols < 1) refuse(PyExc_RuntimeError, "a microscaled tensor needs at least one column");
  same_device(scales, codes.device(), "scales");
  if (codes.dim() != 2 || scales.dim() != 2 || codes.size(1) != pitch(cols, format) || scales.size(1) != scale_pitch(cols) ||
      codes.size(0) != scales.size(0))
    refuse(PyExc_RuntimeError, "codes and scales of %lld columns in %s must be (rows, %lld) and (rows, %lld)", (long long)cols,
           format == NES_MXFP4 ? "mxfp4" : "mxfp8", (long long)pitch(cols, format), (long long)scale_pitch(cols));
  if (reinterpret_cast<uintptr_t>(codes.data_ptr()) % 32) codes = codes.clone();       // read in aligned 16- and 32-byte pieces
  if (reinterpret_cast<uintptr_t>(scales.data_ptr()) % 4) scales = scales.clone();
  return Py_BuildValue("(NNL)", THPVariable_Wrap(codes), THPVariable_Wrap(scales), (long long)codes.size(0));
}

// The tensors of blocks that exist already, looked at again where they are used: the object that holds them may have been given
// others, or one of them resized, since `blocks` saw them.  `like`: the codes that scales belong to.
void as_made(const at::Tensor& t, int64_t width, const char* name, const at::Tensor* like = nullptr) {
  if (t.scalar_type() != at::kByte || t.dim() != 2 || t.size(1) != width || !t.is_contiguous() || (like && t.size(0) != like->size(0)))
    refuse(PyExc_RuntimeError, "%s of a microscaled tensor must be contiguous uint8 of %lld bytes to a row, and as many rows of codes as of scales", name,
           (long long)width);
  if (like) same_device(t, like->device(), name);
}

PyObject* quantize(PyObject* const* a) {
  const Rows x(a[0], "input");
  const int64_t format = whole(a[1]);
  at::Tensor codes = bytes(x.t, x.rows, pitch(x.cols, format)), scales = bytes(x.t, x.rows, scale_pitch(x.cols));
  const Launch launch(x.t.device());
  run("nes_mx_quantize", [&] {
    return nes_mx_quantize(x.t.data_ptr(), x.kind, codes.data_ptr(), scales.data_ptr<uint8_t>(), x.rows, x.cols, int(format), launch.stream);
  });
  return blocks_tuple(codes, scales, x);
}

// the first `width` bytes of every row of `t` with leading dimensions `lead`, as elements of `type`
PyObject* view_rows(const at::Tensor& t, PyObject* lead, int64_t width, at::ScalarType type) {
  const std::vector<int64_t> sizes = sizes_of(lead, width, t.size(0));
  std::vector<int64_t> strides(sizes.size(), 1);
  int64_t stride = t.size(1);
  for (size_t i = sizes.size() - 1; i-- > 0;) {
    strides[i] = stride;
    stride *= sizes[i];
  }
  return THPVariable_Wrap(t.as_strided(sizes, strides).view(type));
}

// (codes, cols, lead, format)
PyObject* elements(PyObject* const* a) {
  const at::Tensor& codes = cuda_tensor(a[0], "codes");
  const int64_t cols = whole(a[1]);
  const int64_t format = whole(a[3]);
  as_made(codes, pitch(cols, format), "codes");
  if (format == NES_MXFP8) return view_rows(codes, a[2], cols, at::kFloat8_e4m3fn);
  at::Tensor out = empty(sizes_of(a[2], cols, codes.size(0)), at::kFloat8_e4m3fn, codes);
  const Launch launch(codes.device());
  run("nes_mx_elements", [&] { return nes_mx_elements(codes.data_ptr(), static_cast<uint8_t*>(out.data_ptr()), codes.size(0), cols, launch.stream); });
  return THPVariable_Wrap(out);
}

// (scales, cols, lead)
PyObject* block_scales(PyObject* const* a) {
  const at::Tensor& scales = cuda_tensor(a[0], "scales");
  const int64_t cols = whole(a[1]);
  as_made(scales, scale_pitch(cols), "scales");
  return view_rows(scales, a[2], (cols + 31) / 32, at::kFloat8_e8m0fnu);
}

at::ScalarType dtype_argument(PyObject* o) {
  if (!THPDtype_Check(o)) refuse(PyExc_NotImplementedError, "nesgpu_b200: the result must have dtype float32, bfloat16 or float16, got %S", o);
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}

// (codes, scales, cols, lead, format, dtype)
PyObject* dequantize(PyObject* const* a) {
  const at::Tensor &codes = cuda_tensor(a[0], "codes"), &scales = cuda_tensor(a[1], "scales");
  const int64_t cols = whole(a[2]), format = whole(a[4]);
  const at::ScalarType type = dtype_argument(a[5]);
  const int kind = kind_of(type, "the result");
  as_made(codes, pitch(cols, format), "codes");
  as_made(scales, scale_pitch(cols), "scales", &codes);
  at::Tensor out = empty(sizes_of(a[3], cols, codes.size(0)), type, codes);
  const Launch launch(codes.device());
  run("nes_mx_dequantize", [&] {
    return nes_mx_dequantize(codes.data_ptr(), scales.data_ptr<uint8_t>(), out.data_ptr(), kind, codes.size(0), cols, int(format), launch.stream);
  });
  return THPVariable_Wrap(out);
}

// (input, its scales or None, its lead or None, its cols, its format, weight codes, weight scales, in_features, weight format, bias, dtype, out)
PyObject* linear(PyObject* const* a) {
  const bool microscaled = a[1] != Py_None;
  const int64_t x_format = whole(a[4]), in_features = whole(a[7]), w_format = whole(a[8]);
  const at::Tensor &w = cuda_tensor(a[5], "weight codes"), &w_scales = cuda_tensor(a[6], "weight scales");
  as_made(w, pitch(in_features, w_format), "codes");
  as_made(w_scales, scale_pitch(in_features), "scales", &w);
  const int64_t out_features = w.size(0);
  std::optional<Rows> plain;
  if (!microscaled) plain.emplace(a[0], "input");
  const at::Tensor& x = microscaled ? cuda_tensor(a[0], "codes") : plain->t;
  const at::Tensor* x_scales = microscaled ? &cuda_tensor(a[1], "scales") : nullptr;
  if (microscaled) {
    as_made(x, pitch(whole(a[3]), x_format), "codes");
    as_made(*x_scales, scale_pitch(whole(a[3])), "scales", &x);
  }
  const int64_t rows = microscaled ? x.size(0) : plain->rows, cols = microscaled ? whole(a[3]) : plain->cols;
  const bool has_out = a[11] != Py_None;
  at::ScalarType type = microscaled ? at::kFloat : x.scalar_type();
  if (a[10] != Py_None) type = dtype_argument(a[10]);
  else if (has_out && THPVariable_Check(a[11])) type = THPVariable_Unpack(a[11]).scalar_type();
  const int kind = kind_of(type, "the result");
  if (cols != in_features)
    refuse(PyExc_RuntimeError, "expected last dimension %lld, got %lld", (long long)in_features, (long long)cols);
  const at::Device device = x.device();
  same_device(w, device, "weight");
  at::Tensor bias;
  if (a[9] != Py_None) {
    bias = of_type(a[9], "bias", at::kFloat);
    if (bias.dim() != 1 || bias.size(0) != out_features)
      refuse(PyExc_RuntimeError, "bias must have shape (%lld,)", (long long)out_features);
    same_device(bias, device, "bias");
  }
  at::Tensor y;
  if (has_out) {
    y = cuda_tensor(a[11], "out");
    if (y.device() != device || y.scalar_type() != type || !y.is_contiguous() || y.numel() != rows * out_features)
      refuse(PyExc_RuntimeError, "out must be a contiguous %S tensor of %lld elements on %s", dtype_object(type), (long long)(rows * out_features),
             device.str().c_str());
  } else if (microscaled) {
    y = empty(sizes_of(a[2], out_features, rows), type, x);
  } else {
    std::vector<int64_t> sizes(x.sizes().begin(), x.sizes().end());
    sizes.back() = out_features;
    y = empty(sizes, type, x);
  }
  const Launch launch(device);
  // a workspace of this call's own: calls captured into different graphs share nothing
  at::Tensor scratch;
  const int64_t need = microscaled ? 0 : nes_mx_linear_fwd_scratch_bytes(rows, out_features, in_features, int(x_format));
  if (need) scratch = empty({need}, at::kByte, x);
  run("nes_mx_linear_fwd", [&] {
    return nes_mx_linear_fwd(x.data_ptr(), x_scales ? x_scales->data_ptr<uint8_t>() : nullptr, microscaled ? 0 : plain->kind, int(x_format), w.data_ptr(),
                             w_scales.data_ptr<uint8_t>(), int(w_format), bias.defined() ? bias.data_ptr<float>() : nullptr, y.data_ptr(), kind, rows,
                             out_features, in_features, need ? scratch.data_ptr() : nullptr, need, launch.stream);
  });
  return THPVariable_Wrap(y);
}

// (input, weight, eps, residual, noise, antithetic, format); format 0: y has the input's type
PyObject* rms_norm(PyObject* const* a) {
  const Rows x(a[0], "input");
  const double eps = PyFloat_AsDouble(a[2]);
  if (eps == -1.0 && PyErr_Occurred()) throw Raised();
  if (!(eps >= 0)) refuse(PyExc_RuntimeError, "eps must not be negative, got %R", a[2]);
  const bool antithetic = truth(a[5]);
  const at::Device device = x.t.device();
  const int64_t format = whole(a[6]);
  at::Tensor in = aligned(x.t), residual, h, weight, noise;
  if (a[3] != Py_None) {
    if (!THPVariable_Check(a[3]) || THPVariable_Unpack(a[3]).sizes() != x.t.sizes()) refuse(PyExc_RuntimeError, "residual must have the input's shape");
    residual = aligned(of_type(a[3], "residual", x.t.scalar_type()));
    same_device(residual, device, "residual");
    h = empty(x.t.sizes(), x.t.scalar_type(), x.t);
  }
  if (a[1] != Py_None) {
    weight = aligned(of_type(a[1], "weight", at::kFloat));
    if (weight.dim() != 1 || weight.size(0) != x.cols) refuse(PyExc_RuntimeError, "weight must have shape (%lld,)", (long long)x.cols);
    same_device(weight, device, "weight");
  }
  int64_t members = 0;
  if (a[4] != Py_None) {
    noise = aligned(of_type(a[4], "noise", at::kFloat));
    if (noise.dim() != 2 || noise.size(0) == 0 || noise.size(1) != x.cols)
      refuse(PyExc_RuntimeError, "noise must have shape (members, %lld)", (long long)x.cols);
    members = noise.size(0);
    if (x.rows % members)
      refuse(PyExc_RuntimeError, "batch size %lld is not a multiple of directions %lld", (long long)x.rows, (long long)members);
    same_device(noise, device, "noise");
  }
  at::Tensor y, scales;
  if (format) {
    y = bytes(x.t, x.rows, pitch(x.cols, format));
    scales = bytes(x.t, x.rows, scale_pitch(x.cols));
  } else {
    y = empty(x.t.sizes(), x.t.scalar_type(), x.t);
  }
  const Launch launch(device);
  auto data = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
  run("nes_rms_norm_fwd", [&] {
    return nes_rms_norm_fwd(in.data_ptr(), data(residual), data(h), static_cast<const float*>(data(weight)), static_cast<const float*>(data(noise)),
                            y.data_ptr(), static_cast<uint8_t*>(data(scales)), x.rows, x.cols, members, antithetic, x.kind, int(format), float(eps),
                            launch.stream);
  });
  PyObject* first = format ? blocks_tuple(y, scales, x) : THPVariable_Wrap(y);
  if (!h.defined()) return first;
  return Py_BuildValue("(NN)", first, THPVariable_Wrap(h));
}

template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Raised&) {
  } catch (...) {
    torch::translate_exception_to_python(std::current_exception());      // torch.OutOfMemoryError and the like, as PyTorch's own calls raise
  }
  return nullptr;
}

template <PyObject* (*F)(PyObject* const*), int N>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N>)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method<blocks, 4>("blocks"), method<quantize, 2>("quantize"), method<elements, 4>("elements"), method<block_scales, 3>("block_scales"),
                         method<dequantize, 6>("dequantize"), method<linear, 12>("linear"), method<rms_norm, 7>("rms_norm"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "nesgpu_b200._host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
