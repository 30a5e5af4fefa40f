// CPython module `_tk8s_layer`: the 8-bit layer (kernels.h) on torch tensors. It checks arguments,
// allocates what a call returns and its workspace, and launches on the current stream of the
// tensors' device; tritonk8ssupervisor_amd/ops/fp8.py documents the calls and names the results.
// Native because a call on one token is a few microseconds of GPU time: the same work in Python
// took 10 to 20.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/EmptyTensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/HIPContextLight.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <optional>
#include <string>

#include "tk8s/common.h"
#include "tk8s/kernels.h"

namespace {

using at::ScalarType;
using at::Tensor;
using tk8s::LayerType;

constexpr int64_t kBlock = 128;

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
int64_t blocks_of(int64_t n) { return (n + kBlock - 1) / kBlock; }

template <class... A> [[noreturn]] void wrong_value(const A&... a) { throw std::invalid_argument(c10::str(a...)); }
template <class... A> [[noreturn]] void wrong_type(const A&... a) { throw torch::TypeError(c10::str(a...)); }

std::string shape_of(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + (t.dim() == 1 ? ",)" : ")");
}

const Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) wrong_type(name, " must be a tensor, not ", Py_TYPE(o)->tp_name);
  const Tensor& t = THPVariable_Unpack(o);
  if (t.is_neg()) wrong_value(name, " is negated only when it is read: give its resolve_neg()");  // its memory has the other sign
  if (t._is_zerotensor()) wrong_value(name, " is zeros without memory: give a copy of it");
  return t;
}

const Tensor& matrix(PyObject* o, const char* name) {
  const Tensor& t = tensor(o, name);
  if (t.dim() != 2) wrong_value(name, " must have 2 dimensions, not ", t.dim());
  if (t.layout() != at::kStrided) wrong_value(name, " must be a dense tensor");
  if (t.size(1) > 1 && t.stride(1) != 1)
    wrong_value("the rows of ", name, " must be contiguous (stride ", t.stride(1), " between columns)");
  return t;
}

std::optional<LayerType> layer_type(ScalarType t) {
  switch (t) {
    case ScalarType::Float: return LayerType::kF32;
    case ScalarType::BFloat16: return LayerType::kBF16;
    case ScalarType::Half: return LayerType::kF16;
    default: return std::nullopt;
  }
}

LayerType typed(const Tensor& t, const char* name) {
  const auto type = layer_type(t.scalar_type());
  if (!type) wrong_value(name, " must be float32, bfloat16 or float16, not ", t.scalar_type());
  return *type;
}

const Tensor& like(PyObject* o, const char* name, const Tensor& x, const char* of) {
  const Tensor& t = matrix(o, name);
  if (t.scalar_type() != x.scalar_type() || t.sizes() != x.sizes())
    wrong_value(name, " must be ", shape_of(x), " ", x.scalar_type(), " like ", of, ", not ", shape_of(t), " ", t.scalar_type());
  return t;
}

const Tensor& vector(PyObject* o, const char* name, int64_t size, ScalarType type) {
  const Tensor& t = tensor(o, name);
  if (t.dim() != 1 || t.size(0) != size || (t.scalar_type() != type && t.scalar_type() != ScalarType::Float) ||
      (size > 1 && t.stride(0) != 1))
    wrong_value(name, " must be ", size, " contiguous values of ", type, type == ScalarType::Float ? "" : " or Float", ", not ",
                shape_of(t), " ", t.scalar_type());
  return t;
}

// The tensors' one GPU, current while this lives, and its current stream.
class Device {
 public:
  Device(std::initializer_list<const Tensor*> tensors) : device_((*tensors.begin())->device()) {
    if (!device_.is_cuda()) wrong_value("the 8-bit layer runs on a GPU; the tensors are on ", device_.str());
    for (const Tensor* t : tensors)
      if (t && t->device() != device_) wrong_value("all tensors must be on one GPU, not on ", device_.str(), " and ", t->device().str());
    int now = -1;
    TK8S_HIP_CHECK(hipGetDevice(&now));
    if (now != device_.index()) guard_.emplace(device_);
    stream_ = c10::hip::getCurrentHIPStream(device_.index()).stream();
  }
  hipStream_t stream() const { return stream_; }
  // A tensor with memory of its own, from torch's allocator for the device that is current here. (The general
  // way looks for the device again: 0.2 us for each of the four results of a norm of one token, which takes 5.)
  Tensor empty(at::IntArrayRef sizes, ScalarType type) const {
    return at::detail::empty_generic(sizes, at::cuda::getCUDADeviceAllocator(), c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt);
  }

 private:
  c10::Device device_;
  std::optional<c10::DeviceGuard> guard_;
  hipStream_t stream_ = nullptr;
};

// Room for rows x cols values in 8 bits and for the scales of scale_rows rows (or tiles), block by block.
// Rows start on 16-byte boundaries; wide ones on 128-byte ones, so that a tile's part of a row is
// whole lines (the transposed rounding of 10007 x 8192: 88 us at a pitch of 10016 bytes, 61 at 10112).
struct Packed {
  Tensor values, scales;
  tk8s::Fp8Matrix at{};
};

int64_t pitch_of(int64_t cols) { return up(cols, cols > 512 ? 128 : 16); }
Packed packed(const Device& dev, int64_t rows, int64_t cols, int64_t scale_rows) {
  const int64_t ld = pitch_of(cols), lds = up(scale_rows, 16), blocks = blocks_of(cols);
  Packed p{dev.empty({rows, ld}, ScalarType::Float8_e4m3fn), dev.empty({blocks, lds}, ScalarType::Float8_e8m0fnu)};
  p.at = {static_cast<uint8_t*>(p.values.data_ptr()), static_cast<size_t>(ld), static_cast<uint8_t*>(p.scales.data_ptr()),
          static_cast<size_t>(lds)};
  p.values.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef({rows, cols}), at::IntArrayRef({ld, 1}));
  p.scales.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef({scale_rows, blocks}), at::IntArrayRef({1, lds}));
  return p;
}

template <class T = void> T* data(const Tensor* t) { return t ? static_cast<T*>(t->data_ptr()) : nullptr; }
size_t pitch(const Tensor* t) { return t ? static_cast<size_t>(t->stride(0)) : 0; }

PyObject* tuple_of(std::initializer_list<const Tensor*> tensors) {
  PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(tensors.size()));
  Py_ssize_t i = 0;
  for (const Tensor* t : tensors) {
    if (!t) Py_INCREF(Py_None);
    PyTuple_SET_ITEM(out, i++, t ? THPVariable_Wrap(*t) : Py_None);
  }
  return out;
}

void expect(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) wrong_type("expected ", want, " arguments, not ", got);
}

// (x, layout: 0 rows, 1 columns, 2 both, 3 tiles) -> (values, scales[, values of the columns, scales])
PyObject* quantize(PyObject* const* args, Py_ssize_t nargs) {
  expect(nargs, 2);
  const Tensor& x = matrix(args[0], "x");
  const LayerType type = typed(x, "x");
  const long layout = PyLong_AsLong(args[1]);
  const int64_t rows = x.size(0), cols = x.size(1);
  const Device dev({&x});
  tk8s::QuantizeArgs a{x.data_ptr(), pitch(&x), static_cast<size_t>(rows), static_cast<size_t>(cols), {}, {}, {}};
  Packed p, q;
  if (layout == 0 || layout == 2) p = packed(dev, rows, cols, rows), a.rows_out = p.at;
  if (layout == 1 || layout == 2) q = packed(dev, cols, rows, cols), a.cols_out = q.at;
  if (layout == 3) p = packed(dev, rows, cols, blocks_of(rows)), a.tiles_out = p.at;
  tk8s::fp8_quantize(a, type, dev.stream());
  if (layout == 2) return tuple_of({&p.values, &p.scales, &q.values, &q.scales});
  return layout == 1 ? tuple_of({&q.values, &q.scales}) : tuple_of({&p.values, &p.scales});
}

// (x, weight, residual or None, eps, quantized, normed) -> (h, values, scales, y, rstd)
PyObject* rms_norm(PyObject* const* args, Py_ssize_t nargs) {
  expect(nargs, 6);
  const Tensor& x = matrix(args[0], "x");
  const LayerType type = typed(x, "x");
  const int64_t rows = x.size(0), cols = x.size(1);
  const Tensor* residual = args[2] == Py_None ? nullptr : &like(args[2], "residual", x, "x");
  const Tensor& weight = vector(args[1], "weight", cols, x.scalar_type());
  const double eps = PyFloat_AsDouble(args[3]);
  if (eps == -1.0 && PyErr_Occurred()) return nullptr;
  if (!(eps >= 0.0)) wrong_value("eps must not be negative, but is ", eps);
  const bool quantized = args[4] == Py_True, normed = args[5] == Py_True;
  const Device dev({&x, &weight, residual});
  Tensor h = residual ? dev.empty({rows, cols}, x.scalar_type()) : x, y;
  Packed p;
  if (quantized) p = packed(dev, rows, cols, rows);
  if (normed) y = dev.empty({rows, cols}, x.scalar_type());
  Tensor rstd = dev.empty({rows}, ScalarType::Float);
  const size_t ld = static_cast<size_t>(cols);
  tk8s::rms_norm_fp8({x.data_ptr(), pitch(&x), data<const void>(residual), pitch(residual), weight.data_ptr(),
                      residual ? h.data_ptr() : nullptr, ld, p.at.values, p.at.ld, p.at.scales, p.at.ld_scales,
                      normed ? y.data_ptr() : nullptr, ld, data<float>(&rstd), static_cast<size_t>(rows), ld, eps},
                     type, *layer_type(weight.scalar_type()), dev.stream());
  return tuple_of({&h, quantized ? &p.values : nullptr, quantized ? &p.scales : nullptr, normed ? &y : nullptr, &rstd});
}

// (dy, h, weight, rstd, dh or None) -> (dx, dweight)
PyObject* rms_norm_backward(PyObject* const* args, Py_ssize_t nargs) {
  expect(nargs, 5);
  const Tensor& h = matrix(args[1], "h");
  const LayerType type = typed(h, "h");
  const int64_t rows = h.size(0), cols = h.size(1);
  const Tensor& dy = like(args[0], "dy", h, "h");
  const Tensor* dh = args[4] == Py_None ? nullptr : &like(args[4], "dh", h, "h");
  const Tensor& weight = vector(args[2], "weight", cols, h.scalar_type());
  const Tensor& rstd = vector(args[3], "rstd", rows, ScalarType::Float);
  const Device dev({&h, &dy, &weight, &rstd, dh});
  Tensor dx = dev.empty({rows, cols}, h.scalar_type());
  if (rows == 0 || cols == 0) {
    Tensor none = at::zeros({cols}, h.options().dtype(ScalarType::Float));
    return tuple_of({&dx, &none});
  }
  Tensor dw = dev.empty({cols}, ScalarType::Float), work;
  const size_t n = static_cast<size_t>(rows), ld = static_cast<size_t>(cols);
  const size_t work_bytes = tk8s::rms_norm_backward_workspace(n, ld);
  if (work_bytes) work = dev.empty({static_cast<int64_t>(work_bytes)}, ScalarType::Byte);
  tk8s::rms_norm_backward({dy.data_ptr(), pitch(&dy), h.data_ptr(), pitch(&h), weight.data_ptr(), data<const float>(&rstd),
                           data<const void>(dh), pitch(dh), dx.data_ptr(), ld, data<float>(&dw),
                           work_bytes ? reinterpret_cast<float*>(work.data_ptr()) : nullptr, n, ld},
                          type, *layer_type(weight.scalar_type()), dev.stream());
  return tuple_of({&dx, &dw});
}

// A product's operand: values and scales, with the layout the kernels take.
struct Operand {
  const Tensor* values;
  Tensor scales;
  bool by_tile = false;
  tk8s::Fp8Matrix at{};
};

Operand operand(PyObject* o, const char* name, bool tiles) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 2)
    wrong_type(name, " must be a (values, scales) pair, as quantize() returns it");
  const std::string vname = std::string(name) + "'s values", sname = std::string(name) + "'s scales";
  Operand p;
  const Tensor& values = matrix(PyTuple_GET_ITEM(o, 0), vname.c_str());
  const Tensor& scales = tensor(PyTuple_GET_ITEM(o, 1), sname.c_str());
  if (values.scalar_type() != ScalarType::Float8_e4m3fn) wrong_value(vname, " must be float8_e4m3fn, not ", values.scalar_type());
  if (scales.scalar_type() != ScalarType::Float8_e8m0fnu) wrong_value(sname, " must be float8_e8m0fnu, not ", scales.scalar_type());
  const int64_t rows = values.size(0), cols = values.size(1), blocks = blocks_of(cols);
  auto shaped = [&](int64_t r) { return scales.dim() == 2 && scales.size(0) == r && scales.size(1) == blocks; };
  p.by_tile = tiles && shaped(blocks_of(rows)) && blocks_of(rows) != rows;
  if (!p.by_tile && !shaped(rows))
    wrong_value(sname, " must be (", rows, ", ", blocks, ")", tiles ? " or a scale for each 128 x 128" : "", ", not ", shape_of(scales));
  const int64_t ld = rows > 1 && cols ? values.stride(0) : up(cols, 16);
  if (ld % 16 || reinterpret_cast<uintptr_t>(values.data_ptr()) % 16)
    wrong_value("the rows of ", vname, " must start on 16-byte boundaries, as quantize() lays them out");
  p.values = &values;
  p.scales = scales;
  p.at = {static_cast<uint8_t*>(values.data_ptr()), static_cast<size_t>(ld), nullptr, 0};
  return p;
}

// The kernels read the scales of one block four rows at a time: scales that lie otherwise are copied.
void lay_out_scales(Operand& p, const Device& dev) {
  const int64_t n = p.scales.size(0), blocks = p.scales.size(1);
  int64_t lds = blocks > 1 ? p.scales.stride(1) : up(n, 16);
  const int64_t room = static_cast<int64_t>(p.scales.storage().nbytes()) - p.scales.storage_offset();
  if (p.scales.numel() && ((n > 1 && p.scales.stride(0) != 1) || lds % 4 || reinterpret_cast<uintptr_t>(p.scales.data_ptr()) % 4 ||
                           (blocks - 1) * lds + up(n, 4) > room)) {
    lds = up(n, 16);
    Tensor laid = dev.empty({blocks, lds}, ScalarType::Float8_e8m0fnu);
    laid.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef({n, blocks}), at::IntArrayRef({1, lds}));
    p.scales = laid.copy_(p.scales);
  }
  p.at.scales = static_cast<uint8_t*>(p.scales.data_ptr());
  p.at.ld_scales = static_cast<size_t>(lds);
}

// (a, b, dtype, out or None) -> c
PyObject* matmul(PyObject* const* args, Py_ssize_t nargs) {
  expect(nargs, 4);
  Operand a = operand(args[0], "a", false), b = operand(args[1], "b", true);
  const int64_t m = a.values->size(0), k = a.values->size(1), n = b.values->size(0);
  if (b.values->size(1) != k) wrong_value("a and b must have as many columns, not ", k, " and ", b.values->size(1));
  const Tensor* out = nullptr;
  if (args[3] != Py_None) {
    out = &matrix(args[3], "out");
    if (out->size(0) > 1 && out->stride(0) < out->size(1)) wrong_value("the rows of out overlap: it cannot be written to");
    if (out->size(0) != m || out->size(1) != n) wrong_value("out must be (", m, ", ", n, "), not ", shape_of(*out));
    if (out->requires_grad() && at::GradMode::is_enabled())
      wrong_value("out requires grad, and nothing is recorded for autograd: write to it under torch.no_grad()");
  }
  if (!out && !THPDtype_Check(args[2])) wrong_type("dtype must be a torch.dtype, not ", Py_TYPE(args[2])->tp_name);
  const ScalarType st = out ? out->scalar_type() : reinterpret_cast<THPDtype*>(args[2])->scalar_type;
  const auto type = layer_type(st);
  if (!type) wrong_value("the result's dtype must be float32, bfloat16 or float16, not ", st);
  const Device dev({a.values, &a.scales, b.values, &b.scales, out});
  lay_out_scales(a, dev);
  lay_out_scales(b, dev);
  Tensor c = out ? *out : dev.empty({m, n}, st);
  tk8s::fp8_matmul({a.at, b.at, b.by_tile, c.data_ptr(), static_cast<size_t>(m > 1 ? c.stride(0) : n), static_cast<size_t>(m),
                    static_cast<size_t>(n), static_cast<size_t>(k)},
                   *type, dev.stream());
  if (out && !out->is_inference()) out->unsafeGetTensorImpl()->bump_version();  // autograd may have kept what it held
  return THPVariable_Wrap(c);
}

// torch's errors as torch raises them; std::invalid_argument is ValueError, as in the other modules.
template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  try {
    return F(args, nargs);
  } catch (const std::invalid_argument& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"quantize", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(entry<quantize>)), METH_FASTCALL, nullptr},
    {"rms_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(entry<rms_norm>)), METH_FASTCALL, nullptr},
    {"rms_norm_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(entry<rms_norm_backward>)), METH_FASTCALL, nullptr},
    {"matmul", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(entry<matmul>)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tk8s_layer", "the 8-bit layer on torch tensors", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tk8s_layer() { return PyModule_Create(&module); }
