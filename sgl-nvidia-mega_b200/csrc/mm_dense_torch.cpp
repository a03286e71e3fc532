// The dense 8-bit operators' calls on torch tensors: checks, outputs and workspace from
// torch's allocator, the tensors' device and its current stream, then one call of the C ABI
// (include/megamoe.h). Python's share of such a call (attribute lookups, ctypes, four
// torch.empty) took 14 to 24 us, several times the kernel of a decode step; here it is 4 to 9.
// megamoe/dense.py holds the documented functions.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <optional>
#include <string>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "megamoe.h"

namespace {

using at::ScalarType;
using at::Tensor;

// A type as Python names it.
std::string type_name(ScalarType t) {
  switch (t) {
    case ScalarType::BFloat16: return "bfloat16";
    case ScalarType::Half: return "float16";
    case ScalarType::Float: return "float32";
    case ScalarType::Double: return "float64";
    case ScalarType::Char: return "int8";
    case ScalarType::Byte: return "uint8";
    case ScalarType::Int: return "int32";
    case ScalarType::Long: return "int64";
    default: return c10::toString(t);
  }
}

int dtype_code(ScalarType t, const char *name) {
  switch (t) {
    case ScalarType::BFloat16: return MM_DTYPE_BF16;
    case ScalarType::Half: return MM_DTYPE_FP16;
    case ScalarType::Float: return MM_DTYPE_FP32;
    default: TORCH_CHECK_VALUE(false, name, ": bf16, fp16 or fp32, not ", type_name(t));
  }
}

std::string shape(const Tensor &t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}

// Argument i of a call, None and missing ones as null.
struct Args {
  PyObject *const *v;
  Py_ssize_t n;
  bool has(int i) const { return i < n && v[i] != Py_None; }
  const Tensor &tensor(int i, const char *name) const {
    TORCH_CHECK_TYPE(i < n && THPVariable_Check(v[i]), name, " must be a tensor");
    return THPVariable_Unpack(v[i]);
  }
  ScalarType dtype(int i, const char *name) const {
    TORCH_CHECK_TYPE(i < n && THPDtype_Check(v[i]), name, " must be a torch.dtype");
    return reinterpret_cast<THPDtype *>(v[i])->scalar_type;
  }
  bool truth(int i) const {
    const int t = PyObject_IsTrue(v[i]);
    if (t < 0) throw python_error();
    return t == 1;
  }
  double number(int i, const char *name) const {
    TORCH_CHECK_TYPE(i < n, name, " is missing");
    const double d = PyFloat_AsDouble(v[i]);
    if (d == -1.0 && PyErr_Occurred()) throw python_error();
    return d;
  }
};

at::Device cuda(const Tensor &t, const char *name) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA tensor");
  return t.device();
}

// Checks a tensor of contiguous rows ([rows, cols]; -1: any); its row stride.
int64_t row_stride(const Tensor &t, const char *name, at::Device device, ScalarType type, int64_t rows, int64_t cols) {
  TORCH_CHECK_VALUE(t.layout() == at::kStrided && t.dim() == 2 && t.scalar_type() == type && t.device() == device &&
                        (rows < 0 || t.size(0) == rows) && (cols < 0 || t.size(1) == cols),
                    name, ": expected a ", type_name(type), " [", rows < 0 ? std::string("T") : std::to_string(rows), ", ",
                    cols < 0 ? std::string("K") : std::to_string(cols), "] tensor on ", device, ", got ", shape(t), " ",
                    type_name(t.scalar_type()), " on ", t.device());
  TORCH_CHECK_VALUE(t.size(1) <= 1 || t.stride(1) == 1, name, ": rows must be contiguous (stride 1 along the last dimension)");
  TORCH_CHECK_VALUE(t.size(0) < (int64_t(1) << 31) && t.size(1) < (int64_t(1) << 31), name, ": sizes below 2^31, got ", shape(t));
  return t.size(0) > 1 ? t.stride(0) : std::max<int64_t>(t.size(1), 1);
}

// The same of int8 rows, which start on 16-byte boundaries.
int64_t code_stride(const Tensor &t, const char *name, at::Device device, int64_t rows, int64_t cols) {
  int64_t ld = row_stride(t, name, device, ScalarType::Char, rows, cols);
  if (t.size(0) <= 1) ld = (ld + 15) / 16 * 16;  // one row, or none, needs no stride of its own
  TORCH_CHECK_VALUE(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && ld % 16 == 0, name,
                    ": int8 rows must start on 16-byte boundaries (row stride ", ld,
                    "); rms_norm and quantize_int8 return them so, weights are laid out once with a padded row stride");
  return ld;
}

// Checks n contiguous values ([n] or [n, 1]); their address.
void *values(const Tensor &t, const char *name, int64_t n, at::Device device, ScalarType type) {
  TORCH_CHECK_VALUE(t.layout() == at::kStrided && t.scalar_type() == type && t.numel() == n && t.dim() >= 1 && t.size(0) == n &&
                        t.device() == device && t.is_contiguous(),
                    name, ": expected ", n, " contiguous ", type_name(type), " values on ", device, ", got ", shape(t), " ",
                    type_name(t.scalar_type()), " on ", t.device());
  return t.data_ptr();
}

Tensor empty(at::IntArrayRef sizes, ScalarType type, at::Device device) {
  return Tensor(at::detail::empty_cuda(sizes, type, device, std::nullopt));
}

// A call's outputs. Small ones share one allocation (an allocation costs about 0.5 us of host
// time, a tensor on a part of one 0.1): at most kTogether bytes, so that an output which
// outlives the others holds little beside itself.
constexpr int64_t kTogether = int64_t(1) << 20;
class Outputs {
 public:
  Outputs(int64_t bytes, at::Device device) : device_(device) {
    if (bytes <= kTogether) block_ = empty({bytes}, ScalarType::Byte, device);
  }
  // What a tensor takes of a block.
  static int64_t room(int64_t values, int64_t size) { return (values * size + 511) / 512 * 512; }
  Tensor take(at::IntArrayRef sizes, ScalarType type) {
    if (!block_.defined()) return empty(sizes, type, device_);
    int64_t n = 1;
    for (const int64_t s : sizes) n *= s;
    const int64_t size = static_cast<int64_t>(c10::elementSize(type));
    auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(block_.storage()), block_.key_set(), c10::scalarTypeToTypeMeta(type));
    impl->set_sizes_contiguous(sizes);
    impl->set_storage_offset(at_ / size);
    at_ += room(n, size);
    return Tensor(std::move(impl));
  }

 private:
  at::Device device_;
  Tensor block_;
  int64_t at_ = 0;
};

// int8 [rows, cols] whose rows start on 16-byte boundaries.
int64_t code_ld(int64_t cols) { return (cols + 15) / 16 * 16; }
Tensor code_rows(Outputs &out, int64_t rows, int64_t cols) {
  Tensor t = out.take({rows, code_ld(cols)}, ScalarType::Char);
  return code_ld(cols) == cols ? t : t.narrow(1, 0, cols);
}

void check(int rc, const char *what) {
  if (rc == MM_OK) return;
  TORCH_CHECK_VALUE(rc != MM_ERR_INVALID && rc != MM_ERR_UNSUPPORTED, what, ": ", mm_last_error());
  TORCH_CHECK(false, what, ": ", mm_last_error(), " (status ", rc, ")");
}

PyObject *wrap(Tensor &t) {
  if (t.defined()) return THPVariable_Wrap(std::move(t));
  Py_RETURN_NONE;
}

// (x, gamma, eps, residual, quant, with_norm, out, residual_out) -> (norm, codes, scales, residual)
PyObject *rms_norm(PyObject *, PyObject *const *v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Args a{v, n};
  const Tensor &x = a.tensor(0, "x"), &gamma = a.tensor(1, "gamma");
  const at::Device device = cuda(x, "x");
  const ScalarType type = x.scalar_type();
  mm_norm_args m = {};
  m.dtype = dtype_code(type, "x");
  m.ld_x = row_stride(x, "x", device, type, -1, -1);
  const int64_t tokens = x.size(0), hidden = x.size(1);
  m.quant = MM_QUANT_NONE;
  if (a.has(4)) {
    const char *q = PyUnicode_Check(v[4]) ? PyUnicode_AsUTF8(v[4]) : nullptr;
    if (q && std::strcmp(q, "mxfp8") == 0) m.quant = MM_QUANT_MXFP8;
    else if (q && std::strcmp(q, "int8") == 0) m.quant = MM_QUANT_INT8;
    else TORCH_CHECK_VALUE(false, "quant: None, 'mxfp8' or 'int8'");
  }
  TORCH_CHECK_VALUE(hidden >= 1 && (m.quant != MM_QUANT_MXFP8 || hidden % 32 == 0), "rows of ", hidden,
                    " values (mxfp8: a multiple of 32)");
  TORCH_CHECK_VALUE(gamma.scalar_type() == type || gamma.scalar_type() == ScalarType::Float, "gamma: ", type_name(type), " or fp32, not ",
                    type_name(gamma.scalar_type()));
  m.gamma_dtype = dtype_code(gamma.scalar_type(), "gamma");
  m.gamma = values(gamma, "gamma", hidden, device, gamma.scalar_type());
  m.eps = static_cast<float>(a.number(2, "eps"));
  m.x = x.data_ptr();
  m.tokens = static_cast<int32_t>(tokens);
  m.hidden = static_cast<int32_t>(hidden);
  const bool has_with = a.has(5), with = has_with && a.truth(5);
  const bool wants_norm = m.quant == MM_QUANT_NONE || with || a.has(6);
  TORCH_CHECK_VALUE(!(wants_norm && has_with && !with), "with_norm=False needs quant and no out");
  TORCH_CHECK_VALUE(a.has(3) || !a.has(7), "residual_out needs residual");
  const c10::cuda::CUDAGuard guard(device);
  Tensor norm, codes, scales, residual;
  const int64_t es = static_cast<int64_t>(x.element_size()), n_all = tokens * hidden;
  Outputs outputs((a.has(3) && !a.has(7) ? Outputs::room(n_all, es) : 0) + (wants_norm && !a.has(6) ? Outputs::room(n_all, es) : 0) +
                      (m.quant ? Outputs::room(tokens * code_ld(hidden), 1) : 0) +
                      (m.quant == MM_QUANT_MXFP8 ? Outputs::room(n_all / 32, 1) : m.quant ? Outputs::room(tokens, 4) : 0),
                  device);
  if (a.has(3)) {
    const Tensor &r = a.tensor(3, "residual");
    m.ld_residual = row_stride(r, "residual", device, type, tokens, hidden);
    m.residual = r.data_ptr();
    residual = a.has(7) ? a.tensor(7, "residual_out") : outputs.take({tokens, hidden}, type);
    m.ld_residual_out = row_stride(residual, "residual_out", device, type, tokens, hidden);
    m.residual_out = residual.data_ptr();
  }
  if (wants_norm) {
    norm = a.has(6) ? a.tensor(6, "out") : outputs.take({tokens, hidden}, type);
    m.ld_norm = row_stride(norm, "out", device, type, tokens, hidden);
    m.norm_out = norm.data_ptr();
  }
  if (m.quant == MM_QUANT_MXFP8) {
    codes = outputs.take({tokens, hidden}, ScalarType::Float8_e4m3fn);
    scales = outputs.take({tokens, hidden / 32}, ScalarType::Float8_e8m0fnu);
  } else if (m.quant == MM_QUANT_INT8) {
    codes = code_rows(outputs, tokens, hidden);
    scales = outputs.take({tokens}, ScalarType::Float);
  }
  if (m.quant) {
    m.codes = codes.data_ptr();
    m.scales = scales.data_ptr();
    m.ld_codes = code_ld(hidden);
  }
  check(mm_rms_norm(&m, c10::cuda::getCurrentCUDAStream(device.index()).stream()), "rms_norm");
  PyObject *out[4] = {wrap(norm), wrap(codes), wrap(scales), wrap(residual)};
  PyObject *t = PyTuple_New(4);
  for (int i = 0; i < 4; ++i) PyTuple_SET_ITEM(t, i, out[i]);
  return t;
  END_HANDLE_TH_ERRORS
}

// (x) -> (codes, scales)
PyObject *quantize_int8(PyObject *, PyObject *const *v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Args a{v, n};
  const Tensor &x = a.tensor(0, "x");
  const at::Device device = cuda(x, "x");
  const int dtype = dtype_code(x.scalar_type(), "x");
  const int64_t ld = row_stride(x, "x", device, x.scalar_type(), -1, -1), tokens = x.size(0), hidden = x.size(1);
  TORCH_CHECK_VALUE(hidden >= 1, "x: rows of at least one value, got ", shape(x));
  const c10::cuda::CUDAGuard guard(device);
  Outputs outputs(Outputs::room(tokens * code_ld(hidden), 1) + Outputs::room(tokens, 4), device);
  Tensor codes = code_rows(outputs, tokens, hidden), scales = outputs.take({tokens}, ScalarType::Float);
  check(mm_quantize_int8(x.data_ptr(), ld, dtype, static_cast<int8_t *>(codes.data_ptr()), code_ld(hidden),
                         static_cast<float *>(scales.data_ptr()), static_cast<int32_t>(tokens), static_cast<int32_t>(hidden),
                         c10::cuda::getCurrentCUDAStream(device.index()).stream()),
        "quantize_int8");
  PyObject *t = PyTuple_New(2);
  PyTuple_SET_ITEM(t, 0, wrap(codes));
  PyTuple_SET_ITEM(t, 1, wrap(scales));
  return t;
  END_HANDLE_TH_ERRORS
}

constexpr int64_t kMostDepth = (int64_t(1) << 17) - 1;

// (x, x_scale, weight, weight_scale, bias, out_dtype, out) -> out
PyObject *int8_linear(PyObject *, PyObject *const *v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Args a{v, n};
  const Tensor &x = a.tensor(0, "x"), &xs = a.tensor(1, "x_scale"), &w = a.tensor(2, "weight"), &ws = a.tensor(3, "weight_scale");
  const at::Device device = cuda(x, "x");
  const int64_t ld_x = code_stride(x, "x", device, -1, -1), tokens = x.size(0), depth = x.size(1);
  const int64_t ld_w = code_stride(w, "weight", device, -1, depth), features = w.size(0);
  const ScalarType type = a.dtype(5, "out_dtype");
  const int dtype = dtype_code(type, "out_dtype");
  TORCH_CHECK_VALUE(features >= 1 && depth >= 1 && depth <= kMostDepth, "weight: ", features, " features of depth ", depth,
                    " (1..", kMostDepth, ")");
  const float *px = static_cast<float *>(values(xs, "x_scale", tokens, device, ScalarType::Float));
  const float *pw = static_cast<float *>(values(ws, "weight_scale", features, device, ScalarType::Float));
  const float *pb = a.has(4) ? static_cast<float *>(values(a.tensor(4, "bias"), "bias", features, device, ScalarType::Float)) : nullptr;
  const c10::cuda::CUDAGuard guard(device);
  Tensor out = a.has(6) ? a.tensor(6, "out") : empty({tokens, features}, type, device);
  const int64_t ld_out = row_stride(out, "out", device, type, tokens, features);
  check(mm_int8_linear(static_cast<int8_t *>(x.data_ptr()), ld_x, px, static_cast<int8_t *>(w.data_ptr()), ld_w, pw, pb,
                       out.data_ptr(), ld_out, dtype, static_cast<int32_t>(tokens), static_cast<int32_t>(features),
                       static_cast<int32_t>(depth), c10::cuda::getCurrentCUDAStream(device.index()).stream()),
        "int8_linear");
  return wrap(out);
  END_HANDLE_TH_ERRORS
}

// (x, x_scale, w13, w13_scale, w2, w2_scale, clamp, out_dtype, out) -> out
PyObject *int8_ffn(PyObject *, PyObject *const *v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Args a{v, n};
  const Tensor &x = a.tensor(0, "x"), &w13 = a.tensor(2, "w13"), &w2 = a.tensor(4, "w2");
  const at::Device device = cuda(x, "x");
  mm_int8_ffn_args m = {};
  m.ld_x = code_stride(x, "x", device, -1, -1);
  const int64_t tokens = x.size(0), hidden = x.size(1);
  m.ld_w13 = code_stride(w13, "w13", device, -1, hidden);
  const int64_t inter = w13.size(0) / 2;
  TORCH_CHECK_VALUE(w13.size(0) == 2 * inter && inter >= 1 && inter <= kMostDepth && hidden >= 1 && hidden <= kMostDepth,
                    "w13: expected int8 [2I, H] with I and H in 1..", kMostDepth, ", got ", shape(w13));
  m.ld_w2 = code_stride(w2, "w2", device, hidden, inter);
  if (a.has(6)) {
    m.clamp = static_cast<float>(a.number(6, "clamp"));
    TORCH_CHECK_VALUE(m.clamp > 0.0f && std::isfinite(m.clamp), "clamp: a positive number or None, not ", m.clamp);
  }
  const ScalarType type = a.dtype(7, "out_dtype");
  m.out_dtype = dtype_code(type, "out_dtype");
  m.x_scale = static_cast<float *>(values(a.tensor(1, "x_scale"), "x_scale", tokens, device, ScalarType::Float));
  m.w13_scale = static_cast<float *>(values(a.tensor(3, "w13_scale"), "w13_scale", 2 * inter, device, ScalarType::Float));
  m.w2_scale = static_cast<float *>(values(a.tensor(5, "w2_scale"), "w2_scale", hidden, device, ScalarType::Float));
  const c10::cuda::CUDAGuard guard(device);
  Tensor out = a.has(8) ? a.tensor(8, "out") : empty({tokens, hidden}, type, device);
  m.ld_out = row_stride(out, "out", device, type, tokens, hidden);
  m.tokens = static_cast<int32_t>(tokens);
  m.hidden = static_cast<int32_t>(hidden);
  m.inter = static_cast<int32_t>(inter);
  m.workspace_bytes = mm_int8_ffn_workspace(m.tokens, m.inter);
  const Tensor space = empty({m.workspace_bytes}, ScalarType::Byte, device);
  m.x = static_cast<int8_t *>(x.data_ptr());
  m.w13 = static_cast<int8_t *>(w13.data_ptr());
  m.w2 = static_cast<int8_t *>(w2.data_ptr());
  m.out = out.data_ptr();
  m.workspace = space.data_ptr();
  check(mm_int8_ffn(&m, c10::cuda::getCurrentCUDAStream(device.index()).stream()), "int8_ffn");
  return wrap(out);
  END_HANDLE_TH_ERRORS
}

#define FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(rms_norm), FAST(quantize_int8), FAST(int8_linear), FAST(int8_ffn), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_dense", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__dense() { return PyModule_Create(&module); }
