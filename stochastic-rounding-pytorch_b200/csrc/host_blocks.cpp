// _srs_blocks: tensor front end of the FP8 block entry points (a CPython module).
//
// quantize, matmul and linear check their tensors, allocate results and enqueue on
// the current stream of the tensors' device: what a Python wrapper would do at 20 us a
// call, for kernels of 3 to 20 us.  The entry points are the C ABI's, given by
// address (bind), so that the kernels stay in libsrs_b200.so.  A function returns the
// negative status of an entry point as an int; the caller turns it into the error.
#include <Python.h>

#include <cstdint>
#include <string>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "srs_b200.h"

namespace {

constexpr int64_t kBlock = 128;

decltype(&srs_quantize_blocks) g_quantize = nullptr;
decltype(&srs_matmul_blocks) g_matmul = nullptr;
decltype(&srs_copy_rows) g_copy_rows = nullptr;
decltype(&srs_linear_blocks) g_linear = nullptr;
decltype(&srs_linear_workspace) g_linear_workspace = nullptr;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int source_format(const at::Tensor& x, const char* what) {
  switch (x.scalar_type()) {
    case at::kFloat: return SRS_FMT_F32;
    case at::kBFloat16: return SRS_FMT_BF16;
    case at::kHalf: return SRS_FMT_F16;
    default:
      TORCH_CHECK_TYPE(false, what, " takes FP32, BF16 or FP16, got ", x.scalar_type());
  }
}

at::ScalarType result_type(int format) {
  return format == SRS_FMT_F32 ? at::kFloat : format == SRS_FMT_BF16 ? at::kBFloat16 : at::kHalf;
}

struct Blocks {
  at::Tensor data, scale;
};

Blocks empty_blocks(int64_t rows, int64_t cols, int format, bool square, const at::Tensor& like) {
  // Row pitches of 16 bytes' multiples, as the products' copies need them.
  const int64_t pitch = ceil_div(cols, 16) * 16;
  Blocks b;
  b.data = at::empty({rows, pitch}, like.options().dtype(format == SRS_FMT_E4M3
                                                             ? at::kFloat8_e4m3fn
                                                             : at::kFloat8_e5m2));
  if (pitch != cols) b.data = b.data.narrow(1, 0, cols);
  b.scale = at::empty({square ? ceil_div(rows, kBlock) : rows, ceil_div(cols, kBlock)},
                      like.options().dtype(at::kFloat8_e8m0fnu));
  return b;
}

void* address(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
int64_t pitch(const at::Tensor& t) { return t.defined() ? t.stride(0) : 0; }

// orientation: 1 rows, 2 columns, 3 both
int quantize(const at::Tensor& x, int format, int rule, bool square, uint32_t seed,
             uint32_t offset, int orientation, Blocks* straight, Blocks* turned) {
  const int x_format = source_format(x, "quantize_blocks");
  TORCH_CHECK_VALUE(x.dim() == 2, "quantize_blocks needs a matrix, got shape ", x.sizes());
  const at::Tensor src = x.stride(1) != 1 && x.size(1) > 1 ? x.contiguous() : x;
  const int64_t rows = x.size(0), cols = x.size(1);
  if (orientation & 1) *straight = empty_blocks(rows, cols, format, square, x);
  if (orientation & 2) *turned = empty_blocks(cols, rows, format, square, x);
  if (x.numel() == 0) return SRS_OK;
  return g_quantize(src.data_ptr(), x_format, rows, cols, src.stride(0), format, rule,
                    square ? 1 : 0, seed, offset, address(straight->data), pitch(straight->data),
                    address(straight->scale), pitch(straight->scale), address(turned->data),
                    pitch(turned->data), address(turned->scale), pitch(turned->scale),
                    c10::cuda::getCurrentCUDAStream(x.device().index()).stream());
}

// The operand of a BlockTensor; data laid out otherwise than the products' copies need
// (16-byte rows) are copied once, `b` keeps the copy alive.
int operand(const char* name, Blocks* b, srs_blocks* out) {
  at::Tensor &data = b->data, &scale = b->scale;
  const bool e4m3 = data.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK_TYPE(e4m3 || data.scalar_type() == at::kFloat8_e5m2, name,
                   ": block data are float8_e4m3fn or float8_e5m2, got ", data.scalar_type());
  TORCH_CHECK_TYPE(scale.scalar_type() == at::kFloat8_e8m0fnu, name,
                   ": block scales are float8_e8m0fnu, got ", scale.scalar_type());
  TORCH_CHECK_VALUE(data.dim() == 2 && scale.dim() == 2, name,
                    ": data and scale must be matrices");
  TORCH_CHECK_VALUE(data.device() == scale.device(), name,
                    ": data and scale must be on the same CUDA device");
  const int64_t rows = data.size(0), cols = data.size(1), blocks = ceil_div(cols, kBlock);
  const int64_t high = scale.size(0);
  TORCH_CHECK_VALUE(scale.size(1) == blocks && (high == rows || high == ceil_div(rows, kBlock)),
                    name, ": scale of shape ", scale.sizes(), " does not fit data of shape ",
                    data.sizes());
  if (data.numel() != 0) {
    if (data.stride(1) != 1 && cols > 1) data = data.contiguous();
    if (data.stride(0) % 16 != 0 || reinterpret_cast<uintptr_t>(data.data_ptr()) % 16 != 0 ||
        data.stride(0) < cols) {
      at::Tensor copy = at::empty({rows, ceil_div(cols, 16) * 16}, data.options());
      if (int rc = g_copy_rows(data.data_ptr(), data.stride(0), rows, cols, copy.data_ptr(),
                               copy.stride(0),
                               c10::cuda::getCurrentCUDAStream(data.device().index()).stream()))
        return rc;
      data = copy;
    }
    if ((scale.stride(1) != 1 && blocks > 1) || scale.stride(0) < blocks)
      scale = scale.view(at::kByte).contiguous().view(at::kFloat8_e8m0fnu);
  }
  out->data = reinterpret_cast<uint64_t>(data.data_ptr());
  out->scale = reinterpret_cast<uint64_t>(scale.data_ptr());
  out->rows = rows;
  out->pitch = data.stride(0);
  out->scale_pitch = scale.stride(0);
  out->format = e4m3 ? SRS_FMT_E4M3 : SRS_FMT_E5M2;
  out->square = high != rows;
  return SRS_OK;
}

int matmul(Blocks a, Blocks b, int format, at::Tensor* out) {
  TORCH_CHECK_VALUE(a.data.device() == b.data.device(),
                    "all tensors must be on the same CUDA device");
  TORCH_CHECK_VALUE(a.data.dim() != 2 || b.data.dim() != 2 || a.data.size(1) == b.data.size(1),
                    "rows of different lengths: ", a.data.sizes(), " and ", b.data.sizes());
  const int64_t k = a.data.dim() == 2 ? a.data.size(1) : 0;
  srs_blocks left{}, right{};
  if (int rc = operand("a", &a, &left)) return rc;
  if (int rc = operand("b", &b, &right)) return rc;
  *out = at::empty({left.rows, right.rows}, a.data.options().dtype(result_type(format)));
  if (out->numel() == 0) return SRS_OK;
  return g_matmul(&left, &right, k, out->data_ptr(), format,
                  c10::cuda::getCurrentCUDAStream(a.data.device().index()).stream());
}

const at::Tensor& tensor(PyObject* obj, const char* what) {
  TORCH_CHECK_TYPE(THPVariable_Check(obj), what, " must be a tensor");
  return THPVariable_Unpack(obj);
}

PyObject* pack(const Blocks& straight, const Blocks& turned, int orientation) {
  PyObject* out = PyTuple_New(orientation == 3 ? 4 : 2);
  if (out == nullptr) return nullptr;
  Py_ssize_t i = 0;
  if (orientation & 1) {
    PyTuple_SET_ITEM(out, i++, THPVariable_Wrap(straight.data));
    PyTuple_SET_ITEM(out, i++, THPVariable_Wrap(straight.scale));
  }
  if (orientation & 2) {
    PyTuple_SET_ITEM(out, i++, THPVariable_Wrap(turned.data));
    PyTuple_SET_ITEM(out, i++, THPVariable_Wrap(turned.scale));
  }
  return out;
}

PyObject* py_bind(PyObject*, PyObject* args) {
  unsigned long long quantize_at, matmul_at, copy_at, linear_at, workspace_at;
  if (!PyArg_ParseTuple(args, "KKKKK", &quantize_at, &matmul_at, &copy_at, &linear_at,
                        &workspace_at))
    return nullptr;
  g_linear = reinterpret_cast<decltype(g_linear)>(static_cast<uintptr_t>(linear_at));
  g_linear_workspace =
      reinterpret_cast<decltype(g_linear_workspace)>(static_cast<uintptr_t>(workspace_at));
  g_quantize = reinterpret_cast<decltype(g_quantize)>(static_cast<uintptr_t>(quantize_at));
  g_matmul = reinterpret_cast<decltype(g_matmul)>(static_cast<uintptr_t>(matmul_at));
  g_copy_rows = reinterpret_cast<decltype(g_copy_rows)>(static_cast<uintptr_t>(copy_at));
  Py_RETURN_NONE;
}

PyObject* py_quantize(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject* x;
  int format, rule, square, orientation;
  unsigned int seed, offset;
  if (!PyArg_ParseTuple(args, "OiiiIIi", &x, &format, &rule, &square, &seed, &offset,
                        &orientation))
    return nullptr;
  c10::NoGradGuard no_grad;
  const at::Tensor& t = tensor(x, "x");
  const c10::cuda::OptionalCUDAGuard guard(t.device());
  Blocks straight, turned;
  const int rc = quantize(t, format, rule, square != 0, seed, offset, orientation, &straight,
                          &turned);
  if (rc != SRS_OK) return PyLong_FromLong(rc);
  return pack(straight, turned, orientation);
  END_HANDLE_TH_ERRORS
}

PyObject* py_matmul(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *a, *a_scale, *b, *b_scale;
  int format;
  if (!PyArg_ParseTuple(args, "OOOOi", &a, &a_scale, &b, &b_scale, &format)) return nullptr;
  c10::NoGradGuard no_grad;
  const at::Tensor& left = tensor(a, "a's data");
  const c10::cuda::OptionalCUDAGuard guard(left.device());
  at::Tensor out;
  const int rc = matmul({left, tensor(a_scale, "a's scale")},
                        {tensor(b, "b's data"), tensor(b_scale, "b's scale")}, format, &out);
  if (rc != SRS_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// x (..., K) quantised to nearest in rows, times the weight's blocks.
PyObject* py_linear(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *x, *w, *w_scale;
  int format;
  if (!PyArg_ParseTuple(args, "OOOi", &x, &w, &w_scale, &format)) return nullptr;
  c10::NoGradGuard no_grad;
  const at::Tensor& t = tensor(x, "x");
  const at::Tensor& weight = tensor(w, "the weight's data");
  const c10::cuda::OptionalCUDAGuard guard(t.device());
  const int x_format = source_format(t, "block_linear");
  TORCH_CHECK_VALUE(t.device() == weight.device(), "all tensors must be on the same CUDA device");
  TORCH_CHECK_VALUE(t.dim() > 0, "block_linear needs at least one dimension");
  at::Tensor flat = t.dim() == 2 ? t : t.dim() == 1 ? t.unsqueeze(0) : t.flatten(0, -2);
  const int64_t tokens = flat.size(0), k = flat.size(1);
  if (flat.stride(1) != 1 && k > 1) flat = flat.contiguous();
  Blocks blocks{weight, tensor(w_scale, "the weight's scale")};
  srs_blocks matrix{};
  int rc = operand("weight", &blocks, &matrix);
  at::Tensor out;
  if (rc == SRS_OK) {
    out = at::empty({tokens, matrix.rows}, t.options());
    const int64_t bytes = g_linear_workspace(tokens, k);
    const at::Tensor space = at::empty({bytes}, t.options().dtype(at::kByte));
    rc = g_linear(flat.data_ptr(), x_format, tokens, k, flat.stride(0), format, &matrix,
                  out.data_ptr(), space.data_ptr(), bytes,
                  c10::cuda::getCurrentCUDAStream(t.device().index()).stream());
  }
  if (rc != SRS_OK) return PyLong_FromLong(rc);
  if (t.dim() != 2) {
    std::vector<int64_t> sizes(t.sizes().begin(), t.sizes().end());
    sizes.back() = weight.size(0);
    out = out.reshape(sizes);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"bind", py_bind, METH_VARARGS,
     "bind(quantize, matmul, copy_rows, linear, linear_workspace): entry point addresses."},
    {"quantize", py_quantize, METH_VARARGS,
     "quantize(x, format, rule, square, seed, offset, orientation) -> tensors or a status."},
    {"matmul", py_matmul, METH_VARARGS,
     "matmul(a, a_scale, b, b_scale, format) -> tensor or a status."},
    {"linear", py_linear, METH_VARARGS, "linear(x, w, w_scale, format) -> tensor or a status."},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_srs_blocks",
                       "Tensor front end of the FP8 block entry points.", -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__srs_blocks(void) { return PyModule_Create(&kModule); }
