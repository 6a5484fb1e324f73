// _srs_blocks: tensor front end of the FP8 block entry points (a CPython module).
//
// quantize, matmul and linear check their tensors, allocate results and enqueue on
// the current stream of the tensors' device: what a Python wrapper would do at 20 us a
// call, for kernels of 3 to 20 us.  The entry points are the C ABI's, given by
// address (bind), so that the kernels stay in libsrs_b200.so.  A function returns the
// negative status of an entry point as an int; the caller turns it into the error.
#include "host_blocks.h"

namespace {

decltype(&srs_quantize_blocks) g_quantize = nullptr;
decltype(&srs_matmul_blocks) g_matmul = nullptr;
decltype(&srs_linear_blocks) g_linear = nullptr;
decltype(&srs_linear_workspace) g_linear_workspace = nullptr;

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
  refuse_tangents("block_linear", {&t});
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
