// _srs_groups: tensor front end of the operators on rows in groups (a CPython module):
// checks, allocation and launch in one call, as _srs_blocks does for the FP8 block entry points.
// A function returns the negative status of an entry point as an int; the caller turns it
// into the error.
#include "host_blocks.h"

namespace {

decltype(&srs_group_rows) g_group_rows = nullptr;
decltype(&srs_quantize_stack) g_quantize_stack = nullptr;
decltype(&srs_quantize_groups) g_quantize_groups = nullptr;
decltype(&srs_group_columns) g_group_columns = nullptr;
decltype(&srs_group_scales) g_group_scales = nullptr;
decltype(&srs_expert_matmul) g_expert_matmul = nullptr;
decltype(&srs_expert_linear) g_expert_linear = nullptr;
decltype(&srs_expert_gradient) g_expert_gradient = nullptr;
decltype(&srs_linear_workspace) g_linear_workspace = nullptr;
decltype(&srs_adapter_workspace) g_adapter_workspace = nullptr;
decltype(&srs_adapter_linear) g_adapter_linear = nullptr;
decltype(&srs_adapter_gradient_workspace) g_gradient_workspace = nullptr;
decltype(&srs_adapter_gradient) g_adapter_gradient = nullptr;

void* stream_of(const at::Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

// `ends` as int32 on x's device (int64 is converted).
at::Tensor checked_ends(const at::Tensor& ends, const at::Tensor& x, const char* what) {
  TORCH_CHECK_TYPE(ends.scalar_type() == at::kInt || ends.scalar_type() == at::kLong, what,
                   ": ends are int32 or int64, got ", ends.scalar_type());
  TORCH_CHECK_VALUE(ends.dim() == 1 && ends.numel() > 0, what,
                    ": ends must have one dimension and one entry a group, got shape ",
                    ends.sizes());
  TORCH_CHECK_VALUE(ends.device() == x.device(), "all tensors must be on the same CUDA device");
  return ends.to(at::kInt).contiguous();
}

srs_block_copy copy_of(const Blocks& b) {
  srs_block_copy c{};
  if (!b.data.defined()) return c;
  c.data = reinterpret_cast<uint64_t>(b.data.data_ptr());
  c.scale = reinterpret_cast<uint64_t>(b.scale.data_ptr());
  const int64_t last = b.data.dim() - 2;
  c.pitch = b.data.stride(last);
  c.scale_pitch = b.scale.stride(last);
  if (last == 1) {
    c.stride = b.data.stride(0);
    c.scale_stride = b.scale.stride(0);
  }
  return c;
}

Blocks empty_stack(int64_t matrices, int64_t rows, int64_t cols, int format, bool square,
                   const at::Tensor& like) {
  const int64_t row_bytes = ceil_div(cols, 16) * 16;
  Blocks b;
  b.data = at::empty({matrices, rows, row_bytes},
                     like.options().dtype(format == SRS_FMT_E4M3 ? at::kFloat8_e4m3fn
                                                                 : at::kFloat8_e5m2));
  if (row_bytes != cols) b.data = b.data.narrow(2, 0, cols);
  b.scale = at::empty({matrices, square ? ceil_div(rows, kBlock) : rows, ceil_div(cols, kBlock)},
                      like.options().dtype(at::kFloat8_e8m0fnu));
  return b;
}

// The weights of all groups, (groups, n, k), as one operand of groups * n rows; data or scales
// laid out otherwise are copied once, `b` keeps the copies alive.
int stack_operand(const char* name, Blocks* b, srs_blocks* out) {
  at::Tensor &data = b->data, &scale = b->scale;
  const bool e4m3 = data.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK_TYPE(e4m3 || data.scalar_type() == at::kFloat8_e5m2, name,
                   ": block data are float8_e4m3fn or float8_e5m2, got ", data.scalar_type());
  TORCH_CHECK_TYPE(scale.scalar_type() == at::kFloat8_e8m0fnu, name,
                   ": block scales are float8_e8m0fnu, got ", scale.scalar_type());
  TORCH_CHECK_VALUE(data.dim() == 3 && scale.dim() == 3, name,
                    ": data and scale must be stacks of matrices");
  TORCH_CHECK_VALUE(data.device() == scale.device(), name,
                    ": data and scale must be on the same CUDA device");
  const int64_t groups = data.size(0), n = data.size(1), k = data.size(2);
  const int64_t blocks = ceil_div(k, kBlock), high = scale.size(1);
  TORCH_CHECK_VALUE(scale.size(0) == groups && scale.size(2) == blocks &&
                        (high == n || high == ceil_div(n, kBlock)),
                    name, ": scale of shape ", scale.sizes(), " does not fit data of shape ",
                    data.sizes());
  // the pitch of all rows, where one describes them
  const auto pitch_of = [](const at::Tensor& t, int64_t least) -> int64_t {
    if (t.size(2) > 1 && t.stride(2) != 1) return -1;
    if (t.size(0) == 1 && t.size(1) == 1) return least;
    const int64_t p = t.size(1) > 1 ? t.stride(1) : t.stride(0);
    return p >= t.size(2) && (t.size(0) == 1 || t.stride(0) == t.size(1) * p) ? p : -1;
  };
  int64_t data_pitch = ceil_div(k, 16) * 16, scale_pitch = blocks;
  if (data.numel() != 0) {
    data_pitch = pitch_of(data, data_pitch);
    if (data_pitch < 0 || data_pitch % 16 != 0 ||
        reinterpret_cast<uintptr_t>(data.data_ptr()) % 16 != 0) {
      const at::Tensor flat = data.contiguous();
      data_pitch = ceil_div(k, 16) * 16;
      at::Tensor copy = at::empty({groups, n, data_pitch}, data.options());
      if (int rc = g_copy_rows(flat.data_ptr(), k, groups * n, k, copy.data_ptr(), data_pitch,
                               stream_of(data)))
        return rc;
      data = copy;
    }
    scale_pitch = pitch_of(scale, blocks);
    if (scale_pitch < 0) {
      scale = scale.view(at::kByte).contiguous().view(at::kFloat8_e8m0fnu);
      scale_pitch = blocks;
    }
  }
  out->data = reinterpret_cast<uint64_t>(data.data_ptr());
  out->scale = reinterpret_cast<uint64_t>(scale.data_ptr());
  out->rows = groups * n;
  out->pitch = data_pitch;
  out->scale_pitch = scale_pitch;
  out->format = e4m3 ? SRS_FMT_E4M3 : SRS_FMT_E5M2;
  out->square = high != n;
  return SRS_OK;
}

PyObject* wrap(std::initializer_list<at::Tensor> tensors) {
  PyObject* out = PyTuple_New((Py_ssize_t)tensors.size());
  if (out == nullptr) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& t : tensors) PyTuple_SET_ITEM(out, i++, THPVariable_Wrap(t));
  return out;
}

template <class F>
bool bind_one(PyObject* table, const char* name, F* to) {
  PyObject* address = PyDict_GetItemString(table, name);
  if (address == nullptr) {
    PyErr_Format(PyExc_KeyError, "%s", name);
    return false;
  }
  const unsigned long long at = PyLong_AsUnsignedLongLong(address);
  if (PyErr_Occurred()) return false;
  *to = reinterpret_cast<F>(static_cast<uintptr_t>(at));
  return true;
}

PyObject* py_bind(PyObject*, PyObject* args) {
  PyObject* t;
  if (!PyArg_ParseTuple(args, "O!", &PyDict_Type, &t)) return nullptr;
  if (!bind_one(t, "srs_group_rows", &g_group_rows) ||
      !bind_one(t, "srs_quantize_stack", &g_quantize_stack) ||
      !bind_one(t, "srs_quantize_groups", &g_quantize_groups) ||
      !bind_one(t, "srs_group_columns", &g_group_columns) ||
      !bind_one(t, "srs_group_scales", &g_group_scales) ||
      !bind_one(t, "srs_expert_matmul", &g_expert_matmul) ||
      !bind_one(t, "srs_expert_linear", &g_expert_linear) ||
      !bind_one(t, "srs_expert_gradient", &g_expert_gradient) ||
      !bind_one(t, "srs_linear_workspace", &g_linear_workspace) ||
      !bind_one(t, "srs_adapter_workspace", &g_adapter_workspace) ||
      !bind_one(t, "srs_adapter_linear", &g_adapter_linear) ||
      !bind_one(t, "srs_adapter_gradient_workspace", &g_gradient_workspace) ||
      !bind_one(t, "srs_adapter_gradient", &g_adapter_gradient) ||
      !bind_one(t, "srs_copy_rows", &g_copy_rows))
    return nullptr;
  Py_RETURN_NONE;
}

PyObject* py_group_rows(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject* obj;
  int groups;
  if (!PyArg_ParseTuple(args, "Oi", &obj, &groups)) return nullptr;
  c10::NoGradGuard no_grad;
  const at::Tensor& index = tensor(obj, "index");
  const c10::cuda::OptionalCUDAGuard guard(index.device());
  TORCH_CHECK_TYPE(index.scalar_type() == at::kInt || index.scalar_type() == at::kLong,
                   "group_rows: indices are int32 or int64, got ", index.scalar_type());
  TORCH_CHECK_VALUE(groups > 0, "group_rows: groups must be positive, got ", groups);
  const at::Tensor flat = index.contiguous();
  const auto ints = index.options().dtype(at::kInt);
  at::Tensor order = at::empty({index.numel()}, ints), ends = at::empty({groups}, ints);
  const int rc = g_group_rows(flat.data_ptr(), (int)index.element_size(), index.numel(), groups,
                              static_cast<int32_t*>(order.data_ptr()),
                              static_cast<int32_t*>(ends.data_ptr()), stream_of(index));
  if (rc != SRS_OK) return PyLong_FromLong(rc);
  return wrap({order, ends});
  END_HANDLE_TH_ERRORS
}

PyObject* py_quantize_stack(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject* obj;
  int format, rule, square, orientation;
  unsigned int seed, offset;
  if (!PyArg_ParseTuple(args, "OiiiIIi", &obj, &format, &rule, &square, &seed, &offset,
                        &orientation))
    return nullptr;
  c10::NoGradGuard no_grad;
  const at::Tensor& x = tensor(obj, "x");
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  const int x_format = source_format(x, "quantize_blocks");
  TORCH_CHECK_VALUE(x.dim() == 3, "a stack of matrices has three dimensions, got shape ",
                    x.sizes());
  const at::Tensor src = x.stride(2) != 1 && x.size(2) > 1 ? x.contiguous() : x;
  const int64_t matrices = x.size(0), rows = x.size(1), cols = x.size(2);
  Blocks straight, turned;
  if (orientation & 1) straight = empty_stack(matrices, rows, cols, format, square != 0, x);
  if (orientation & 2) turned = empty_stack(matrices, cols, rows, format, square != 0, x);
  if (x.numel() != 0) {
    const srs_block_copy copy = copy_of(straight), copy_t = copy_of(turned);
    const int rc = g_quantize_stack(src.data_ptr(), x_format, matrices, rows, cols, src.stride(1),
                                    src.stride(0), format, rule, square, seed, offset, &copy,
                                    &copy_t, stream_of(x));
    if (rc != SRS_OK) return PyLong_FromLong(rc);
  }
  if (orientation == 3) return wrap({straight.data, straight.scale, turned.data, turned.scale});
  const Blocks& one = orientation == 1 ? straight : turned;
  return wrap({one.data, one.scale});
  END_HANDLE_TH_ERRORS
}

// The transposed copy of a matrix whose rows are in groups; with `rows` the copy by rows, too.
PyObject* py_quantize_groups(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *obj, *ends_obj;
  int format, rule, rows;
  unsigned int seed;
  if (!PyArg_ParseTuple(args, "OOiiIi", &obj, &ends_obj, &format, &rule, &seed, &rows))
    return nullptr;
  c10::NoGradGuard no_grad;
  const at::Tensor& x = tensor(obj, "x");
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  const int x_format = source_format(x, "quantize_groups");
  TORCH_CHECK_VALUE(x.dim() == 2, "quantize_groups needs a matrix, got shape ", x.sizes());
  const at::Tensor ends = checked_ends(tensor(ends_obj, "ends"), x, "quantize_groups");
  const at::Tensor src = x.stride(1) != 1 && x.size(1) > 1 ? x.contiguous() : x;
  const int64_t height = x.size(0), cols = x.size(1);
  const int groups = (int)ends.numel();
  Blocks straight, turned;
  if (rows) straight = empty_blocks(height, cols, format, false, x);
  turned.data = at::empty({cols, g_group_columns(height, groups)},
                          x.options().dtype(format == SRS_FMT_E4M3 ? at::kFloat8_e4m3fn
                                                                   : at::kFloat8_e5m2));
  turned.scale = at::empty({cols, ceil_div(g_group_scales(height, groups), 4) * 4},
                           x.options().dtype(at::kFloat8_e8m0fnu));
  if (x.numel() != 0) {
    const srs_block_copy copy = copy_of(straight), copy_t = copy_of(turned);
    const int rc = g_quantize_groups(src.data_ptr(), x_format, height, cols, src.stride(0),
                                     static_cast<const int32_t*>(ends.data_ptr()), groups, format,
                                     rule, seed, 0u, &copy, &copy_t, stream_of(x));
    if (rc != SRS_OK) return PyLong_FromLong(rc);
  }
  if (rows) return wrap({straight.data, straight.scale, turned.data, turned.scale});
  return wrap({turned.data, turned.scale});
  END_HANDLE_TH_ERRORS
}

void check_groups(const at::Tensor& ends, const at::Tensor& weight) {
  TORCH_CHECK_VALUE(weight.dim() != 3 || ends.numel() == weight.size(0), "ends of ", ends.numel(),
                    " groups do not fit weights of shape ", weight.sizes());
}

PyObject* py_expert_matmul(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *a_obj, *a_scale, *w_obj, *w_scale, *ends_obj;
  int format;
  if (!PyArg_ParseTuple(args, "OOOOOi", &a_obj, &a_scale, &w_obj, &w_scale, &ends_obj, &format))
    return nullptr;
  c10::NoGradGuard no_grad;
  Blocks a{tensor(a_obj, "a's data"), tensor(a_scale, "a's scale")};
  Blocks w{tensor(w_obj, "the weight's data"), tensor(w_scale, "the weight's scale")};
  const c10::cuda::OptionalCUDAGuard guard(a.data.device());
  const at::Tensor ends = checked_ends(tensor(ends_obj, "ends"), a.data, "expert_linear");
  TORCH_CHECK_VALUE(a.data.device() == w.data.device(),
                    "all tensors must be on the same CUDA device");
  check_groups(ends, w.data);
  const int64_t rows = a.data.size(0), n = w.data.size(1), k = w.data.size(2);
  srs_blocks left{}, right{};
  int rc = operand("a", &a, &left);
  if (rc == SRS_OK) rc = stack_operand("weight", &w, &right);
  at::Tensor out;
  if (rc == SRS_OK) {
    out = at::empty({rows, n}, a.data.options().dtype(result_type(format)));
    left.square = 0;  // (one row: both forms have one scale a block)
    if (out.numel() != 0)
      rc = g_expert_matmul(&left, &right, (int)ends.numel(),
                           static_cast<const int32_t*>(ends.data_ptr()), k, out.data_ptr(), format,
                           stream_of(out));
  }
  if (rc != SRS_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// x (rows, k) quantised to nearest in rows, times the blocks of its rows' groups.
PyObject* py_expert_linear(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *obj, *w_obj, *w_scale, *ends_obj;
  int format;
  if (!PyArg_ParseTuple(args, "OOOOi", &obj, &w_obj, &w_scale, &ends_obj, &format)) return nullptr;
  c10::NoGradGuard no_grad;
  const at::Tensor& x = tensor(obj, "x");
  Blocks w{tensor(w_obj, "the weight's data"), tensor(w_scale, "the weight's scale")};
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  const int x_format = source_format(x, "expert_linear");
  const at::Tensor ends = checked_ends(tensor(ends_obj, "ends"), x, "expert_linear");
  TORCH_CHECK_VALUE(x.device() == w.data.device(), "all tensors must be on the same CUDA device");
  check_groups(ends, w.data);
  const int64_t rows = x.size(0), k = x.size(1), n = w.data.size(1);
  const at::Tensor src = x.stride(1) != 1 && k > 1 ? x.contiguous() : x;
  srs_blocks matrix{};
  int rc = stack_operand("weight", &w, &matrix);
  at::Tensor out;
  if (rc == SRS_OK) {
    out = at::empty({rows, n}, x.options());
    const int64_t bytes = g_linear_workspace(rows, k);
    const at::Tensor space = at::empty({bytes}, x.options().dtype(at::kByte));
    if (out.numel() != 0)
      rc = g_expert_linear(src.data_ptr(), x_format, rows, k, src.stride(0), format, &matrix,
                           (int)ends.numel(), static_cast<const int32_t*>(ends.data_ptr()),
                           out.data_ptr(), space.data_ptr(), bytes, stream_of(x));
  }
  if (rc != SRS_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// Transposed copies of two matrices whose `rows` rows are in groups -> (groups, m, n).
PyObject* py_expert_gradient(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *a_obj, *a_scale, *b_obj, *b_scale, *ends_obj;
  long long rows;
  int format;
  if (!PyArg_ParseTuple(args, "OOOOLOi", &a_obj, &a_scale, &b_obj, &b_scale, &rows, &ends_obj,
                        &format))
    return nullptr;
  c10::NoGradGuard no_grad;
  const Blocks a{tensor(a_obj, "a's data"), tensor(a_scale, "a's scale")};
  const Blocks b{tensor(b_obj, "b's data"), tensor(b_scale, "b's scale")};
  const c10::cuda::OptionalCUDAGuard guard(a.data.device());
  const at::Tensor ends = checked_ends(tensor(ends_obj, "ends"), a.data, "expert_linear");
  srs_blocks left{}, right{};
  for (const auto& [from, to] : {std::make_pair(&a, &left), std::make_pair(&b, &right)}) {
    to->data = reinterpret_cast<uint64_t>(from->data.data_ptr());
    to->scale = reinterpret_cast<uint64_t>(from->scale.data_ptr());
    to->rows = from->data.size(0);
    to->pitch = from->data.stride(0);
    to->scale_pitch = from->scale.stride(0);
    to->format = from->data.scalar_type() == at::kFloat8_e4m3fn ? SRS_FMT_E4M3 : SRS_FMT_E5M2;
  }
  at::Tensor out = at::empty({ends.numel(), left.rows, right.rows},
                             a.data.options().dtype(result_type(format)));
  int rc = SRS_OK;
  if (out.numel() != 0)
    rc = g_expert_gradient(&left, &right, rows, (int)ends.numel(),
                           static_cast<const int32_t*>(ends.data_ptr()), out.data_ptr(), format,
                           stream_of(out));
  if (rc != SRS_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// A 16-bit matrix, or a stack of them, whose rows start on 16-byte boundaries; one laid out
// otherwise is copied once.  `whole`: rows of whole 16 bytes as well.
at::Tensor aligned(const at::Tensor& t, bool whole) {
  const int64_t last = t.dim() - 1, cols = t.size(last);
  bool good = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
              (cols <= 1 || t.stride(last) == 1) && (!whole || cols % 8 == 0);
  for (int64_t d = 0; d < last; ++d)
    good = good && (t.size(d) <= 1 || (t.stride(d) % 8 == 0 && (d != last - 1 || t.stride(d) >= cols)));
  if (good || t.numel() == 0) return t;
  std::vector<int64_t> sizes(t.sizes().begin(), t.sizes().end());
  sizes[last] = ceil_div(cols, 8) * 8;
  at::Tensor copy = at::empty(sizes, t.options()).narrow(last, 0, cols);
  copy.copy_(t);
  return copy;
}

// Elements from one index of dimension `d` to the next; of one index alone, `otherwise`.
int64_t step_of(const at::Tensor& t, int64_t d, int64_t otherwise) {
  return t.size(d) > 1 ? t.stride(d) : otherwise;
}

struct Adapters {
  at::Tensor down, up, scale, order, ends;
  srs_adapters c{};
};

void set_adapters(Adapters* a, const at::Tensor& x, int64_t in, int64_t out, PyObject* down,
                  PyObject* up, PyObject* scale, double factor, PyObject* order, PyObject* ends) {
  const char* what = "adapter_linear";
  a->down = tensor(down, "down");
  a->up = tensor(up, "up");
  TORCH_CHECK_TYPE(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, what,
                   " takes BF16 or FP16, got ", x.scalar_type());
  TORCH_CHECK_TYPE(
      a->down.scalar_type() == x.scalar_type() && a->up.scalar_type() == x.scalar_type(), what,
      ": adapters in x's dtype ", x.scalar_type(), " needed, got ", a->down.scalar_type(), " and ",
      a->up.scalar_type());
  TORCH_CHECK_VALUE(a->down.device() == x.device() && a->up.device() == x.device(),
                    "all tensors must be on the same CUDA device");
  TORCH_CHECK_VALUE(a->down.dim() == 3 && a->up.dim() == 3 && a->down.size(0) == a->up.size(0) &&
                        a->down.size(1) == a->up.size(2) && a->down.size(2) == in &&
                        a->up.size(1) == out,
                    what, ": down of shape ", a->down.sizes(), " and up of shape ", a->up.sizes(),
                    " do not fit a projection from ", in, " to ", out);
  const int64_t count = a->down.size(0), rank = a->down.size(1);
  TORCH_CHECK_VALUE(rank > 0 && rank <= SRS_ADAPTER_MAX_RANK, what, ": the rank must be in [1, ",
                    SRS_ADAPTER_MAX_RANK, "], got ", rank);
  a->ends = checked_ends(tensor(ends, "ends"), x, what);
  TORCH_CHECK_VALUE(a->ends.numel() == count, what, ": ends of ", a->ends.numel(),
                    " groups do not fit ", count, " adapters");
  const at::Tensor& places = tensor(order, "order");
  TORCH_CHECK_TYPE(places.scalar_type() == at::kInt || places.scalar_type() == at::kLong, what,
                   ": the order is int32 or int64, got ", places.scalar_type());
  TORCH_CHECK_VALUE(places.device() == x.device() && places.dim() == 1 &&
                        places.numel() == x.size(0),
                    what, ": order of shape ", places.sizes(), " does not fit ", x.size(0),
                    " tokens on ", x.device());
  a->order = places.to(at::kInt).contiguous();
  if (scale != Py_None) {
    a->scale = tensor(scale, "scale");
    TORCH_CHECK_TYPE(a->scale.scalar_type() == at::kFloat, what, ": scales are FP32, got ",
                     a->scale.scalar_type());
    TORCH_CHECK_VALUE(a->scale.device() == x.device() && a->scale.dim() == 1 &&
                          a->scale.numel() == count,
                      what, ": scales of shape ", a->scale.sizes(), " do not fit ", count,
                      " adapters on ", x.device());
    a->scale = a->scale.contiguous();
    a->c.scale = reinterpret_cast<uint64_t>(a->scale.data_ptr());
  }
  a->down = aligned(a->down, false);
  a->up = aligned(a->up, true);
  srs_adapters& c = a->c;
  c.down = reinterpret_cast<uint64_t>(a->down.data_ptr());
  c.up = reinterpret_cast<uint64_t>(a->up.data_ptr());
  c.order = reinterpret_cast<uint64_t>(a->order.data_ptr());
  c.ends = reinterpret_cast<uint64_t>(a->ends.data_ptr());
  c.down_pitch = step_of(a->down, 1, ceil_div(in, 8) * 8);
  c.down_stride = step_of(a->down, 0, 0);
  c.up_pitch = step_of(a->up, 1, ceil_div(rank, 8) * 8);
  c.up_stride = step_of(a->up, 0, 0);
  c.factor = (float)factor;
  c.count = (int32_t)count;
  c.rank = (int32_t)rank;
  c.format = x.scalar_type() == at::kBFloat16 ? SRS_FMT_BF16 : SRS_FMT_F16;
}

// x (tokens, k), blocks of the projection (None: the low part alone) -> (d or None, low,
// largest).  turned: x is the output's gradient.
PyObject* py_adapter_linear(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *x_obj, *w_obj, *w_scale, *down, *up, *scale, *order, *ends;
  int format, rule, turned, keep;
  unsigned int seed;
  double factor;
  if (!PyArg_ParseTuple(args, "OiiIOOOOOdOOii", &x_obj, &format, &rule, &seed, &w_obj, &w_scale,
                        &down, &up, &scale, &factor, &order, &ends, &turned, &keep))
    return nullptr;
  c10::NoGradGuard no_grad;
  const at::Tensor& given = tensor(x_obj, "x");
  const c10::cuda::OptionalCUDAGuard guard(given.device());
  const int64_t tokens = given.size(0), k = given.size(1);
  Blocks blocks;
  const bool project = w_obj != Py_None;
  const int64_t n = tensor(turned ? down : up, "adapters").size(turned ? 2 : 1);
  if (project) {
    blocks = {tensor(w_obj, "the weight's data"), tensor(w_scale, "the weight's scale")};
    TORCH_CHECK_VALUE(given.device() == blocks.data.device(),
                      "all tensors must be on the same CUDA device");
    TORCH_CHECK_VALUE(blocks.data.dim() == 2 && blocks.data.size(1) == k &&
                          blocks.data.size(0) == n,
                      "adapter_linear: a weight of shape ", blocks.data.sizes(),
                      " does not fit a projection from ", k, " to ", n);
  }
  Adapters a;
  set_adapters(&a, given, turned ? n : k, turned ? k : n, down, up, scale, factor, order, ends);
  const at::Tensor x = aligned(given, false);
  srs_blocks matrix{};
  int rc = project ? operand("weight", &blocks, &matrix) : SRS_OK;
  at::Tensor out, low, largest;
  if (rc == SRS_OK) {
    if (project) out = at::empty({tokens, n}, x.options());
    if (keep) {
      low = at::empty({tokens, a.c.rank}, x.options().dtype(at::kFloat));
      // (the sums of FP16 gradients are scaled by it)
      if (a.c.format == SRS_FMT_F16)
        largest = at::empty({a.c.count}, x.options().dtype(at::kInt));
    }
    const int64_t bytes =
        g_adapter_workspace(tokens, k, project ? n : 0, a.c.count, a.c.rank);
    const at::Tensor space = at::empty({bytes}, x.options().dtype(at::kByte));
    if (tokens != 0)
      rc = g_adapter_linear(
          x.data_ptr(), tokens, k, step_of(x, 0, ceil_div(k, 8) * 8), format, rule, seed,
          project ? &matrix : nullptr, &a.c, turned, project ? out.data_ptr() : nullptr,
          keep ? static_cast<float*>(low.data_ptr()) : nullptr,
          largest.defined() ? static_cast<uint32_t*>(largest.data_ptr()) : nullptr,
          space.data_ptr(), bytes, stream_of(x));
  }
  if (rc != SRS_OK) return PyLong_FromLong(rc);
  PyObject* result = PyTuple_New(3);
  if (result == nullptr) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor* t : {&out, &low, &largest}) {
    if (t->defined()) {
      PyTuple_SET_ITEM(result, i++, THPVariable_Wrap(*t));
    } else {
      Py_INCREF(Py_None);
      PyTuple_SET_ITEM(result, i++, Py_None);
    }
  }
  return result;
  END_HANDLE_TH_ERRORS
}

// Sums over the tokens of each adapter of z (tokens, cols) by low: (count, rank, cols) or,
// turned, (count, cols, rank).
PyObject* py_adapter_gradient(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *z_obj, *low_obj, *largest_obj, *order_obj, *ends_obj;
  int turned;
  if (!PyArg_ParseTuple(args, "OOOOOi", &z_obj, &low_obj, &largest_obj, &order_obj, &ends_obj,
                        &turned))
    return nullptr;
  c10::NoGradGuard no_grad;
  const at::Tensor& given = tensor(z_obj, "z");
  const c10::cuda::OptionalCUDAGuard guard(given.device());
  const at::Tensor &low = tensor(low_obj, "low");
  const at::Tensor ends = checked_ends(tensor(ends_obj, "ends"), given, "adapter_linear");
  const at::Tensor order = tensor(order_obj, "order").to(at::kInt).contiguous();
  const at::Tensor z = aligned(given, false);
  const int64_t tokens = z.size(0), cols = z.size(1), rank = low.size(1), count = ends.numel();
  at::Tensor out = turned ? at::empty({count, cols, rank}, z.options())
                          : at::empty({count, rank, cols}, z.options());
  const int64_t bytes = g_gradient_workspace(tokens, cols, (int)count, (int)rank);
  const at::Tensor space = at::empty({bytes}, z.options().dtype(at::kByte));
  int rc = SRS_OK;
  if (out.numel() != 0)
    rc = g_adapter_gradient(
        z.data_ptr(), z.scalar_type() == at::kBFloat16 ? SRS_FMT_BF16 : SRS_FMT_F16, tokens, cols,
        step_of(z, 0, ceil_div(cols, 8) * 8), static_cast<const float*>(low.data_ptr()),
        largest_obj != Py_None
            ? static_cast<const uint32_t*>(tensor(largest_obj, "largest").data_ptr())
            : nullptr,
        (int)count, (int)rank, static_cast<const int32_t*>(order.data_ptr()),
        static_cast<const int32_t*>(ends.data_ptr()), turned, out.data_ptr(), space.data_ptr(),
        bytes, stream_of(z));
  if (rc != SRS_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"bind", py_bind, METH_VARARGS, "bind({name: address}): the library's entry points."},
    {"group_rows", py_group_rows, METH_VARARGS, "group_rows(index, groups) -> order, ends."},
    {"quantize_stack", py_quantize_stack, METH_VARARGS,
     "quantize_stack(x, format, rule, square, seed, offset, orientation) -> tensors."},
    {"quantize_groups", py_quantize_groups, METH_VARARGS,
     "quantize_groups(x, ends, format, rule, seed, rows) -> tensors."},
    {"expert_matmul", py_expert_matmul, METH_VARARGS,
     "expert_matmul(a, a_scale, w, w_scale, ends, format) -> tensor."},
    {"expert_linear", py_expert_linear, METH_VARARGS,
     "expert_linear(x, w, w_scale, ends, format) -> tensor."},
    {"expert_gradient", py_expert_gradient, METH_VARARGS,
     "expert_gradient(a_t, a_scale, b_t, b_scale, rows, ends, format) -> tensor."},
    {"adapter_linear", py_adapter_linear, METH_VARARGS,
     "adapter_linear(x, format, rule, seed, w, w_scale, down, up, scale, factor, order, ends, "
     "turned, keep) -> (d, low, largest)."},
    {"adapter_gradient", py_adapter_gradient, METH_VARARGS,
     "adapter_gradient(z, low, largest, order, ends, turned) -> tensor."},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_srs_groups",
                       "Tensor front end of the operators on rows in groups.", -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__srs_groups(void) { return PyModule_Create(&kModule); }
