// _srs_groups: tensor front end of the operators on rows in groups (a CPython module): checks,
// allocation, launches and the gradients' bookkeeping in one call.  In Python a training call of
// small matrices took 180 us of the host's time, most of it between the launches.
#include <torch/csrc/autograd/custom_function.h>

#include "host_blocks.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

decltype(&srs_last_error) g_last_error = nullptr;
decltype(&srs_group_rows) g_group_rows = nullptr;
decltype(&srs_quantize_stack) g_quantize_stack = nullptr;
decltype(&srs_quantize_groups) g_quantize_groups = nullptr;
decltype(&srs_group_columns) g_group_columns = nullptr;
decltype(&srs_group_scales) g_group_scales = nullptr;
decltype(&srs_matmul_blocks) g_matmul = nullptr;
decltype(&srs_expert_matmul) g_expert_matmul = nullptr;
decltype(&srs_expert_linear) g_expert_linear = nullptr;
decltype(&srs_expert_gradient) g_expert_gradient = nullptr;
decltype(&srs_linear_workspace) g_linear_workspace = nullptr;
decltype(&srs_adapter_workspace) g_adapter_workspace = nullptr;
decltype(&srs_adapter_linear) g_adapter_linear = nullptr;
decltype(&srs_adapter_gradient_workspace) g_gradient_workspace = nullptr;
decltype(&srs_adapter_gradient) g_adapter_gradient = nullptr;

// The error of an entry point: ValueError for arguments, RuntimeError else.
void check(int rc) {
  if (rc == SRS_OK) return;
  TORCH_CHECK_VALUE(rc != SRS_ERR_INVALID_ARGUMENT, g_last_error());
  TORCH_CHECK(false, g_last_error());
}

void* stream_of(const at::Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

const int32_t* ints(const at::Tensor& t) { return static_cast<const int32_t*>(t.data_ptr()); }

// `ends` as int32 on x's device (int64 is converted, what is too large for int32 to its largest).
at::Tensor checked_ends(const at::Tensor& ends, const at::Tensor& x, const char* what) {
  TORCH_CHECK_TYPE(ends.scalar_type() == at::kInt || ends.scalar_type() == at::kLong, what,
                   ": ends are int32 or int64, got ", ends.scalar_type());
  TORCH_CHECK_VALUE(ends.dim() == 1 && ends.numel() > 0, what,
                    ": ends must have one dimension and one entry a group, got shape ",
                    ends.sizes());
  TORCH_CHECK_VALUE(ends.device() == x.device(), "all tensors must be on the same CUDA device");
  if (ends.scalar_type() == at::kLong) return ends.clamp(0, INT32_MAX).to(at::kInt).contiguous();
  return ends.contiguous();
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
srs_blocks stack_operand(const char* name, Blocks* b) {
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
      check(g_copy_rows(flat.data_ptr(), k, groups * n, k, copy.data_ptr(), data_pitch,
                        stream_of(data)));
      data = copy;
    }
    scale_pitch = pitch_of(scale, blocks);
    if (scale_pitch < 0) {
      scale = scale.view(at::kByte).contiguous().view(at::kFloat8_e8m0fnu);
      scale_pitch = blocks;
    }
  }
  srs_blocks out{};
  out.data = reinterpret_cast<uint64_t>(data.data_ptr());
  out.scale = reinterpret_cast<uint64_t>(scale.data_ptr());
  out.rows = groups * n;
  out.pitch = data_pitch;
  out.scale_pitch = scale_pitch;
  out.format = e4m3 ? SRS_FMT_E4M3 : SRS_FMT_E5M2;
  out.square = high != n;
  return out;
}

// A 16-bit matrix, or a stack of them, whose rows start on 16-byte boundaries; one laid out
// otherwise is copied once.  `whole`: with memory up to 16 bytes behind the last row, too.
at::Tensor aligned(const at::Tensor& t, bool whole) {
  const int64_t last = t.dim() - 1, cols = t.size(last);
  if (t.numel() == 0) return t;
  bool good = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
              (cols <= 1 || t.stride(last) == 1);
  int64_t end = t.storage_offset() + ceil_div(cols, 8) * 8;
  for (int64_t d = 0; d < last; ++d) {
    good = good && (t.size(d) <= 1 || (t.stride(d) % 8 == 0 && (d != last - 1 || t.stride(d) >= cols)));
    end += (t.size(d) - 1) * t.stride(d);
  }
  good = good && (!whole || 2 * end <= (int64_t)t.storage().nbytes());
  if (good) return t;
  std::vector<int64_t> sizes(t.sizes().begin(), t.sizes().end());
  sizes[last] = ceil_div(cols, 8) * 8;
  const at::Tensor wide = at::empty(sizes, t.options());
  at::Tensor copy = sizes[last] == cols ? wide : wide.narrow(last, 0, cols);
  if (t.is_contiguous())
    check(g_copy_rows(t.data_ptr(), 2 * cols, t.numel() / cols, 2 * cols, wide.data_ptr(),
                      2 * sizes[last], stream_of(t)));
  else
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

// The adapters of a projection from `in` to `out`; `scale` undefined: `factor` alone.
Adapters adapters_of(const at::Tensor& x, int64_t in, int64_t out, const at::Tensor& down,
                     const at::Tensor& up, const at::Tensor& scale, double factor,
                     const at::Tensor& places, const at::Tensor& ends) {
  const char* what = "adapter_linear";
  Adapters given, *a = &given;
  a->down = down;
  a->up = up;
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
  a->ends = checked_ends(ends, x, what);
  TORCH_CHECK_VALUE(a->ends.numel() == count, what, ": ends of ", a->ends.numel(),
                    " groups do not fit ", count, " adapters");
  TORCH_CHECK_TYPE(places.scalar_type() == at::kInt || places.scalar_type() == at::kLong, what,
                   ": the order is int32 or int64, got ", places.scalar_type());
  TORCH_CHECK_VALUE(places.device() == x.device() && places.dim() == 1 &&
                        places.numel() == x.size(0),
                    what, ": order of shape ", places.sizes(), " does not fit ", x.size(0),
                    " tokens on ", x.device());
  a->order = places.to(at::kInt).contiguous();
  if (scale.defined()) {
    a->scale = scale;
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
  return given;
}

// ---------------------------------------------------------------- operators --

// How a gradient is quantised.
struct Rounding {
  int format, rule;
  uint32_t seed;
};
constexpr int kBoth = 3, kRows = 1, kColumns = 2;

// One matrix (two dimensions) or a stack of them in blocks; orientation: kRows, kColumns, kBoth.
void quantize(const at::Tensor& x, const Rounding& how, bool square, uint32_t offset,
              int orientation, Blocks* straight, Blocks* turned) {
  const int x_format = source_format(x, "quantize_blocks");
  const bool stack = x.dim() == 3;
  const int64_t last = x.dim() - 1;
  const at::Tensor src = x.stride(last) != 1 && x.size(last) > 1 ? x.contiguous() : x;
  const int64_t matrices = stack ? x.size(0) : 1, rows = x.size(last - 1), cols = x.size(last);
  const auto make = [&](int64_t high, int64_t wide) {
    return stack ? empty_stack(matrices, high, wide, how.format, square, x)
                 : empty_blocks(high, wide, how.format, square, x);
  };
  if (orientation & kRows) *straight = make(rows, cols);
  if (orientation & kColumns) *turned = make(cols, rows);
  if (x.numel() == 0) return;
  const srs_block_copy copy = straight != nullptr ? copy_of(*straight) : srs_block_copy{};
  const srs_block_copy copy_t = turned != nullptr ? copy_of(*turned) : srs_block_copy{};
  check(g_quantize_stack(src.data_ptr(), x_format, matrices, rows, cols, src.stride(last - 1),
                         stack ? src.stride(0) : 0, how.format, how.rule, square, how.seed, offset,
                         &copy, &copy_t, stream_of(x)));
}

// The transposed copy of a matrix whose rows are in groups; beside it the copy by rows.
void quantize_groups(const at::Tensor& x, const at::Tensor& ends, const Rounding& how,
                     Blocks* straight, Blocks* turned) {
  const int x_format = source_format(x, "expert_linear");
  const at::Tensor src = x.stride(1) != 1 && x.size(1) > 1 ? x.contiguous() : x;
  const int64_t height = x.size(0), cols = x.size(1);
  const int groups = (int)ends.numel();
  if (straight != nullptr) *straight = empty_blocks(height, cols, how.format, false, x);
  turned->data = at::empty({cols, g_group_columns(height, groups)},
                           x.options().dtype(how.format == SRS_FMT_E4M3 ? at::kFloat8_e4m3fn
                                                                        : at::kFloat8_e5m2));
  turned->scale = at::empty({cols, g_group_scales(height, groups)},
                            x.options().dtype(at::kFloat8_e8m0fnu));
  if (x.numel() == 0) return;
  const srs_block_copy copy = straight != nullptr ? copy_of(*straight) : srs_block_copy{};
  const srs_block_copy copy_t = copy_of(*turned);
  check(g_quantize_groups(src.data_ptr(), x_format, height, cols, src.stride(0), ints(ends), groups,
                          how.format, how.rule, how.seed, 0u, &copy, &copy_t, stream_of(x)));
}

// a[i] w_e^T for the rows i of group e.
at::Tensor expert_matmul(Blocks a, Blocks w, const at::Tensor& ends, at::ScalarType type,
                         int format) {
  srs_blocks left{};
  check(operand("a", &a, &left));
  const srs_blocks right = stack_operand("weight", &w);
  const int64_t n = w.data.size(1), k = w.data.size(2);
  at::Tensor out = at::empty({left.rows, n}, a.data.options().dtype(type));
  left.square = 0;  // (one row: both forms have one scale a block)
  if (out.numel() != 0)
    check(g_expert_matmul(&left, &right, (int)ends.numel(), ints(ends), k, out.data_ptr(), format,
                          stream_of(out)));
  return out;
}

srs_blocks turned_operand(const Blocks& b) {
  srs_blocks o{};
  o.data = reinterpret_cast<uint64_t>(b.data.data_ptr());
  o.scale = reinterpret_cast<uint64_t>(b.scale.data_ptr());
  o.rows = b.data.size(0);
  o.pitch = b.data.stride(0);
  o.scale_pitch = b.scale.stride(0);
  o.format = b.data.scalar_type() == at::kFloat8_e4m3fn ? SRS_FMT_E4M3 : SRS_FMT_E5M2;
  return o;
}

// a_e^T b_e of two matrices of `rows` rows from their transposed copies.
at::Tensor expert_gradient(const Blocks& a, const Blocks& b, int64_t rows, const at::Tensor& ends,
                           at::ScalarType type, int format) {
  const srs_blocks left = turned_operand(a), right = turned_operand(b);
  at::Tensor out =
      at::empty({ends.numel(), left.rows, right.rows}, a.data.options().dtype(type));
  if (out.numel() != 0)
    check(g_expert_gradient(&left, &right, rows, (int)ends.numel(), ints(ends), out.data_ptr(),
                            format, stream_of(out)));
  return out;
}

int format_of(at::ScalarType type) {
  return type == at::kFloat ? SRS_FMT_F32 : type == at::kBFloat16 ? SRS_FMT_BF16 : SRS_FMT_F16;
}

void once(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what,
              " has a first derivative only: its backward pass cannot be differentiated");
}

struct ExpertLinear : torch::autograd::Function<ExpertLinear> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight,
                            const at::Tensor& ends, int64_t format, int64_t grad_format,
                            int64_t grad_rule, int64_t seed, bool need_x, bool need_w) {
    const Rounding nearest{(int)format, SRS_RULE_NEAREST, 0u};
    Blocks tokens, tokens_t, matrix, matrix_t;
    if (need_w) quantize_groups(x, ends, nearest, &tokens, &tokens_t);
    else quantize(x, nearest, false, 0u, kRows, &tokens, nullptr);
    quantize(weight, nearest, true, 0u, need_x ? kBoth : kRows, &matrix,
             need_x ? &matrix_t : nullptr);
    ctx->save_for_backward(
        {ends, tokens_t.data, tokens_t.scale, matrix_t.data, matrix_t.scale});
    ctx->saved_data["how"] = std::vector<int64_t>{grad_format, grad_rule, seed, need_x, need_w,
                                                  (int64_t)x.scalar_type(),
                                                  (int64_t)weight.scalar_type()};
    return expert_matmul(tokens, matrix, ends, x.scalar_type(), format_of(x.scalar_type()));
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("expert_linear");
    const std::vector<int64_t> s = ctx->saved_data["how"].toIntVector();
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &dy = grads[0], &ends = saved[0];
    const c10::cuda::OptionalCUDAGuard guard(dy.device());
    const Rounding how{(int)s[0], (int)s[1], (uint32_t)s[2]};
    const bool need_x = s[3] != 0, need_w = s[4] != 0;
    const auto x_type = (at::ScalarType)s[5], w_type = (at::ScalarType)s[6];
    Blocks rows, columns;
    if (need_w) quantize_groups(dy, ends, how, need_x ? &rows : nullptr, &columns);
    else quantize(dy, how, false, 0u, kRows, &rows, nullptr);
    variable_list out(9);
    if (need_x) out[0] = expert_matmul(rows, {saved[3], saved[4]}, ends, x_type, format_of(x_type));
    if (need_w)
      out[1] = expert_gradient(columns, {saved[1], saved[2]}, dy.size(0), ends, w_type,
                               format_of(w_type));
    return out;
  }
};

// ----------------------------------------------------------------- adapters --

struct Low {
  at::Tensor values, largest;
};

// x (tokens, k) by the projection's blocks (undefined: the low part alone) and the adapters;
// turned: x is the result's gradient.
at::Tensor adapter_product(const at::Tensor& given, const Rounding& how, Blocks blocks,
                           const at::Tensor& down, const at::Tensor& up, const at::Tensor& scale,
                           double factor, const at::Tensor& order, const at::Tensor& ends,
                           bool turned, Low* low) {
  const int64_t tokens = given.size(0), k = given.size(1);
  const bool project = blocks.data.defined();
  TORCH_CHECK_VALUE(down.dim() == 3 && up.dim() == 3, "adapter_linear: down of shape ",
                    down.sizes(), " and up of shape ", up.sizes(), " are not stacks of matrices");
  const int64_t n = turned ? down.size(2) : up.size(1);
  if (project) {
    TORCH_CHECK_VALUE(given.device() == blocks.data.device(),
                      "all tensors must be on the same CUDA device");
    TORCH_CHECK_VALUE(blocks.data.dim() == 2 && blocks.data.size(1) == k &&
                          blocks.data.size(0) == n,
                      "adapter_linear: a weight of shape ", blocks.data.sizes(),
                      " does not fit a projection from ", k, " to ", n);
  }
  const Adapters a = adapters_of(given, turned ? n : k, turned ? k : n, down, up, scale, factor,
                                 order, ends);
  const at::Tensor x = aligned(given, false);
  srs_blocks matrix{};
  if (project) check(operand("weight", &blocks, &matrix));
  at::Tensor out;
  if (project) out = at::empty({tokens, n}, x.options());
  if (low != nullptr) {
    low->values = at::empty({tokens, a.c.rank}, x.options().dtype(at::kFloat));
    // (the sums of FP16 gradients are scaled by it)
    if (a.c.format == SRS_FMT_F16)
      low->largest = at::empty({a.c.count}, x.options().dtype(at::kInt));
  }
  if (tokens == 0) return out;
  const int64_t bytes = g_adapter_workspace(tokens, k, project ? n : 0, a.c.count, a.c.rank);
  const at::Tensor space = at::empty({bytes}, x.options().dtype(at::kByte));
  check(g_adapter_linear(
      x.data_ptr(), tokens, k, step_of(x, 0, ceil_div(k, 8) * 8), how.format, how.rule, how.seed,
      project ? &matrix : nullptr, &a.c, turned, project ? out.data_ptr() : nullptr,
      low != nullptr ? static_cast<float*>(low->values.data_ptr()) : nullptr,
      low != nullptr && low->largest.defined() ? static_cast<uint32_t*>(low->largest.data_ptr())
                                               : nullptr,
      space.data_ptr(), bytes, stream_of(x)));
  return out;
}

// A sum over the tokens of each adapter of z (tokens, cols) by low: (adapters, rank, cols) or,
// turned, (adapters, cols, rank).
struct Sum {
  at::Tensor z;
  const Low* low;
  bool turned;
  at::Tensor out;
};

// One or two sums in one call.
void adapter_gradients(std::vector<Sum>& sums, const at::Tensor& order, const at::Tensor& ends) {
  srs_adapter_sum jobs[2] = {};
  int64_t cols = 0, filled = 0;
  int n = 0;
  const int64_t count = ends.numel();
  for (Sum& sum : sums) {
    sum.z = aligned(sum.z, false);
    const int64_t wide = sum.z.size(1), rank = sum.low->values.size(1);
    sum.out = sum.turned ? at::empty({count, wide, rank}, sum.z.options())
                         : at::empty({count, rank, wide}, sum.z.options());
    srs_adapter_sum& job = jobs[n++];
    job.z = reinterpret_cast<uint64_t>(sum.z.data_ptr());
    job.z_pitch = step_of(sum.z, 0, ceil_div(wide, 8) * 8);
    job.cols = wide;
    job.low = reinterpret_cast<uint64_t>(sum.low->values.data_ptr());
    if (sum.low->largest.defined())
      job.largest = reinterpret_cast<uint64_t>(sum.low->largest.data_ptr());
    job.out = reinterpret_cast<uint64_t>(sum.out.data_ptr());
    job.turned = sum.turned;
    cols += wide;
    filled += sum.out.numel();
  }
  if (filled == 0) return;
  const at::Tensor& z = sums[0].z;
  const int64_t tokens = z.size(0), rank = sums[0].low->values.size(1);
  const int64_t bytes = g_gradient_workspace(tokens, cols, (int)count, (int)rank);
  const at::Tensor space = at::empty({bytes}, z.options().dtype(at::kByte));
  check(g_adapter_gradient(jobs, n, format_of(z.scalar_type()), tokens, (int)count, (int)rank,
                           ints(order), ints(ends), space.data_ptr(), bytes, stream_of(z)));
}

at::Tensor flat(const at::Tensor& x) {
  return x.dim() == 2 ? x : x.dim() == 1 ? x.unsqueeze(0) : x.flatten(0, -2);
}

// (no view: autograd refuses to change one in place that was made inside a function)
at::Tensor shaped(const at::Tensor& rows, at::IntArrayRef like) {
  if (like.size() == 2) return rows;
  std::vector<int64_t> sizes(like.begin(), like.end());
  sizes.back() = rows.size(1);
  return at::_unsafe_view(rows, sizes);
}

// What of a call is no leaf.
struct AdapterInputs {
  Blocks kept, turned;  // undefined: the weight itself is given
  at::Tensor scale, order, ends;
  double factor;
  int format;
  Rounding grad;
  std::vector<int64_t> need;  // gradients of x, weight, down, up
};

struct AdapterLinear : torch::autograd::Function<AdapterLinear> {
  enum { kX, kDown, kUp, kScale, kOrder, kEnds, kLow, kLargest, kMatrix, kMatrixScale, kTokens,
         kTokensScale };

  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x,
                            const std::optional<at::Tensor>& weight, const at::Tensor& down,
                            const at::Tensor& up, const AdapterInputs& in) {
    const Rounding nearest{in.format, SRS_RULE_NEAREST, 0u};
    const std::vector<int64_t>& need = in.need;
    Blocks matrix = in.kept, matrix_t = in.turned, tokens_t;
    const at::Tensor rows = flat(x);
    if (weight.has_value()) {
      matrix_t = {};
      quantize(*weight, nearest, true, 0u, need[0] ? kBoth : kRows, &matrix,
               need[0] ? &matrix_t : nullptr);
    }
    Low low;
    // (a copy that the kernels' alignment asks for is made once for both passes)
    const at::Tensor x_rows = aligned(rows, false), a = aligned(down, false), b = aligned(up, true);
    const at::Tensor y = adapter_product(x_rows, nearest, matrix, a, b, in.scale, in.factor,
                                         in.order, in.ends, false, need[3] ? &low : nullptr);
    if (need[1]) quantize(rows, nearest, false, 0u, kColumns, nullptr, &tokens_t);
    if (!need[0]) matrix_t = {};
    ctx->save_for_backward({need[2] ? x_rows : at::Tensor(), a, b, in.scale, in.order, in.ends,
                            low.values, low.largest, matrix_t.data, matrix_t.scale, tokens_t.data,
                            tokens_t.scale});
    ctx->saved_data["need"] = need;
    ctx->saved_data["how"] = std::vector<int64_t>{
        in.grad.format, in.grad.rule, (int64_t)in.grad.seed,
        (int64_t)(weight.has_value() ? weight->scalar_type() : at::kFloat)};
    ctx->saved_data["factor"] = in.factor;
    ctx->saved_data["sizes"] = x.sizes().vec();
    return shaped(y, x.sizes());
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("adapter_linear");
    const std::vector<int64_t> need = ctx->saved_data["need"].toIntVector();
    const std::vector<int64_t> s = ctx->saved_data["how"].toIntVector();
    const double factor = ctx->saved_data["factor"].toDouble();
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor dy = aligned(flat(grads[0]), false);
    const c10::cuda::OptionalCUDAGuard guard(dy.device());
    const Rounding how{(int)s[0], (int)s[1], (uint32_t)s[2]};
    const at::Tensor &order = saved[kOrder], &ends = saved[kEnds];
    variable_list out(5);
    std::vector<Sum> sums;
    Low back;
    const Low low{saved[kLow], saved[kLargest]};
    if (need[0] || need[2]) {
      const at::Tensor dx =
          adapter_product(dy, how, {saved[kMatrix], saved[kMatrixScale]}, saved[kDown], saved[kUp],
                          saved[kScale], factor, order, ends, true, need[2] ? &back : nullptr);
      if (need[0]) out[0] = shaped(dx, ctx->saved_data["sizes"].toIntVector());
      if (need[2]) sums.push_back({saved[kX], &back, false, {}});
    }
    if (need[3]) sums.push_back({dy, &low, true, {}});
    if (!sums.empty()) {
      adapter_gradients(sums, order, ends);
      for (const Sum& sum : sums) out[sum.turned ? 3 : 2] = sum.out;
    }
    if (need[1]) {
      const auto type = (at::ScalarType)s[3];
      Blocks columns, tokens{saved[kTokens], saved[kTokensScale]};
      quantize(dy, how, false, 0u, kColumns, nullptr, &columns);
      srs_blocks left{}, right{};
      check(operand("a", &columns, &left));
      check(operand("b", &tokens, &right));
      out[1] = at::empty({left.rows, right.rows}, dy.options().dtype(type));
      if (out[1].numel() != 0)
        check(g_matmul(&left, &right, dy.size(0), out[1].data_ptr(), format_of(type),
                       stream_of(dy)));
    }
    return out;
  }
};

// ------------------------------------------------------------------- module --

at::Tensor optional(PyObject* obj, const char* what) {
  return obj == Py_None ? at::Tensor() : tensor(obj, what);
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
  if (!bind_one(t, "srs_last_error", &g_last_error) ||
      !bind_one(t, "srs_group_rows", &g_group_rows) ||
      !bind_one(t, "srs_quantize_stack", &g_quantize_stack) ||
      !bind_one(t, "srs_quantize_groups", &g_quantize_groups) ||
      !bind_one(t, "srs_group_columns", &g_group_columns) ||
      !bind_one(t, "srs_group_scales", &g_group_scales) ||
      !bind_one(t, "srs_matmul_blocks", &g_matmul) ||
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
  const at::Tensor given = index.contiguous();
  const auto options = index.options().dtype(at::kInt);
  at::Tensor order = at::empty({index.numel()}, options), ends = at::empty({groups}, options);
  check(g_group_rows(given.data_ptr(), (int)index.element_size(), index.numel(), groups,
                     static_cast<int32_t*>(order.data_ptr()),
                     static_cast<int32_t*>(ends.data_ptr()), stream_of(index)));
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
  TORCH_CHECK_VALUE(x.dim() == 3, "a stack of matrices has three dimensions, got shape ",
                    x.sizes());
  Blocks straight, turned;
  quantize(x, {format, rule, seed}, square != 0, offset, orientation, &straight, &turned);
  if (orientation == kBoth)
    return wrap({straight.data, straight.scale, turned.data, turned.scale});
  const Blocks& one = orientation == kRows ? straight : turned;
  return wrap({one.data, one.scale});
  END_HANDLE_TH_ERRORS
}

// weight: the experts' matrices, or (with w_scale) their blocks.
PyObject* py_expert_linear(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *x_obj, *w_obj, *w_scale, *ends_obj;
  int format, grad_format, grad_rule;
  unsigned int seed;
  if (!PyArg_ParseTuple(args, "OOOOiiiI", &x_obj, &w_obj, &w_scale, &ends_obj, &format,
                        &grad_format, &grad_rule, &seed))
    return nullptr;
  const at::Tensor &x = tensor(x_obj, "x"), &weight = tensor(w_obj, "weight");
  const bool kept = w_scale != Py_None;
  refuse_tangents("expert_linear", {&x, &weight});
  TORCH_CHECK_VALUE(x.dim() == 2 && weight.dim() == 3 && x.size(1) == weight.size(2),
                    "x of shape ", x.sizes(), " does not fit expert weights of shape ",
                    weight.sizes());
  const at::Tensor& given = tensor(ends_obj, "ends");
  TORCH_CHECK_VALUE(given.dim() == 1 && given.size(0) == weight.size(0), "ends of shape ",
                    given.sizes(), " do not fit ", weight.size(0), " experts");
  TORCH_CHECK_VALUE(x.device() == weight.device(), "all tensors must be on the same CUDA device");
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  const int x_format = source_format(x, "expert_linear");
  if (!kept) source_format(weight, "expert_linear");
  const bool grad = at::GradMode::is_enabled();
  const bool need_x = grad && x.requires_grad(), need_w = grad && !kept && weight.requires_grad();
  at::Tensor ends;
  {
    c10::NoGradGuard no_grad;
    ends = checked_ends(given, x, "expert_linear");
  }
  if (need_x || need_w) {
    TORCH_CHECK_VALUE(!kept,
                      "a BlockTensor weight has no backward pass; pass the weight itself or run "
                      "under torch.no_grad()");
    return THPVariable_Wrap(ExpertLinear::apply(x, weight, ends, (int64_t)format,
                                                (int64_t)grad_format, (int64_t)grad_rule,
                                                (int64_t)seed, need_x, need_w));
  }
  c10::NoGradGuard no_grad;
  Blocks w{weight, kept ? tensor(w_scale, "the weight's scale") : at::Tensor()};
  if (!kept) quantize(weight, {format, SRS_RULE_NEAREST, 0u}, true, 0u, kRows, &w, nullptr);
  const srs_blocks matrix = stack_operand("weight", &w);
  const int64_t rows = x.size(0), k = x.size(1);
  const at::Tensor src = x.stride(1) != 1 && k > 1 ? x.contiguous() : x;
  at::Tensor out = at::empty({rows, weight.size(1)}, x.options());
  if (out.numel() != 0) {
    const int64_t bytes = g_linear_workspace(rows, k);
    const at::Tensor space = at::empty({bytes}, x.options().dtype(at::kByte));
    check(g_expert_linear(src.data_ptr(), x_format, rows, k, src.stride(0), format, &matrix,
                          (int)ends.numel(), ints(ends), out.data_ptr(), space.data_ptr(), bytes,
                          stream_of(x)));
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// weight: the projection's matrix, or None with its blocks (and those of its transpose).
PyObject* py_adapter_linear(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject *x_obj, *w_obj, *kept_obj, *kept_scale, *turned_obj, *turned_scale, *down_obj, *up_obj;
  PyObject *scale_obj, *order_obj, *ends_obj;
  double factor;
  int format, grad_format, grad_rule;
  unsigned int seed;
  if (!PyArg_ParseTuple(args, "OOOOOOOOOdOOiiiI", &x_obj, &w_obj, &kept_obj, &kept_scale,
                        &turned_obj, &turned_scale, &down_obj, &up_obj, &scale_obj, &factor,
                        &order_obj, &ends_obj, &format, &grad_format, &grad_rule, &seed))
    return nullptr;
  const at::Tensor &x = tensor(x_obj, "x"), &down = tensor(down_obj, "down");
  const at::Tensor& up = tensor(up_obj, "up");
  const at::Tensor weight = optional(w_obj, "weight"), scale = optional(scale_obj, "scale");
  const at::Tensor &order = tensor(order_obj, "order"), &ends = tensor(ends_obj, "ends");
  Blocks kept{optional(kept_obj, "the weight's data"), optional(kept_scale, "the weight's scale")};
  const Blocks turned{optional(turned_obj, "the transpose's data"),
                      optional(turned_scale, "the transpose's scale")};
  refuse_tangents("adapter_linear", {&x, &weight, &down, &up, &scale});
  const at::Tensor& matrix = weight.defined() ? weight : kept.data;
  TORCH_CHECK_VALUE(x.dim() > 0, "adapter_linear needs at least one dimension");
  TORCH_CHECK_VALUE(matrix.dim() == 2 && x.size(-1) == matrix.size(1), "x of shape ", x.sizes(),
                    " does not fit a weight of shape ", matrix.sizes());
  TORCH_CHECK_VALUE(x.device() == matrix.device(), "all tensors must be on the same CUDA device");
  if (turned.data.defined())
    TORCH_CHECK_VALUE(turned.data.dim() == 2 && turned.data.size(0) == matrix.size(1) &&
                          turned.data.size(1) == matrix.size(0),
                      "blocks of shapes ", matrix.sizes(), " and ", turned.data.sizes(),
                      " are not of a matrix and its transpose");
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  const bool grad = at::GradMode::is_enabled();
  const std::vector<int64_t> need{grad && x.requires_grad(),
                                  grad && weight.defined() && weight.requires_grad(),
                                  grad && down.requires_grad(), grad && up.requires_grad()};
  if (need[0] || need[1] || need[2] || need[3]) {
    TORCH_CHECK_VALUE(!need[0] || weight.defined() || turned.data.defined(),
                      "a BlockTensor weight has no backward pass; pass the blocks of both "
                      "orientations or the weight itself, or run under torch.no_grad()");
    AdapterInputs in{kept, turned, scale, {}, {}, factor, format, {grad_format, grad_rule, seed},
                     need};
    {
      c10::NoGradGuard no_grad;
      in.order = order.to(at::kInt);
      in.ends = checked_ends(ends, x, "adapter_linear");
    }
    return THPVariable_Wrap(AdapterLinear::apply(
        x, weight.defined() ? std::optional<at::Tensor>(weight) : std::nullopt, down, up, in));
  }
  c10::NoGradGuard no_grad;
  const Rounding nearest{format, SRS_RULE_NEAREST, 0u};
  if (weight.defined()) quantize(weight, nearest, true, 0u, kRows, &kept, nullptr);
  const at::Tensor y = adapter_product(flat(x), nearest, kept, down, up, scale, factor, order, ends,
                                       false, nullptr);
  return THPVariable_Wrap(shaped(y, x.sizes()));
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"bind", py_bind, METH_VARARGS, "bind({name: address}): the library's entry points."},
    {"group_rows", py_group_rows, METH_VARARGS, "group_rows(index, groups) -> order, ends."},
    {"quantize_stack", py_quantize_stack, METH_VARARGS,
     "quantize_stack(x, format, rule, square, seed, offset, orientation) -> tensors."},
    {"expert_linear", py_expert_linear, METH_VARARGS,
     "expert_linear(x, weight, w_scale, ends, format, grad_format, grad_rule, seed) -> tensor."},
    {"adapter_linear", py_adapter_linear, METH_VARARGS,
     "adapter_linear(x, weight, kept, kept_scale, turned, turned_scale, down, up, scale, factor, "
     "order, ends, format, grad_format, grad_rule, seed) -> tensor."},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_srs_groups",
                       "Tensor front end of the operators on rows in groups.", -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__srs_groups(void) { return PyModule_Create(&kModule); }
