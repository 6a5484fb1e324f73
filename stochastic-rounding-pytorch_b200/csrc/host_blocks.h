// What the tensor front ends of the FP8 block entry points share: blocks as tensors, their
// allocation and checks.  Included once by each module, which sets g_copy_rows.
#pragma once

#include <Python.h>

#include <cstdint>
#include <string>
#include <vector>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "srs_b200.h"

namespace {

constexpr int64_t kBlock = 128;

decltype(&srs_copy_rows) g_copy_rows = nullptr;

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

const at::Tensor& tensor(PyObject* obj, const char* what) {
  TORCH_CHECK_TYPE(THPVariable_Check(obj), what, " must be a tensor");
  return THPVariable_Unpack(obj);
}

// Nothing here has a rule for forward-mode differentiation: a tangent would be lost without a word.
void refuse_tangents(const char* what, std::initializer_list<const at::Tensor*> inputs) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const at::Tensor* t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), what,
                                " has no forward-mode derivative");
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

}  // namespace
