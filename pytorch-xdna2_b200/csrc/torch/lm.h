// Shared by the language-model operators (xdna_train.lm): argument checks, row
// views and their bindings.
#pragma once

#include <torch/extension.h>

#include "xdna.h"

namespace xdna {

inline void check_device(const char* op, const at::Tensor& t, const char* what, c10::Device device) {
  TORCH_CHECK(t.defined() && t.device() == device, op, ": ", what, " must be on ", device, " like the other tensors",
              t.defined() ? ", it is on " : "", t.defined() ? t.device().str() : std::string());
}

inline c10::Device xdna_device(const char* op, const at::Tensor& t, const char* what) {
  TORCH_CHECK(t.device().type() == kXdna, op, ": ", what, " must be an xdna tensor, it is on ", t.device());
  return t.device();
}

inline int float_code(at::ScalarType t) { return t == at::kBFloat16 ? B2_BF16 : t == at::kFloat ? B2_F32 : -1; }
inline int index_code(at::ScalarType t) { return t == at::kInt ? B2_I32 : t == at::kLong ? B2_I64 : -1; }

// t as [rows][cols] with contiguous columns and rows that do not overlap: t
// itself where it is that already (no view is made: these run once or more per
// operand and call), a view where its strides allow one, else a copy.
inline bool rows_ok(const at::Tensor& m, int64_t rows, int64_t cols) {
  return (cols <= 1 || m.stride(1) == 1) && (rows <= 1 || m.stride(0) >= cols);
}
inline at::Tensor as_rows(const at::Tensor& t, int64_t rows, int64_t cols) {
  if (t.dim() == 2 && rows_ok(t, rows, cols)) return t;
  at::NoGradGuard no_grad;
  at::Tensor m = t.reshape({rows, cols});
  return rows_ok(m, rows, cols) ? m : m.contiguous();
}
inline int64_t row_stride(const at::Tensor& m) { return m.size(0) > 1 ? m.stride(0) : std::max<int64_t>(m.size(1), 1); }

inline void no_double_backward(const char* op) {
  TORCH_CHECK(!at::GradMode::is_enabled(), op, ": its backward is not differentiable (create_graph=True)");
}

void bind_embedding(pybind11::module_& m);  // embed_ops.cpp
void bind_distill(pybind11::module_& m);    // distill_ops.cpp
void bind_gated(pybind11::module_& m);      // gated_ops.cpp

}  // namespace xdna
