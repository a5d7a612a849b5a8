// xdna_train.lm.embedding: the scaled token lookup and its dense gradient
// (b2_embedding_fwd / b2_embedding_bwd).
#include <c10/cuda/CUDAGuard.h>

#include "lm.h"

namespace xdna {
namespace {

constexpr const char* kOp = "xdna embedding";

struct Dims {
  int64_t T, V, D;
};

Dims check(const at::Tensor& ids, const at::Tensor& weight) {
  const c10::Device dev = xdna_device(kOp, weight, "weight");
  check_device(kOp, ids, "ids", dev);
  TORCH_CHECK(index_code(ids.scalar_type()) >= 0, kOp, ": ids must be int32 or int64, not ", ids.scalar_type());
  TORCH_CHECK(float_code(weight.scalar_type()) >= 0, kOp, ": weight must be bfloat16 or float32, not ",
              weight.scalar_type());
  TORCH_CHECK(weight.dim() == 2, kOp, ": weight must be [vocabulary, width], it has ", weight.dim(), " dimensions");
  return {ids.numel(), weight.size(0), weight.size(1)};
}

at::Tensor forward_impl(const at::Tensor& ids_in, const at::Tensor& weight, double scale) {
  const Dims d = check(ids_in, weight);
  const c10::Device dev = weight.device();
  c10::cuda::CUDAGuard g(dev.index());
  std::vector<int64_t> sizes = ids_in.sizes().vec();
  sizes.push_back(d.D);
  at::Tensor y = empty(sizes, weight.scalar_type(), dev.index());
  if (y.numel() == 0) return y;
  materialize(ids_in);
  materialize(weight);
  const at::Tensor ids = ids_in.contiguous();
  const at::Tensor w = as_rows(weight, d.V, d.D);
  const cudaStream_t st = stream(dev.index());
  KernelTimer kt("lm.embedding", 2.0 * double(y.numel()) * double(y.element_size()), st);
  XDNA_B2(b2_embedding_fwd(ids.data_ptr(), index_code(ids.scalar_type()), d.T, w.data_ptr(), row_stride(w),
                           float_code(w.scalar_type()), d.V, d.D, float(scale), y.data_ptr(), st));
  count_launch("lm.embedding");
  return y;
}

at::Tensor backward_impl(const at::Tensor& ids_in, const at::Tensor& dy_in, int64_t V, int64_t D, double scale,
                         int64_t padding_idx) {
  const c10::Device dev = dy_in.device();
  c10::cuda::CUDAGuard g(dev.index());
  const int64_t T = ids_in.numel();
  at::Tensor dw = empty({V, D}, dy_in.scalar_type(), dev.index());
  if (dw.numel() == 0) return dw;
  materialize(ids_in);
  materialize(dy_in);
  const at::Tensor ids = ids_in.contiguous();
  const at::Tensor dy = as_rows(dy_in, T, D);
  const int64_t bytes = int64_t(b2_embedding_bwd_workspace_bytes(T, V, D));
  at::Tensor ws;  // few tokens need none
  if (bytes) ws = empty({bytes}, at::kByte, dev.index());
  const cudaStream_t st = stream(dev.index());
  KernelTimer kt("lm.embedding_bwd", double(dw.numel() + dy.numel()) * double(dw.element_size()), st);
  XDNA_B2(b2_embedding_bwd(ids.data_ptr(), index_code(ids.scalar_type()), T, dy.data_ptr(), row_stride(dy),
                           float_code(dy.scalar_type()), V, D, float(scale), padding_idx, dw.data_ptr(),
                           bytes ? ws.data_ptr() : nullptr, size_t(bytes), st));
  count_launch("lm.embedding_bwd");
  return dw;
}

class Embedding : public torch::autograd::Function<Embedding> {
 public:
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& weight, const at::Tensor& ids,
                            double scale, int64_t padding_idx) {
    ctx->save_for_backward({ids});
    ctx->saved_data["V"] = weight.size(0);
    ctx->saved_data["D"] = weight.size(1);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding_idx"] = padding_idx;
    return forward_impl(ids, weight, scale);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    no_double_backward(kOp);
    at::Tensor dw;
    if (grads[0].defined())
      dw = backward_impl(ctx->get_saved_variables()[0], grads[0], ctx->saved_data["V"].toInt(),
                         ctx->saved_data["D"].toInt(), ctx->saved_data["scale"].toDouble(),
                         ctx->saved_data["padding_idx"].toInt());
    return {dw, at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

at::Tensor embedding(const at::Tensor& ids, const at::Tensor& weight, double scale, int64_t padding_idx) {
  const Dims d = check(ids, weight);
  TORCH_CHECK(padding_idx >= -1 && padding_idx < std::max<int64_t>(d.V, 1), kOp, ": padding_idx ", padding_idx,
              " is outside the vocabulary of ", d.V);
  if (at::GradMode::is_enabled() && weight.requires_grad())
    return Embedding::apply(weight, ids, scale, padding_idx);
  return forward_impl(ids, weight, scale);
}

}  // namespace

void bind_embedding(pybind11::module_& m) {
  m.def("lm_embedding", &embedding, pybind11::call_guard<pybind11::gil_scoped_release>());
}

}  // namespace xdna
