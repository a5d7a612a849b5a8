// xdna_train.lm.distill_loss: the distillation loss from a teacher's top
// logits (b2_distill_loss_fwd / b2_distill_loss_bwd).
//
// With a gradient wanted the forward pass writes it too, for an upstream
// gradient of 1, while it holds each row on chip; the backward hands that
// tensor out after b2_distill_loss_bwd has rewritten the rows whose upstream
// gradient turned out to be another.  A second backward through the same graph
// computes the gradient into a tensor of its own.
#include <c10/cuda/CUDAGuard.h>

#include "lm.h"

namespace xdna {
namespace {

constexpr const char* kOp = "xdna distill_loss";

struct Call {
  at::Tensor z, t, ids, weight;  // [N][V], [N][K], [N][K], [N] or undefined
  double tau;
  int64_t reduction;
};

// The arguments checked and brought to rows (a copy only where strides need one).
Call check(const at::Tensor& logits, const at::Tensor& teacher, const at::Tensor& ids,
           const std::optional<at::Tensor>& weight, double tau, int64_t reduction) {
  const c10::Device dev = xdna_device(kOp, logits, "logits");
  check_device(kOp, teacher, "teacher_logits", dev);
  check_device(kOp, ids, "teacher_ids", dev);
  TORCH_CHECK(float_code(logits.scalar_type()) >= 0, kOp, ": logits must be bfloat16 or float32, not ",
              logits.scalar_type());
  TORCH_CHECK(float_code(teacher.scalar_type()) >= 0, kOp, ": teacher_logits must be bfloat16 or float32, not ",
              teacher.scalar_type());
  TORCH_CHECK(index_code(ids.scalar_type()) >= 0, kOp, ": teacher_ids must be int32 or int64, not ",
              ids.scalar_type());
  TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) > 0, kOp, ": logits must be [..., vocabulary]");
  TORCH_CHECK(teacher.sizes() == ids.sizes(), kOp, ": teacher_logits ", teacher.sizes(), " and teacher_ids ",
              ids.sizes(), " must have one shape");
  TORCH_CHECK(teacher.dim() == logits.dim() &&
                  teacher.sizes().slice(0, teacher.dim() - 1) == logits.sizes().slice(0, logits.dim() - 1),
              kOp, ": teacher_logits ", teacher.sizes(), " must have the rows of logits ", logits.sizes());
  TORCH_CHECK(tau > 0 && std::isfinite(tau), kOp, ": temperature must be positive, not ", tau);
  const int64_t V = logits.size(-1), K = teacher.size(-1), N = logits.numel() / V;
  Call c{as_rows(logits, N, V), as_rows(teacher, N, K), as_rows(ids, N, K), at::Tensor(), tau,
         reduction};
  if (weight.has_value() && weight->defined()) {
    check_device(kOp, *weight, "row_weight", dev);
    TORCH_CHECK(weight->scalar_type() == at::kFloat, kOp, ": row_weight must be float32, not ", weight->scalar_type());
    TORCH_CHECK(weight->sizes() == logits.sizes().slice(0, logits.dim() - 1), kOp, ": row_weight ", weight->sizes(),
                " must have one value for each row of logits ", logits.sizes());
    at::NoGradGuard no_grad;
    c.weight = weight->dim() == 1 && weight->is_contiguous() ? *weight : weight->reshape({N}).contiguous();
  }
  for (const at::Tensor* t : {&c.z, &c.t, &c.ids, &c.weight})
    if (t->defined()) materialize(*t);
  return c;
}

// A gradient tensor for z: z's own row stride where that is not much wider
// than a row, so that both have their 16-byte vectors at the same elements
// (and a padded head's gradient keeps the padding its GEMMs want).
at::Tensor empty_grad(const at::Tensor& z) {
  const int64_t N = z.size(0), V = z.size(1), ld = row_stride(z);
  if (ld <= V || ld > V + V / 8 + 64) return empty({N, V}, z.scalar_type(), z.device().index());
  return empty({N, ld}, z.scalar_type(), z.device().index()).narrow(1, 0, V);
}

std::vector<int64_t> loss_sizes(const at::Tensor& logits, int64_t reduction) {
  if (reduction != 2) return {};
  return logits.sizes().slice(0, logits.dim() - 1).vec();
}

// the loss, and the buffer whose last 2N + 1 values are its statistics; dz may be undefined
std::pair<at::Tensor, at::Tensor> run_fwd(const Call& c, at::IntArrayRef loss_shape, const at::Tensor& dz) {
  const c10::Device dev = c.z.device();
  c10::cuda::CUDAGuard g(dev.index());
  const int64_t N = c.z.size(0), V = c.z.size(1), K = c.t.size(1);
  at::Tensor loss = empty(loss_shape, at::kFloat, dev.index());
  // one allocation: the workspace, then what the backward needs
  const int64_t scratch = (int64_t(b2_distill_workspace_bytes(N)) + 15) / 16 * 4;
  at::Tensor stats = empty({scratch + 2 * N + 1}, at::kFloat, dev.index());
  const cudaStream_t st = stream(dev.index());
  KernelTimer kt("lm.distill", double(N) * double(V) * double(c.z.element_size()) * (dz.defined() ? 2.0 : 1.0), st);
  XDNA_B2(b2_distill_loss_fwd(c.z.data_ptr(), row_stride(c.z), float_code(c.z.scalar_type()), N, V, c.t.data_ptr(),
                              row_stride(c.t), float_code(c.t.scalar_type()), c.ids.data_ptr(), row_stride(c.ids),
                              index_code(c.ids.scalar_type()), K, float(c.tau),
                              c.weight.defined() ? c.weight.data_ptr<float>() : nullptr, int(c.reduction),
                              loss.data_ptr<float>(), stats.data_ptr<float>() + scratch,
                              dz.defined() ? dz.data_ptr() : nullptr, dz.defined() ? row_stride(dz) : V,
                              stats.data_ptr(), size_t(scratch) * 4, st));
  count_launch("lm.distill");
  return {loss, stats};
}

class Distill : public torch::autograd::Function<Distill> {
 public:
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& teacher,
                            const at::Tensor& ids, const std::optional<at::Tensor>& weight, double tau,
                            int64_t reduction) {
    const Call c = check(logits, teacher, ids, weight, tau, reduction);
    at::Tensor dz = empty_grad(c.z);
    auto [loss, stats] = run_fwd(c, loss_sizes(logits, reduction), dz);
    ctx->save_for_backward({logits, teacher, ids, weight.has_value() ? *weight : at::Tensor()});
    ctx->saved_data["stats"] = stats;
    ctx->saved_data["dz"] = dz;
    ctx->saved_data["tau"] = tau;
    ctx->saved_data["reduction"] = reduction;
    return loss;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    no_double_backward(kOp);
    at::Tensor out;
    if (grads[0].defined()) {
      const auto saved = ctx->get_saved_variables();
      const std::optional<at::Tensor> w =
          saved[3].defined() ? std::optional<at::Tensor>(saved[3]) : std::nullopt;
      const Call c = check(saved[0], saved[1], saved[2], w, ctx->saved_data["tau"].toDouble(),
                           ctx->saved_data["reduction"].toInt());
      const at::Tensor stats = ctx->saved_data["stats"].toTensor();
      const c10::Device dev = c.z.device();
      c10::cuda::CUDAGuard g(dev.index());
      at::Tensor dz;
      auto held = ctx->saved_data.find("dz");
      const bool first = held != ctx->saved_data.end();
      if (first) {
        dz = held->second.toTensor();
        ctx->saved_data.erase(held);
      } else {
        dz = empty_grad(c.z);
      }
      const int64_t N = c.z.size(0), V = c.z.size(1), K = c.t.size(1);
      materialize(grads[0]);
      const at::Tensor up = grads[0].contiguous();
      const cudaStream_t st = stream(dev.index());
      XDNA_B2(b2_distill_loss_bwd(c.z.data_ptr(), row_stride(c.z), float_code(c.z.scalar_type()), N, V,
                                  c.t.data_ptr(), row_stride(c.t), float_code(c.t.scalar_type()), c.ids.data_ptr(),
                                  row_stride(c.ids), index_code(c.ids.scalar_type()), K, float(c.tau),
                                  c.weight.defined() ? c.weight.data_ptr<float>() : nullptr, int(c.reduction),
                                  stats.data_ptr<float>() + (stats.numel() - (2 * N + 1)), up.data_ptr<float>(), first ? 1 : 0, dz.data_ptr(),
                                  row_stride(dz), st));
      count_launch("lm.distill_bwd");
      out = dz.sizes() == saved[0].sizes() ? dz : dz.reshape(saved[0].sizes());
    }
    return {out, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

at::Tensor distill_loss(const at::Tensor& logits, const at::Tensor& teacher, const at::Tensor& ids, double tau,
                        const std::optional<at::Tensor>& weight, int64_t reduction) {
  // (the refusals below need grad mode, which is off inside apply)
  if (at::GradMode::is_enabled()) {
    TORCH_CHECK(!teacher.requires_grad(), kOp, ": teacher_logits are constants of the loss; detach() them");
    TORCH_CHECK(!weight.has_value() || !weight->requires_grad(), kOp,
                ": row_weight is a constant of the loss; detach() it");
    if (logits.requires_grad()) return Distill::apply(logits, teacher, ids, weight, tau, reduction);
  }
  const Call c = check(logits, teacher, ids, weight, tau, reduction);
  return run_fwd(c, loss_sizes(logits, reduction), at::Tensor()).first;
}

}  // namespace

void bind_distill(pybind11::module_& m) {
  m.def("lm_distill_loss", &distill_loss, pybind11::call_guard<pybind11::gil_scoped_release>());
}

}  // namespace xdna
