// xdna_train.lm.gated_mlp: the gated feed-forward block
// (b2_gated_mlp_fwd_bf16 / b2_gated_mlp_bwd_bf16).
#include <c10/cuda/CUDAGuard.h>

#include "lm.h"

namespace xdna {
namespace {

constexpr const char* kOp = "xdna gated_mlp";

struct Call {
  at::Tensor x, wg, wu, wd;  // [M][D], [F][D], [F][D], [E][F] with contiguous columns
  int64_t M, D, F, E;
};

Call check(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd) {
  const c10::Device dev = xdna_device(kOp, x, "x");
  const std::pair<const at::Tensor*, const char*> weights[] = {{&wg, "w_gate"}, {&wu, "w_up"}, {&wd, "w_down"}};
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, kOp, ": x must be [..., width]");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16, kOp, ": x must be bfloat16, not ", x.scalar_type());
  for (const auto& [t, what] : weights) {
    check_device(kOp, *t, what, dev);
    TORCH_CHECK(t->scalar_type() == at::kBFloat16, kOp, ": ", what, " must be bfloat16, not ", t->scalar_type());
    TORCH_CHECK(t->dim() == 2 && t->numel() > 0, kOp, ": ", what, " must be a matrix, it is ", t->sizes());
  }
  Call c;
  c.D = x.size(-1);
  c.M = x.numel() / c.D;
  c.F = wg.size(0);
  c.E = wd.size(0);
  TORCH_CHECK(wg.size(1) == c.D && wu.sizes() == wg.sizes() && wd.size(1) == c.F, kOp, ": x ", x.sizes(), ", w_gate ",
              wg.sizes(), ", w_up ", wu.sizes(), " and w_down ", wd.sizes(),
              " do not fit: [..., D], [F, D], [F, D] and [E, F] are wanted");
  for (const at::Tensor* t : {&x, &wg, &wu, &wd}) materialize(*t);
  c.x = as_rows(x, c.M, c.D);
  c.wg = as_rows(wg, c.F, c.D);
  c.wu = as_rows(wu, c.F, c.D);
  c.wd = as_rows(wd, c.E, c.F);
  return c;
}

int64_t saved_width(int64_t F) { return 4 * ((F + 7) / 8 * 8); }

// kept: room for what the backward needs; may be undefined
at::Tensor run_fwd(const Call& c, at::IntArrayRef x_sizes, int64_t act, const at::Tensor& kept) {
  const c10::Device dev = c.x.device();
  c10::cuda::CUDAGuard g(dev.index());
  std::vector<int64_t> sizes = x_sizes.vec();
  sizes.back() = c.E;
  at::Tensor y = empty(sizes, at::kBFloat16, dev.index());
  if (c.M == 0) return y;
  const int64_t bytes = int64_t(b2_gated_mlp_fwd_workspace_bytes(c.M, c.D, c.F, c.E));
  at::Tensor ws = empty({bytes}, at::kByte, dev.index());
  const cudaStream_t st = stream(dev.index());
  KernelTimer kt("lm.gated_mlp", 2.0 * double(c.M) * double(c.F) * (2.0 * double(c.D) + double(c.E)), st);
  XDNA_B2(b2_gated_mlp_fwd_bf16(c.x.data_ptr(), row_stride(c.x), c.wg.data_ptr(), row_stride(c.wg), c.wu.data_ptr(),
                                row_stride(c.wu), c.wd.data_ptr(), row_stride(c.wd), int(act), y.data_ptr(), c.E,
                                kept.defined() ? kept.data_ptr() : nullptr, c.M, c.D, c.F, c.E, ws.data_ptr(),
                                size_t(bytes), st));
  count_launch("lm.gated_mlp");
  return y;
}

class GatedMlp : public torch::autograd::Function<GatedMlp> {
 public:
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& wg,
                            const at::Tensor& wu, const at::Tensor& wd, int64_t act) {
    const Call c = check(x, wg, wu, wd);
    at::Tensor kept = empty({c.M, saved_width(c.F)}, at::kBFloat16, x.device().index());
    ctx->save_for_backward({x, wg, wu, wd, kept});  // released, and seen by hooks, like any saved tensor
    ctx->saved_data["act"] = act;
    return run_fwd(c, x.sizes(), act, kept);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    no_double_backward(kOp);
    torch::autograd::variable_list out(5);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Call c = check(saved[0], saved[1], saved[2], saved[3]);
    const at::Tensor kept = saved[4].contiguous();  // (a hook may have moved it)
    const c10::Device dev = c.x.device();
    c10::cuda::CUDAGuard g(dev.index());
    materialize(grads[0]);
    const at::Tensor dy = as_rows(grads[0], c.M, c.E);
    const int64_t sizes[4][2] = {{c.M, c.D}, {c.F, c.D}, {c.F, c.D}, {c.E, c.F}};
    void* ptr[4] = {};
    for (int i = 0; i < 4; ++i) {
      if (!ctx->needs_input_grad(i)) continue;
      out[i] = i == 0 ? empty(saved[0].sizes(), at::kBFloat16, dev.index())
                      : empty({sizes[i][0], sizes[i][1]}, at::kBFloat16, dev.index());
      ptr[i] = out[i].data_ptr();
    }
    const int64_t bytes = int64_t(b2_gated_mlp_bwd_workspace_bytes(c.M, c.D, c.F, c.E));
    at::Tensor ws = empty({std::max<int64_t>(bytes, 16)}, at::kByte, dev.index());
    const cudaStream_t st = stream(dev.index());
    KernelTimer kt("lm.gated_mlp_bwd", 4.0 * double(c.M) * double(c.F) * (2.0 * double(c.D) + double(c.E)), st);
    XDNA_B2(b2_gated_mlp_bwd_bf16(dy.data_ptr(), row_stride(dy), c.x.data_ptr(), row_stride(c.x), c.wg.data_ptr(),
                                  row_stride(c.wg), c.wu.data_ptr(), row_stride(c.wu), c.wd.data_ptr(),
                                  row_stride(c.wd), int(ctx->saved_data["act"].toInt()), kept.data_ptr(), ptr[0], ptr[1],
                                  ptr[2], ptr[3], c.M, c.D, c.F, c.E, ws.data_ptr(), size_t(bytes), st));
    count_launch("lm.gated_mlp_bwd");
    return out;
  }
};

at::Tensor gated_mlp(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd,
                     int64_t act) {
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || wg.requires_grad() || wu.requires_grad() || wd.requires_grad()))
    return GatedMlp::apply(x, wg, wu, wd, act);
  return run_fwd(check(x, wg, wu, wd), x.sizes(), act, at::Tensor());
}

}  // namespace

void bind_gated(pybind11::module_& m) {
  m.def("lm_gated_mlp", &gated_mlp, pybind11::call_guard<pybind11::gil_scoped_release>());
}

}  // namespace xdna
