"""The plain CPU path of xdna_train.lm against the definitions, and the C
ABI's argument checks that need no GPU."""
import math

import pytest
import torch

from xdna_train import _abi, lm


def test_embedding_on_cpu():
    w = torch.randn(7, 5, requires_grad=True)
    ids = torch.tensor([[1, 6], [1, 0]])
    y = lm.embedding(ids, w, scale=3.0, padding_idx=0)
    assert torch.equal(y, 3.0 * w[ids])
    (dw,) = torch.autograd.grad(y.sum(), [w])
    assert torch.equal(dw[:, 0], torch.tensor([0.0, 6, 0, 0, 0, 0, 3]))
    with pytest.raises(ValueError, match="padding_idx"):
        lm.embedding(ids, w, padding_idx=7)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_distill_loss_on_cpu(reduction):
    g = torch.Generator().manual_seed(0)
    z = torch.randn(4, 9, generator=g, requires_grad=True)
    t = torch.randn(4, 3, generator=g)
    ids = torch.tensor([[0, 4, 8], [1, -1, 2], [-1, -1, -1], [3, 3, 5]])
    w = torch.tensor([1.0, 0.5, 1.0, 2.0])
    tau = 2.0
    loss = lm.distill_loss(z, t, ids, tau, w, reduction)
    rows = []
    for r in range(4):
        kept = [k for k in range(3) if ids[r, k] >= 0]
        p = torch.softmax(t[r, kept] / tau, 0)
        logq = torch.log_softmax(z[r] / tau, 0)
        rows.append(w[r] * tau ** 2 * sum(p[i] * (p[i].log() - logq[ids[r, k]]) for i, k in enumerate(kept)))
    rows = torch.stack([torch.as_tensor(r, dtype=torch.float32) for r in rows])
    ref = {"mean": rows.sum() / w.sum(), "sum": rows.sum(), "none": rows}[reduction]
    assert torch.allclose(loss, ref, rtol=1e-5, atol=1e-6)
    (a,) = torch.autograd.grad(loss.sum(), [z], retain_graph=True)
    (b,) = torch.autograd.grad(ref.sum(), [z])
    assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)


def test_distill_loss_masks_on_cpu():
    z = torch.randn(3, 6)
    z[1] = math.nan
    z[2, 4:] = -math.inf
    z.requires_grad_()
    loss = lm.distill_loss(z, torch.zeros(3, 2), torch.tensor([[0, 1], [0, 1], [2, 3]]),
                           row_weight=torch.tensor([1.0, 0.0, 1.0]))
    (dz,) = torch.autograd.grad(loss, [z])
    assert loss.isfinite() and dz.isfinite().all() and not dz[1].any()


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_gated_mlp_on_cpu(act):
    g = torch.Generator().manual_seed(1)
    x, wg, wu, wd = (torch.randn(*s, generator=g) for s in ((2, 3, 5), (7, 5), (7, 5), (4, 7)))
    fn = getattr(torch.nn.functional, act)
    assert torch.allclose(lm.gated_mlp(x, wg, wu, wd, act), (fn(x @ wg.t()) * (x @ wu.t())) @ wd.t(), atol=1e-5)
    with pytest.raises(ValueError, match="activation"):
        lm.gated_mlp(x, wg, wu, wd, "tanh")


def test_argument_errors_need_no_gpu():
    L = _abi.lib()
    assert L.b2_gated_mlp_fwd_bf16(8, 16, 8, 16, 8, 16, 8, 24, 3, 8, 8, None, 4, 16, 24, 8, 8, 0, None) == 1
    assert b"activation" in L.b2_last_error()
    assert L.b2_gated_mlp_fwd_bf16(8, 15, 8, 16, 8, 16, 8, 24, 0, 8, 8, None, 4, 16, 24, 8, 8, 0, None) == 1
    assert b"row stride" in L.b2_last_error()
    assert L.b2_gated_mlp_fwd_bf16(256, 16, 8, 16, 8, 16, 8, 24, 0, 8, 8, None, 4, 16, 24, 8, 256, 0, None) == 5
    assert L.b2_gated_mlp_bwd_bf16(8, 8, 8, 16, 8, 16, 8, 16, 8, 24, 0, None, 8, 8, 8, 8, 4, 16, 24, 8, 8, 0, None) == 1
    assert b"null pointer" in L.b2_last_error()
    assert L.b2_embedding_fwd(None, _abi.B2_I64, 3, None, 8, _abi.B2_F32, 5, 8, 1.0, None, None) == 1
    assert b"null pointer" in L.b2_last_error()
    assert L.b2_embedding_fwd(8, _abi.B2_F32, 3, 8, 8, _abi.B2_F32, 5, 8, 1.0, 8, None) == 1
    assert b"int32 or int64" in L.b2_last_error()
    assert L.b2_embedding_bwd(8, _abi.B2_I64, 3, 8, 7, _abi.B2_F32, 5, 8, 1.0, -1, 8, 8, 0, None) == 1
    assert b"bad shape" in L.b2_last_error()
    assert L.b2_embedding_fwd(8, _abi.B2_I64, 1 << 31, 8, 8, _abi.B2_F32, 5, 8, 1.0, 8, None) == 3
    args = [8, 50, _abi.B2_F32, 3, 50, 8, 4, _abi.B2_F32, 8, 4, _abi.B2_I64, 4, 1.0, None, 0, 8, 8, None, 50, 8, 0, None]
    assert L.b2_distill_loss_fwd(*args) == 5 and b"workspace" in L.b2_last_error()
    assert L.b2_distill_loss_fwd(*args[:12], -1.0, *args[13:]) == 1 and b"temperature" in L.b2_last_error()
    assert L.b2_distill_loss_fwd(*args[:11], 1025, *args[12:]) == 3 and b"1024" in L.b2_last_error()


def test_wait_limit_is_checked():
    L = _abi.lib()
    assert L.b2_distill_set_wait_limit(-1) == 1 and b"negative" in L.b2_last_error()
    assert L.b2_distill_set_wait_limit(0) == 0


def test_distill_loss_keeps_a_teachers_nan_on_cpu():
    # as on the device: a NaN teacher logit makes its row's loss NaN, unless the entry is absent or the row masked
    z = torch.randn(4, 6)
    t = torch.zeros(4, 3)
    t[:3, 1] = math.nan
    ids = torch.tensor([[0, 1, 2], [3, -1, 4], [0, 1, 2], [0, 1, 2]])
    loss = lm.distill_loss(z, t, ids, row_weight=torch.tensor([1.0, 1.0, 0.0, 1.0]), reduction="none")
    assert loss.isnan().tolist() == [True, False, False, False] and loss[2] == 0
    t[0] = math.nan
    assert lm.distill_loss(z, t, ids, reduction="none").isnan().tolist() == [True, False, True, False]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_embedding_sums_in_fp32_on_cpu(dtype):
    # as on the device: the gradient of a frequent id is rounded once, not after every token (bf16 sums stop at 256)
    w = torch.randn(4, 3).to(dtype).requires_grad_()
    ids = torch.tensor([1] * 1000 + [2] * 3 + [0])
    y = lm.embedding(ids, w, scale=3.0, padding_idx=0)
    assert y.dtype == dtype and torch.equal(y, (3.0 * w.detach().float()).to(dtype)[ids])
    (dw,) = torch.autograd.grad(y, [w], torch.ones_like(y))
    assert dw.dtype == dtype and dw[:, 0].tolist() == [0.0, 3000.0 if dtype == torch.float32 else 3008.0, 9.0, 0.0]


def test_embedding_of_doubles_on_cpu():
    w = torch.randn(5, 3, dtype=torch.float64, requires_grad=True)
    ids = torch.tensor([4, 0, 4])
    assert torch.autograd.gradcheck(lambda t: lm.embedding(ids, t, scale=1.7), [w])
