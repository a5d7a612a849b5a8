"""xdna_train.lm.embedding (b2_embedding_fwd / b2_embedding_bwd) against the
definition in fp64.

Bounds.  The lookup rounds scale * w once in fp32 and once to the weight's
type: |err| <= (2^-8 for bf16, 2^-22 for fp32) * |y|.  A gradient row of n
tokens is an fp32 sum, |err| <= n * 2^-24 * sum |dy| (any order), then scaled
and rounded once."""
import pytest
import torch

import xdna_train
from xdna_train import _abi, lm

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev(cuda):
    return torch.device("xdna", 0)

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -22}


def _ids(kind, T, V, g):
    if kind == "uniform":
        return torch.randint(0, V, (T,), generator=g)
    if kind == "zipf":
        return (torch.exp(torch.rand(T, generator=g).double() * torch.log(torch.tensor(V + 1.0))) - 1).long().clamp(0, V - 1)
    if kind == "one":
        return torch.full((T,), V // 2)
    return torch.arange(T).flip(0) % V  # falling


def _check(ids, w, scale, pad, dev, dy=None, ids_dtype=torch.int64):
    V, D = w.shape
    T = ids.numel()
    wd = w.to(dev).requires_grad_()
    y = lm.embedding(ids.to(ids_dtype).to(dev), wd, scale=scale, padding_idx=pad)
    ref = w.double()[ids.reshape(-1)] * scale
    got = y.detach().double().cpu().reshape(T, D)
    assert y.shape == ids.shape + (D,) and y.dtype == w.dtype
    assert ((got - ref).abs() <= UNIT[w.dtype] * ref.abs()).all()
    dy = torch.randn(T, D).to(w.dtype) if dy is None else dy
    (dw,) = torch.autograd.grad(y, [wd], dy.to(dev).reshape(y.shape))
    flat = ids.reshape(-1)
    keep = torch.ones(T, dtype=torch.bool) if pad is None else flat != pad
    ref = torch.zeros(V, D, dtype=torch.float64).index_add_(0, flat[keep], dy.double().reshape(T, D)[keep])
    mag = torch.zeros(V, D, dtype=torch.float64).index_add_(0, flat[keep], dy.double().abs().reshape(T, D)[keep])
    n = torch.bincount(flat[keep], minlength=V).unsqueeze(1)
    bound = abs(scale) * n * 2.0 ** -24 * mag + UNIT[w.dtype] * (ref * scale).abs()
    err = (dw.double().cpu() - ref * scale).abs()
    assert dw.shape == w.shape and dw.dtype == w.dtype
    assert (err <= bound).all(), (err - bound).max()
    return y, dw


CASES = [
    # tokens, vocabulary, width
    (1, 1, 1), (1, 5, 8), (2, 3, 7), (31, 40, 16), (33, 40, 33), (64, 7, 9), (257, 1000, 130), (1024, 513, 64),
    (512, 300, 40), (513, 300, 40), (500, 90000, 264), (1025, 511, 72), (4096, 700, 12), (2500, 262145, 12), (4097, 3000, 40), (8192, 20000, 24), (8193, 30000, 24), (20011, 100, 18),
    (300000, 50000, 4), (700, 300, 2056), (70, 5000, 3001),
]


@pytest.mark.parametrize("T,V,D", CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["uniform", "zipf", "one", "falling"])
def test_lookup_and_gradient(dev, T, V, D, dtype, kind):
    g = torch.Generator().manual_seed(T + V)
    w = torch.randn(V, D, generator=g).to(dtype)
    dy = torch.randn(T, D, generator=g).to(dtype)
    _check(_ids(kind, T, V, g), w, 1.7, V - 1 if kind == "zipf" and V > 1 else None, dev, dy)


@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
def test_id_types_and_shapes(dev, ids_dtype):
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, 100, (4, 9), generator=g)
    _check(ids, torch.randn(100, 48, generator=g).bfloat16(), 3.0, 7, dev, ids_dtype=ids_dtype)
    assert xdna_train.kernel_stats().get("lm.embedding_bwd", 0) > 0


def test_strided_and_misaligned_inputs(dev):
    g = torch.Generator().manual_seed(4)
    base = torch.randn(50, 70, generator=g).bfloat16().to(dev)
    ids = torch.randint(0, 50, (33, 2), generator=g).to(dev)[:, 0]  # strided ids
    for lo, hi in ((0, 64), (1, 64), (2, 66), (8, 40)):
        w = base[:, lo:hi]
        assert torch.equal(lm.embedding(ids, w), w[ids])
    wt = torch.randn(48, 50, generator=g).to(dev).t()  # columns not contiguous
    assert torch.equal(lm.embedding(ids, wt), wt[ids])
    w = torch.zeros(50, 64, dtype=torch.bfloat16, device=dev, requires_grad=True)
    big = torch.randn(33, 70, generator=g).bfloat16().to(dev)
    for dy in (big[:, 3:67], big[:, 6:70], big[:, :1].expand(33, 64)):
        (dw,) = torch.autograd.grad(lm.embedding(ids, w), [w], dy)
        ref = torch.zeros(50, 64, device=dev, dtype=torch.float64).index_add_(0, ids, dy.double())
        mag = torch.zeros(50, 64, device=dev, dtype=torch.float64).index_add_(0, ids, dy.double().abs())
        assert ((dw.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 33 * 2.0 ** -24 * mag).all()


def test_empty_inputs(dev):
    w = torch.randn(5, 8, device=dev, requires_grad=True)
    y = lm.embedding(torch.empty(0, 3, dtype=torch.int64, device=dev), w)
    assert y.shape == (0, 3, 8)
    (dw,) = torch.autograd.grad(y, [w], torch.empty(0, 3, 8, device=dev))
    assert torch.equal(dw, torch.zeros_like(w))
    assert lm.embedding(torch.zeros(4, dtype=torch.int64, device=dev), torch.empty(3, 0, device=dev)).shape == (4, 0)


def test_ids_outside_the_vocabulary_are_reported(dev):
    xdna_train.device_status(0)
    w = torch.randn(6, 8, device=dev, requires_grad=True)
    ids = torch.tensor([1, 6, -1, -2, 2], device=dev)
    y = lm.embedding(ids, w)
    assert y[[1, 2, 3]].isnan().all() and torch.equal(y[[0, 4]], w[[1, 2]])
    (dw,) = torch.autograd.grad(y, [w], torch.ones(5, 8, device=dev))
    assert torch.equal(dw.sum(1).cpu(), torch.tensor([0.0, 8, 8, 0, 0, 0]))
    assert xdna_train.device_status(0) == 1
    assert xdna_train.device_status(0) == 0


def test_gradient_is_the_same_on_every_run_and_stream(dev):
    g = torch.Generator().manual_seed(5)
    ids = _ids("zipf", 30000, 5000, g).to(dev)
    w = torch.randn(5000, 96, generator=g).to(dev).requires_grad_()
    dy = torch.randn(30000, 96, generator=g).to(dev)
    first = torch.autograd.grad(lm.embedding(ids, w), [w], dy)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [torch.autograd.grad(lm.embedding(ids, w), [w], dy)[0] for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(first, a) for a in again)


def test_gradient_against_differences(dev):
    # the lookup is linear in the weight: a difference quotient of any step is exact up to rounding
    g = torch.Generator().manual_seed(6)
    ids = torch.randint(0, 20, (50,), generator=g).to(dev)
    w = torch.randn(20, 12, generator=g).to(dev).requires_grad_()
    c, d = torch.randn(50, 12, generator=g).to(dev), torch.randn(20, 12, generator=g).to(dev)
    (dw,) = torch.autograd.grad(lm.embedding(ids, w, scale=2.5), [w], c)
    f = lambda e: (lm.embedding(ids, (w + e * d).detach(), scale=2.5).double() * c.double()).sum()  # noqa: E731
    quotient = (f(0.5) - f(-0.5)).item()
    # 600 products, each off by at most 2^-22 of its size (two fp32 roundings of w + e d and of the product)
    bound = 600 * 2.0 ** -22 * 2.5 * (c.abs().max() * (w.abs().max() + d.abs().max())).item()
    assert abs(quotient - (dw.double() * d.double()).sum().item()) <= 2 * bound


def test_refusals(dev):
    w, ids = torch.randn(5, 8, device=dev), torch.zeros(3, dtype=torch.int64, device=dev)
    for bad in (lambda: lm.embedding(ids.float(), w), lambda: lm.embedding(ids, w.half()),
                lambda: lm.embedding(ids, w[0]), lambda: lm.embedding(ids.cpu(), w),
                lambda: lm.embedding(ids, xdna_train.as_cuda(w))):
        with pytest.raises(RuntimeError, match="xdna embedding"):
            bad()
    with pytest.raises(ValueError, match="padding_idx"):
        lm.embedding(ids, w, padding_idx=5)
    wg = w.clone().requires_grad_()
    dy = torch.ones(3, 8, device=dev, requires_grad=True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(lm.embedding(ids, wg), [wg], dy, create_graph=True)
    need = _abi.lib().b2_embedding_bwd_workspace_bytes(3000, 5, 8)
    st = _abi.lib().b2_embedding_bwd(ids.data_ptr(), _abi.B2_I64, 3000, w.data_ptr(), 8, _abi.B2_F32, 5, 8, 1.0, -1,
                                     w.data_ptr(), w.data_ptr(), need - 1, None)
    assert st == 5 and b"workspace" in _abi.lib().b2_last_error()


def test_plain_path_in_mode_0(dev):
    w = torch.randn(9, 8).bfloat16().to(dev).requires_grad_()
    ids = torch.tensor([1, 1, 8], device=dev)
    native = lm.embedding(ids, w, scale=2.0)
    xdna_train.set_npu_mode(0)
    try:
        plain = lm.embedding(ids, w, scale=2.0)
    finally:
        xdna_train.set_npu_mode(2)
    assert torch.equal(native.cpu(), plain.cpu())


@pytest.mark.parametrize("T,V,D", [(33, 40, 33), (512, 300, 40), (513, 300, 40), (3001, 5000, 129), (4096, 700, 12),
                                   (4097, 3000, 40), (20011, 100, 18), (65536, 90000, 72), (262145, 50000, 8),
                                   (300000, 50000, 4)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["uniform", "zipf", "one", "falling"])
def test_sums_of_whole_numbers_are_exact(dev, T, V, D, dtype, kind):
    # whole numbers below 8: fp32 holds every partial sum (at most 7 * 300000 < 2^24) in any order, so that a token
    # lost, counted twice or added to another row shows at any count; the result is rounded once
    g = torch.Generator().manual_seed(T + D)
    ids = _ids(kind, T, V, g)
    pad = V - 1 if kind == "zipf" else None
    dy = torch.randint(-7, 8, (T, D), generator=g).to(dtype)
    w = torch.zeros(V, D, dtype=dtype, device=dev, requires_grad=True)
    (dw,) = torch.autograd.grad(lm.embedding(ids.to(dev), w, padding_idx=pad), [w], dy.to(dev))
    keep = torch.ones(T, dtype=torch.bool) if pad is None else ids != pad
    ref = torch.zeros(V, D, dtype=torch.float64).index_add_(0, ids[keep], dy.double()[keep])
    assert torch.equal(dw.cpu(), ref.to(dtype))


def test_cuda_views_of_results_keep_their_memory(dev):
    # the way out of an operator: the view is all that is left of its result
    want = torch.randn(64, 4096, generator=torch.Generator().manual_seed(7))
    w, ids = want.to(dev), torch.arange(64).to(dev)
    views = [xdna_train.as_cuda(lm.embedding(ids, w)) for _ in range(4)]
    again = [lm.embedding(ids, w, scale=0.0) for _ in range(8)]   # would take the memory of results that are gone
    assert all(torch.equal(v.cpu(), want) for v in views) and not any(a.cpu().any() for a in again)
    part = xdna_train.as_cuda(lm.embedding(ids, w)[3:5, 7:])
    back = xdna_train.as_xdna(xdna_train.as_cuda(lm.embedding(ids, w)))
    again = [lm.embedding(ids, w, scale=0.0) for _ in range(8)]
    assert torch.equal(part.cpu(), want[3:5, 7:]) and torch.equal(back.cpu(), want)
    before = xdna_train.allocator_stats()["allocated_bytes"]
    del views, part, back
    assert xdna_train.allocator_stats()["allocated_bytes"] <= before - 6 * want.numel() * 4
