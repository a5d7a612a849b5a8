"""xdna_train.lm.distill_loss (b2_distill_loss_fwd / _bwd) against its
definition in fp64.

Bounds.  The kernel's logits differences, sums and logarithms are fp32 with a
2^-22 exponential: a log-probability is off by at most 64 * 2^-22 (differences
of up to about 60 nats here) + 2^-20 (sum and logarithm) < 2e-5, and the
probabilities sum to 1, so a row's loss is off by at most
tau^2 * (2e-5 + 2e-6 * |loss|).  A gradient element w tau (q - p) has q and p off
by at most 2e-5 of themselves, and is rounded once to the logits' type."""
import math

import pytest
import torch

import xdna_train
from xdna_train import _abi, lm

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev(cuda):
    return torch.device("xdna", 0)

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -22}


def reference(z, t, ids, tau, w, reduction):
    """(loss, gradient for an upstream gradient of 1, per-element bound of its error before the last rounding)"""
    N, V = z.shape
    z, t, ids = z.cuda().double() / tau, t.cuda().double() / tau, ids.cuda()
    q = torch.softmax(z, 1)
    logq = torch.log_softmax(z, 1)
    t = t.masked_fill(ids < 0, -math.inf)
    has = (t > -math.inf).any(1) | t.isnan().any(1) if t.shape[1] else torch.zeros(N, dtype=torch.bool, device="cuda")
    p = torch.zeros_like(t)
    if t.shape[1]:
        p[has] = torch.softmax(t[has], 1)
    at = ids.long().clamp(min=0)
    terms = torch.where(p == 0, 0.0, p * (torch.log(p) - logq.gather(1, at)))
    rows = tau ** 2 * terms.sum(1)
    target = torch.zeros_like(q).scatter_add_(1, at, p)
    w = torch.ones(N, dtype=torch.float64, device="cuda") if w is None else w.cuda().double()
    on = has & (w != 0)
    rows = torch.where(on, rows * w, 0.0)
    f = w if reduction != "mean" else w / w.sum() if w.sum() != 0 else torch.zeros_like(w)
    grad = torch.where(on[:, None], f[:, None] * tau * (q - target), 0.0)
    slack = torch.where(on[:, None], f.abs()[:, None] * tau * 2e-5 * (q + target), 0.0)
    if reduction == "none":
        return rows, grad, slack
    return (rows.sum() if reduction == "sum" else (rows * f / torch.where(w != 0, w, 1.0)).sum()), grad, slack


def make(N, V, K, dtype, seed, pad=0, weights=True):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(N, V + pad, generator=g) * 3).to(dtype)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(N)]) if K else torch.zeros(N, 0, dtype=torch.long)
    t = (torch.randn(N, K, generator=g) * 3).to(dtype)
    if K > 2:
        ids[torch.rand(N, K, generator=g) < 0.15] = -1
        t[torch.rand(N, K, generator=g) < 0.1] = -math.inf
    w = (torch.rand(N, generator=g) * (torch.rand(N, generator=g) > 0.2)) if weights else None
    return z, t, ids, w


def check(z, t, ids, tau, w, reduction, dev, upstream=None, lo=0, hi=None):
    dtype = z.dtype
    zd = z.to(dev)
    zd = (zd if hi is None else zd[:, lo:hi]).detach().requires_grad_()
    z = z if hi is None else z[:, lo:hi]
    args = (t.to(dev), ids.to(dev), tau, None if w is None else w.to(dev), reduction)
    loss = lm.distill_loss(zd, *args)
    with torch.no_grad():
        plain = lm.distill_loss(zd, *args)
    ref, grad, slack = reference(z, t, ids, tau, w, reduction)
    assert loss.dtype == torch.float32 and torch.equal(torch.nan_to_num(loss.detach()), torch.nan_to_num(plain))
    ref_rows = reference(z, t, ids, tau, w, "none")[0].abs().nan_to_num()
    scale = 1.0 if reduction != "mean" else 1.0 / max(1e-30, len(z) if w is None else w.double().sum().item())
    wsum = float(len(z)) if w is None else w.double().sum().item()
    bound = (tau ** 2 * 2e-5 * (1.0 if reduction == "none" else wsum) + 2e-6 * (ref_rows if reduction == "none"
             else ref_rows.sum())) * scale + 1e-30
    got = xdna_train.as_cuda(loss.detach()).double()
    fine = ref.isfinite()
    assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got.isinf(), ref.isinf())
    assert ((got - ref).abs() <= bound)[fine].all() if ref.dim() else (not fine or abs(got - ref) <= bound)
    up = torch.ones_like(loss) if upstream is None else upstream.to(dev)
    (dz,) = torch.autograd.grad(loss, [zd], up)
    upc = xdna_train.as_cuda(up).double()
    upc = upc[:, None] if upc.dim() else upc
    ref = grad * upc
    got = xdna_train.as_cuda(dz).double()
    assert dz.dtype == dtype and dz.shape == zd.shape
    fine = ref.isfinite()
    assert torch.equal(got.isnan(), ref.isnan())
    assert ((got - ref).abs() <= slack * upc.abs() + UNIT[dtype] * ref.abs() + 1e-37)[fine].all()
    return loss, dz


SHAPES = [  # rows, vocabulary, entries
    (1, 1, 1), (3, 2, 1), (2, 7, 3), (5, 8, 8), (4, 9, 2), (3, 63, 20), (7, 1000, 33), (1, 32768, 8), (2, 33003, 40),
    (200, 5001, 16), (9, 40000, 300), (2, 131072, 64), (1, 300001, 5), (2, 450002, 1024), (1, 900001, 3), (3, 50, 0),
]


@pytest.mark.parametrize("N,V,K", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("reduction,tau", [("mean", 1.0), ("sum", 2.0), ("none", 0.5)])
def test_loss_and_gradient(dev, N, V, K, dtype, reduction, tau):
    z, t, ids, w = make(N, V, K, dtype, N + V + K)
    check(z, t, ids, tau, w if reduction != "sum" else None, reduction, dev)


# many long rows: the persistent kernel, alone and in clusters of 2, 4 and 8, aligned rows and rows of any alignment
MANY = [(1000, 9001, 7), (950, 20000, 9), (900, 32768, 33), (460, 40001, 17), (250, 131072, 64), (131, 262139, 5),
        (450, 36000, 1024)]


@pytest.mark.parametrize("N,V,K", MANY)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_rows(dev, N, V, K, dtype):
    g = torch.Generator().manual_seed(N)
    z = (torch.randn(N, V, generator=g) * 3).to(dtype)
    ids = (torch.randint(0, V, (N, 1), generator=g) + torch.arange(K) * (V // K)) % V  # distinct
    t = (torch.randn(N, K, generator=g) * 3).to(dtype)
    ids[torch.rand(N, K, generator=g) < 0.1] = -1
    ids[5:8] = -1
    t[torch.rand(N, K, generator=g) < 0.1] = -math.inf
    w = torch.rand(N, generator=g) * (torch.rand(N, generator=g) > 0.3)
    w[-3:] = 0
    z[0, 3] = z[1, V - 1] = -math.inf
    z[w == 0] = math.nan
    if K > 4:
        ids[2, 3] = ids[2, 0]              # a repeated entry
    check(z, t, ids, 1.0, w, "mean", dev)
    w[:] = 1
    z = z.nan_to_num(nan=1.0, neginf=-math.inf)
    z[9, 4] = math.nan
    z[10] = -math.inf
    z[11, V - 2] = math.inf
    check(z, t, ids, 2.0, None, "none", dev)


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_int32_ids(dev, reduction):
    z, t, ids, w = make(6, 1003, 9, torch.bfloat16, 1)
    check(z, t, ids.int(), 2.0, w, reduction, dev)
    assert xdna_train.kernel_stats().get("lm.distill", 0) > 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lo,hi", [(0, 1000), (1, 1001), (3, 996), (8, 1008), (0, 100)])
def test_views_of_a_wider_head(dev, dtype, lo, hi):
    z, _, _, _ = make(11, 1015, 1, dtype, 2)
    _, t, ids, w = make(11, hi - lo, 12, dtype, 3)
    check(z, t, ids, 1.0, w, "mean", dev, lo=lo, hi=hi)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_other_upstream_gradients(dev, dtype):
    z, t, ids, w = make(9, 5000, 12, dtype, 4)
    check(z, t, ids, 1.5, w, "mean", dev, upstream=torch.tensor(-0.3))
    check(z, t, ids, 1.5, w, "none", dev, upstream=torch.tensor([1.0, 0, 2, 1, -1, 0.1, 1, 1, 3]))


def test_masked_rows_are_not_read(dev):
    z, t, ids, w = make(8, 3000, 6, torch.float32, 5)
    w = torch.ones(8)
    z[1], w[1] = math.nan, 0.0
    z[2], ids[2] = math.inf, -1
    t[3] = -math.inf                      # entries without any probability
    z[3] = math.nan
    for reduction in ("mean", "sum", "none"):
        loss, dz = check(z, t, ids, 1.0, w, reduction, dev)
        assert loss.isfinite().all() and not dz[1:4].any()
    loss, dz = check(z, t, ids, 1.0, torch.zeros(8), "mean", dev)
    assert loss.item() == 0 and not dz.any()


def test_infinities_and_nan(dev):
    lowest = torch.finfo(torch.bfloat16).min
    z, t, ids, _ = make(8, 2050, 6, torch.bfloat16, 6)
    ids[:] = torch.arange(6) * 300
    t[:] = torch.arange(6.0)
    z[0, 7:] = -math.inf                  # most of the vocabulary closed, entries among it: infinite loss
    z[1, 1:299] = -math.inf               # closed, none of it an entry
    z[2, 1:299] = lowest
    z[3] = -math.inf                      # nothing left
    z[4, 5] = math.nan
    z[5, 5] = math.inf
    t[6, 2] = math.nan
    z[7] = lowest                         # all equal: a uniform distribution
    check(z, t, ids, 1.0, None, "none", dev)


def test_repeated_ids_add_up(dev):
    z, t, ids, w = make(5, 40, 30, torch.float32, 7)
    ids = torch.randint(-1, 6, (5, 30), generator=torch.Generator().manual_seed(1))
    check(z, t, ids, 1.0, w, "sum", dev)


def test_ids_outside_the_vocabulary_are_reported(dev):
    xdna_train.device_status(0)
    z, t, ids, _ = make(3, 100, 4, torch.float32, 8)
    ids[:] = torch.arange(4)
    ids[1, 2] = 100
    zd = z.to(dev).requires_grad_()
    loss = lm.distill_loss(zd, t.to(dev), ids.to(dev), reduction="none")
    (dz,) = torch.autograd.grad(loss.nan_to_num(0.0).sum(), [zd])
    assert loss.isnan().tolist() == [False, True, False]
    assert dz[1].isnan().all() and dz[[0, 2]].isfinite().all()
    assert xdna_train.device_status(0) == 1


def test_second_backward_and_untouched_logits(dev):
    z, t, ids, w = make(6, 700, 5, torch.bfloat16, 9)
    zd = z.to(dev).requires_grad_()
    loss = lm.distill_loss(zd, t.to(dev), ids.to(dev), row_weight=w.to(dev))
    (a,) = torch.autograd.grad(loss, [zd], retain_graph=True)
    keep = a.clone()
    (b,) = torch.autograd.grad(loss * 3.0, [zd])
    assert torch.equal(a, keep) and torch.equal(zd.detach().cpu(), z)
    assert ((b.float() - 3 * a.float()).abs() <= 2.0 ** -7 * b.float().abs() + 1e-30).all()


def test_batched_logits_and_streams(dev):
    z, t, ids, w = make(12, 5000, 7, torch.bfloat16, 10)
    zd, td, idd, wd = z.to(dev), t.to(dev), ids.to(dev), w.to(dev)
    flat = lm.distill_loss(zd, td, idd, row_weight=wd, reduction="none")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        batched = lm.distill_loss(zd.view(3, 4, 5000), td.view(3, 4, 7), idd.view(3, 4, 7), row_weight=wd.view(3, 4),
                                  reduction="none")
    torch.cuda.current_stream().wait_stream(side)
    assert batched.shape == (3, 4) and torch.equal(batched.reshape(-1), flat)
    one = lm.distill_loss(zd[0], td[0], idd[0], row_weight=wd[0], reduction="none")
    assert one.shape == () and one == flat[0]
    empty = lm.distill_loss(zd[:0].requires_grad_(), td[:0], idd[:0])
    assert empty.item() == 0


def test_gradient_against_differences(dev):
    z, t, ids, w = make(4, 300, 10, torch.float32, 11)
    d = torch.randn(4, 300, generator=torch.Generator().manual_seed(2)).to(dev)
    zd, args = z.to(dev).requires_grad_(), (t.to(dev), ids.to(dev), 2.0, w.to(dev), "sum")
    (dz,) = torch.autograd.grad(lm.distill_loss(zd, *args), [zd])
    h = 0.02
    f = lambda e: lm.distill_loss((zd + e * d).detach(), *args).item()  # noqa: E731
    # second order: h^2 / 6 times the third derivative of log-sum-exp along d (at most 2 max|d / tau|^3 tau^2 a row);
    # rounding: the losses' bound over h
    third = 4 * 2.0 ** 2 * 2 * (d.abs().max().item() / 2.0) ** 3
    bound = h * h / 6 * third + 2 * (4 * 2.0 ** 2 * 2e-5) / (2 * h)
    assert abs((f(h) - f(-h)) / (2 * h) - (dz.double() * d.double()).sum().item()) <= bound


def test_refusals(dev):
    z, t, ids, w = (v.to(dev) for v in make(3, 50, 4, torch.float32, 12))
    for bad in (lambda: lm.distill_loss(z.half(), t, ids), lambda: lm.distill_loss(z, t.double(), ids),
                lambda: lm.distill_loss(z, t, ids.float()), lambda: lm.distill_loss(z, t[:, :2], ids),
                lambda: lm.distill_loss(z[:2], t, ids), lambda: lm.distill_loss(z, t.cpu(), ids),
                lambda: lm.distill_loss(z, t, ids, temperature=0.0),
                lambda: lm.distill_loss(z, t, ids, temperature=math.inf),
                lambda: lm.distill_loss(z, t, ids, row_weight=w[:2]),
                lambda: lm.distill_loss(z, t, ids, row_weight=w.double()),
                lambda: lm.distill_loss(z, t.clone().requires_grad_(), ids)):
        with pytest.raises(RuntimeError, match="xdna distill_loss"):
            bad()
    with pytest.raises(ValueError, match="reduction"):
        lm.distill_loss(z, t, ids, reduction="batchmean")
    with pytest.raises(RuntimeError, match="1024 teacher entries"):
        lm.distill_loss(z.repeat(1, 40), t[:, :1].expand(3, 1025).contiguous(), ids[:, :1].expand(3, 1025).contiguous())
    zg = z.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(lm.distill_loss(zg, t, ids), [zg], create_graph=True)
    st = _abi.lib().b2_distill_loss_fwd(z.data_ptr(), 49, _abi.B2_F32, 3, 50, t.data_ptr(), 4, _abi.B2_F32,
                                        ids.data_ptr(), 4, _abi.B2_I64, 4, 1.0, None, 0, z.data_ptr(), z.data_ptr(),
                                        None, 50, z.data_ptr(), 1000, None)
    assert st == 1 and b"row stride" in _abi.lib().b2_last_error()


@pytest.mark.parametrize("N,V", [(900, 9001), (460, 40001), (250, 131072), (131, 262139)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_closed_slices(dev, N, V, dtype):
    # a long part of a row closed (a masked range of the vocabulary), so that some CTA of the row's cluster sees
    # nothing else: infinite loss where a live entry lies in it, as for a single closed logit, else a finite one
    g = torch.Generator().manual_seed(V)
    z = (torch.randn(N, V, generator=g) * 3).to(dtype)
    t = torch.randn(N, 4, generator=g)
    ids = torch.randint(0, V // 8, (N, 4), generator=g) + torch.arange(4) * (V // 4)  # one entry in each quarter
    late, early = slice(V // 2 - 16, V), slice(0, V // 2 + 16)
    z[2, late] = -math.inf                                   # entries on both sides
    z[3, early] = -math.inf
    z[4, late], ids[4, 2:] = -math.inf, -1                   # entries on the open side alone
    z[5, early], ids[5, :2] = -math.inf, -1
    z[6, late], ids[6, :2] = -math.inf, -1                   # on the closed side alone
    z[7, late], t[7, 2:] = -math.inf, -math.inf              # those on the closed side have no probability
    z[8, V // 8 + 16:] = -math.inf                           # all but a first part
    z[9, late], z[9, 1] = -math.inf, math.nan
    z[10, late], z[10, V - 1] = -math.inf, math.nan
    loss, _ = check(z, t, ids, 2.0, None, "none", dev)
    assert loss.isinf().nonzero().flatten().tolist() == [2, 3, 6, 8]
    assert loss.isnan().nonzero().flatten().tolist() == [9, 10]
    w = torch.ones(N)
    w[9:11] = 0
    loss, _ = check(z, t, ids, 2.0, w, "mean", dev)
    assert loss.item() == math.inf


@pytest.mark.parametrize("N,V", [(12, 2051), (900, 9001), (460, 40001)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tau", [1.0, 2.0, 0.05])
def test_logits_far_from_zero(dev, N, V, dtype, tau):
    # a row's loss and gradient depend on its logits' differences alone, wherever the row lies
    g = torch.Generator().manual_seed(V)
    z = torch.randn(N, V, generator=g) * 3
    for r, at in enumerate([100.0, 500.0, 1000.0, 5000.0, 2.0 ** 20, -2.0 ** 20, 2.0 ** 30, 2.0 ** 100, -2.0 ** 126]):
        # steps that the type still tells apart: an eighth (bf16) of `at` is many
        z[r] = at * (1 + (z[r] / 3).clamp(-4, 4).round() * 2.0 ** (-7 if dtype == torch.bfloat16 else -22))
    z[9] = torch.finfo(dtype).min                # all of the row at the type's lowest value: uniform
    z[10], z[10, 7:9] = torch.finfo(dtype).min, 2.0
    z = z.to(dtype)
    ids = torch.randint(0, V // 8, (N, 4), generator=g) + torch.arange(4) * (V // 4)
    t = torch.randn(N, 4, generator=g)
    t[10] = -math.inf
    loss, dz = check(z, t, ids, tau, None, "none", dev)
    assert loss[9].isfinite() and dz[:11].isfinite().all()
    w = torch.ones(N)
    w[4:9] = 0
    check(z, t, ids, tau, w, "sum", dev, upstream=torch.tensor(0.7))


@pytest.mark.parametrize("N,V", [(12, 2050), (900, 9001), (460, 40001), (250, 131072)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tau", [1.0, 0.5, 2.0])
def test_entries_masked_with_the_lowest_value(dev, N, V, dtype, tau):
    # a finite logit, however low, has a finite log-probability (3.4e38 / tau below the others), and the loss
    # p tau 3.4e38 with the teacher's p of e^-4 / 2 here is well inside fp32's range.  p's exponent is exact but for
    # c's rounding and the product's (6 * 2^-23), the other five operations round at 2^-24 to 2^-22: inside 2e-6.
    lowest = torch.finfo(dtype).min
    g = torch.Generator().manual_seed(V)
    z = (torch.randn(N, V, generator=g) * 3).to(dtype)
    t = torch.randn(N, 4, generator=g)
    ids = torch.randint(0, V // 8, (N, 4), generator=g) + torch.arange(4) * (V // 4)
    rows = torch.arange(2, 10)
    t[rows] = torch.tensor([0.0, 0.0, -4.0 * tau, -4.0 * tau])
    z[rows, ids[rows, 3]] = lowest                            # one entry (of row 4: both of the first half)
    z[3, V // 2 - 16:] = lowest                               # a whole range, two entries in it
    z[4, :V // 2 + 16], z[4, ids[4, 3]], t[4] = lowest, 0, t[4].flip(0)
    z[5, 1:], ids[5, 0], t[5, 0] = lowest, 0, 6.0 * tau       # all but the first logit
    loss, _ = check(z, t, ids, tau, None, "none", dev)
    assert loss[2:10].isfinite().all() and (loss[2:10] > 1e33).all()


@pytest.fixture
def short_waits():
    # restored whatever happens
    _abi.call("b2_distill_set_wait_limit", 1)
    yield
    _abi.call("b2_distill_set_wait_limit", 0)


@pytest.mark.parametrize("N,V", [(900, 32768), (460, 40001), (250, 131072), (131, 262139)])
@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("train", [True, False])
def test_a_wait_that_runs_out_ends_the_call(dev, short_waits, N, V, reduction, train):
    # a limit below the time of any copy: the waits give up at the first rows, the kernel ends by itself, reports it
    # and leaves NaN; then the same call without the limit is what it always was
    xdna_train.device_status(0)
    z, t, ids, w = make(N, V, 4, torch.bfloat16, 13)
    w[::3] = 0                                 # masked rows among the others
    zd = z.to(dev).requires_grad_(train)
    args = (t.to(dev), ids.to(dev), 1.0, w.to(dev), reduction)
    loss = lm.distill_loss(zd, *args)
    assert loss.isnan().any()
    assert xdna_train.device_status(0) == 4    # B2_ERR_TIMEOUT
    _abi.call("b2_distill_set_wait_limit", 0)
    check(z, t, ids, 1.0, w, reduction, dev)
    assert xdna_train.device_status(0) == 0


@pytest.mark.parametrize("N,V", [(4000, 12001), (3, 450002), (20, 900001)])
@pytest.mark.parametrize("train", [True, False])
def test_rows_of_a_cluster_whose_wait_runs_out(dev, short_waits, N, V, train):
    # the kernel with a cluster a row (4000 rows that wait for the memory system; rows of several tiles a CTA, whose
    # second copy starts right before its wait): such a row's loss and gradient are NaN, and the call without a limit
    # is right
    xdna_train.device_status(0)
    z, t, ids, _ = make(N, V, 4, torch.float32, 14)
    ids[:, 0], t[:, 0] = 5, 0.0                # every row has an entry
    zd = z.to(dev).requires_grad_(train)
    loss = lm.distill_loss(zd, t.to(dev), ids.to(dev), reduction="none")
    if train:
        (dz,) = torch.autograd.grad(loss.sum(), [zd])
    lost = loss.detach().isnan()
    assert lost.any() and xdna_train.device_status(0) == 4
    if train:
        assert dz[lost].isnan().any(1).all()
    _abi.call("b2_distill_set_wait_limit", 0)
    check(z, t, ids, 1.0, None, "none", dev)
    assert xdna_train.device_status(0) == 0


@pytest.mark.parametrize("N,V,K", [(5, 40000, 12), (9, 70001, 33), (3, 131072, 64), (2, 450002, 1024), (700, 33000, 7)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_other_upstream_gradients_of_long_rows(dev, N, V, K, dtype):
    # rows that the backward takes in several pieces, aligned and not, entries and closed logits in all of them
    z, t, ids, w = make(N, V, K, dtype, 15)
    ids[0, :3] = torch.tensor([0, V - 1, V // 2])
    z[1, V // 3:V // 2] = -math.inf
    check(z, t, ids, 1.5, w, "mean", dev, upstream=torch.tensor(-0.3))
    check(z, t, ids, 1.0, None, "sum", dev, upstream=torch.tensor(3.0))
    up = torch.randn(N, generator=torch.Generator().manual_seed(16))
    up[0], up[-1] = 1.0, 0.0
    check(z, t, ids, 1.5, w, "none", dev, upstream=up)


@pytest.mark.parametrize("lo,hi", [(1, 60001), (3, 59996), (8, 60008)])
def test_other_upstream_gradients_of_long_views(dev, lo, hi):
    z, _, _, _ = make(6, 60015, 1, torch.bfloat16, 17)
    _, t, ids, w = make(6, hi - lo, 12, torch.bfloat16, 18)
    check(z, t, ids, 1.0, w, "mean", dev, upstream=torch.tensor(0.5), lo=lo, hi=hi)
