"""xdna_train.lm.gated_mlp (b2_gated_mlp_fwd_bf16 / _bwd_bf16) against its
formulas in fp64.

Bounds, with eps = 2^-8 (the unit roundoff of bf16's 8-bit significand): h is rounded once, and so
is y; the backward's factors u act'(g) and act(g) are rounded once and dg and du,
products with them, once more; the outputs once.  So an element of y or dw_down
is off by at most 2 eps (1 + 2^-9) and one of dx, dw_gate or dw_up by at most 3
eps (1 + 2^-8) of the sum of its terms' absolute values; fp32 sums of products
and the hardware's exponential add less than 2^-16 of the absolute sums, those
behind dh and g included, for which another eps / 8 is allowed.  These are worst
cases.  The roundings are independent, so the error of a whole tensor in the
2-norm is at most about eps sqrt(k / 6) for k <= 3 roundings (the average of a
rounding's square over a binade): 2 eps bounds that."""
import pytest
import torch

import xdna_train
from xdna_train import _abi, lm

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -8
ACT = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu}


@pytest.fixture
def dev(cuda):
    return torch.device("xdna", 0)


def make(M, D, F, E, seed=0):
    g = torch.Generator().manual_seed(seed + M + D + F + E)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).bfloat16()  # noqa: E731
    return r(M, D), r(F, D, std=D ** -0.5), r(F, D, std=D ** -0.5), r(E, F, std=F ** -0.5), r(M, E, std=0.1)


def reference(x, wg, wu, wd, dy, act):
    """y, dx, dw_gate, dw_up, dw_down, each with its elements' bound"""
    with torch.no_grad():
        x, wg, wu, wd, dy = (t.double().cuda() for t in (x, wg, wu, wd, dy))
        g, u = x @ wg.t(), x @ wu.t()
        if act == "silu":
            s = torch.sigmoid(g)
            a, slope = g * s, s * (1 + g * (1 - s))
        elif act == "gelu":
            cdf = 0.5 * (1 + torch.erf(g / 2 ** 0.5))
            a, slope = g * cdf, cdf + g * torch.exp(-g * g / 2) / (2 * torch.pi) ** 0.5
        else:
            a, slope = torch.relu(g), (g > 0).double()
        h = a * u
        dh = dy @ wd
        dg, du = dh * u * slope, dh * a
        # what fp32 sums may leave in g, u and dh, carried to h, dg and du (act and act' move by at most 1.2 per unit)
        tiny = 2.0 ** -20
        eg, eu, ed = (tiny * (p.abs() @ q.abs()) for p, q in ((x, wg.t()), (x, wu.t()), (dy, wd)))
        eh = 1.2 * (u.abs() * eg + a.abs() * eu)
        edg = ed * (u * slope).abs() + dh.abs() * 1.2 * (eu + u.abs() * eg)
        edu = ed * a.abs() + dh.abs() * 1.2 * eg
        if act == "relu":  # a gate that fp32 may see on the other side of zero
            edg = edg + torch.where(g.abs() <= eg, dh.abs() * u.abs(), 0.0)
        m = lambda p, q: p.abs() @ q.abs()  # noqa: E731
        two, three = 2.13 * EPS, 3.13 * EPS
        return ((h @ wd.t(), two * m(h, wd.t()) + m(eh, wd.t())),
                (dg @ wg + du @ wu, three * (m(dg, wg) + m(du, wu)) + m(edg, wg) + m(edu, wu)),
                (dg.t() @ x, three * m(dg.t(), x) + m(edg.t(), x)), (du.t() @ x, three * m(du.t(), x) + m(edu.t(), x)),
                (dy.t() @ h, two * m(dy.t(), h) + m(dy.t(), eh)))


def close(got, ref, what):
    got = xdna_train.as_cuda(got.detach()).double()
    ref, bound = ref
    assert got.shape == ref.shape, what
    if ref.numel() == 0:
        return
    err = (got - ref).abs()
    assert (err <= bound + 1e-37).all(), (what, (err / (bound + 1e-37)).max().item())
    assert err.norm() <= 2 * EPS * ref.norm() + 1e-30, (what, (err.norm() / ref.norm()).item())


def check(M, D, F, E, act, dev, seed=0):
    x, wg, wu, wd, dy = make(M, D, F, E, seed)
    leaves = [t.to(dev).requires_grad_() for t in (x, wg, wu, wd)]
    y = lm.gated_mlp(*leaves, activation=act)
    with torch.no_grad():
        served = lm.gated_mlp(*leaves, activation=act)
    ref = reference(x, wg, wu, wd, dy, act)
    close(y, ref[0], "y")
    close(served, ref[0], "y without gradients")
    for got, want, what in zip(torch.autograd.grad(y, leaves, dy.to(dev)), ref[1:], ("dx", "dw_gate", "dw_up", "dw_down")):
        close(got, want, what)


SIZES = [
    # M, D, F, E
    (1, 8, 8, 8), (1, 1, 1, 1), (2, 3, 5, 7), (1, 64, 256, 64), (7, 72, 40, 24), (8, 1000, 520, 1000),
    (15, 129, 257, 65), (17, 64, 100, 96), (33, 320, 704, 320), (64, 512, 1024, 512), (65, 136, 1032, 72),
    (127, 256, 384, 256), (129, 200, 333, 201), (256, 256, 256, 256), (257, 264, 520, 136), (300, 1001, 130, 999),
    (513, 512, 1024, 512), (1000, 96, 72, 104), (2048, 64, 128, 64), (16, 4096, 512, 2048), (1, 4096, 1536, 2048),
    (5000, 40, 24, 32), (777, 1001, 530, 1001), (1024, 1024, 2048, 1024),
]


@pytest.mark.parametrize("M,D,F,E", SIZES)
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_forward_and_gradients(dev, M, D, F, E, act):
    check(M, D, F, E, act, dev)


def test_wide_layer(dev):
    check(2560, 1536, 4608, 1536, "silu", dev)


@pytest.mark.parametrize("M", [2, 3, 4, 5, 9, 16, 24, 31, 32, 34, 48, 63, 96, 128, 200])
def test_every_number_of_tokens(dev, M):
    check(M, 256, 688, 256, "silu", dev)
    check(M, 250, 342, 126, "gelu", dev)


def test_strided_and_misaligned_operands(dev):
    M, D, F, E = 40, 96, 136, 88
    x, wg, wu, wd, dy = make(M, D, F, E)
    ref = reference(x, wg, wu, wd, dy, "silu")

    def wide(t, left, extra):  # t inside a wider matrix
        w = torch.zeros(t.shape[0], t.shape[1] + left + extra, dtype=t.dtype)
        w[:, left:left + t.shape[1]] = t
        return w.to(dev)[:, left:left + t.shape[1]]

    for left, extra in ((8, 8), (1, 7), (3, 2), (0, 1)):
        leaves = [wide(t, left, extra).detach().requires_grad_() for t in (x, wg, wu, wd)]
        y = lm.gated_mlp(*leaves)
        close(y, ref[0], "y")
        for got, want in zip(torch.autograd.grad(y, leaves, wide(dy, left, extra)), ref[1:]):
            close(got, want, "gradient")
    leaves = [t.t().contiguous().to(dev).t().detach().requires_grad_() for t in (x, wg, wu, wd)]  # columns strided
    y = lm.gated_mlp(*leaves)
    close(y, ref[0], "y")
    for got, want in zip(torch.autograd.grad(y, leaves, dy.to(dev)), ref[1:]):
        close(got, want, "gradient")
    y = lm.gated_mlp(*leaves)
    for got, want in zip(torch.autograd.grad(y, leaves, dy.to(dev)[:1, :1].expand(M, E)),
                         reference(x, wg, wu, wd, dy[:1, :1].expand(M, E), "silu")[1:]):
        close(got, want, "gradient of a broadcast")


def test_batched_input_and_partial_gradients(dev):
    x, wg, wu, wd, dy = make(24, 64, 80, 48)
    ref = reference(x, wg, wu, wd, dy, "silu")
    for wanted in ((0,), (1, 3), (2,), (3,), (0, 2)):
        leaves = [t.to(dev).requires_grad_(i in wanted) for i, t in enumerate((x, wg, wu, wd))]
        y = lm.gated_mlp(leaves[0].view(2, 3, 4, 64), *leaves[1:])
        assert y.shape == (2, 3, 4, 48)
        grads = torch.autograd.grad(y, [leaves[i] for i in wanted], dy.to(dev).view(2, 3, 4, 48))
        for i, got in zip(wanted, grads):
            close(got, ref[1 + i], "gradient")


def test_no_tokens(dev):
    x, wg, wu, wd, _ = make(0, 16, 24, 8)
    leaves = [t.to(dev).requires_grad_() for t in (x, wg, wu, wd)]
    y = lm.gated_mlp(*leaves)
    assert y.shape == (0, 8)
    dx, *dw = torch.autograd.grad(y, leaves, torch.empty(0, 8, dtype=torch.bfloat16).to(dev))
    assert dx.shape == (0, 16) and all(not g.any() for g in dw)


def test_large_and_special_values(dev):
    x, wg, wu, wd, _ = make(12, 32, 40, 16)
    x[0] = 300.0 * wg[0].sign()             # a gate far in either tail
    x[1] = -300.0 * wg[0].sign()
    x[2, 3] = float("inf")
    x[3, 3] = float("nan")
    for act in ACT:
        y = lm.gated_mlp(x.to(dev), wg.to(dev), wu.to(dev), wd.to(dev), activation=act).cpu()
        assert y[[2, 3]].isnan().all()
        close(y[[0, 1, 4, 5]].to(dev), reference(x[[0, 1, 4, 5]], wg, wu, wd, torch.zeros(4, 16), act)[0], act)


@pytest.mark.parametrize("M", [1, 30, 600])
def test_same_bits_on_every_run_and_stream(dev, M):
    x, wg, wu, wd, dy = (t.to(dev) for t in make(M, 264, 1032, 264))
    leaves = [t.requires_grad_() for t in (x, wg, wu, wd)]

    def once():
        y = lm.gated_mlp(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = once()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_gradient_against_differences(dev):
    """A step h along one direction d moves sum(c * y) by 2h <grad, d> up to third order."""
    M, D, F, E = 64, 64, 96, 64
    x, wg, wu, wd, c = make(M, D, F, E, seed=3)
    leaves = [t.to(dev).requires_grad_() for t in (x, wg, wu, wd)]
    grads = torch.autograd.grad(lm.gated_mlp(*leaves, activation="gelu"), leaves, c.to(dev))
    gen = torch.Generator().manual_seed(1)
    for i, leaf in enumerate((x, wg, wu, wd)):
        d = torch.randn(leaf.shape, generator=gen) * leaf.float().std()
        step = 0.0625
        sides = []
        for sign in (1, -1):
            moved = [t.to(dev) for t in (x, wg, wu, wd)]
            moved[i] = (leaf.float() + sign * step * d).bfloat16().to(dev)
            sides.append((lm.gated_mlp(*moved, activation="gelu").cpu().double() * c.double()).sum().item())
        along = (leaf.float() + step * d).bfloat16().double() - (leaf.float() - step * d).bfloat16().double()
        linear = (grads[i].cpu().double() * along).sum().item()
        # rounding: y's elements are off by about eps / 2 of their rms (independent), each weighted by c, on both
        # sides; the gradient by 2 eps; third order: a step of 1/16 leaves h^2 / 6 < 0.1 % of the curvature terms
        rms = lm.gated_mlp(*[t.to(dev) for t in (x, wg, wu, wd)], activation="gelu").float().square().mean().sqrt().item()
        noise = 6 * EPS * rms * c.double().norm().item()
        scale = grads[i].cpu().double().norm().item() * along.norm().item()
        assert abs((sides[0] - sides[1]) - linear) <= noise + (2 * EPS + 0.002) * scale


def test_autocast_and_mode_0(dev):
    x, wg, wu, wd, _ = make(20, 64, 96, 64)
    native = lm.gated_mlp(*(t.to(dev) for t in (x, wg, wu, wd)))
    with torch.autocast("xdna", torch.bfloat16):
        cast = lm.gated_mlp(x.float().to(dev), *(t.float().to(dev) for t in (wg, wu, wd)))
    assert torch.equal(native, cast)
    xdna_train.set_npu_mode(0)
    try:
        plain = lm.gated_mlp(*(t.to(dev) for t in (x, wg, wu, wd)))
    finally:
        xdna_train.set_npu_mode(2)
    # the plain path rounds g, u, act(g) and h
    assert (plain.float() - native.float()).norm() <= 2 * EPS * native.float().norm()


def test_refusals(dev):
    x, wg, wu, wd, _ = (t.to(dev) for t in make(4, 16, 24, 8))
    for bad in (lambda: lm.gated_mlp(x.float(), wg, wu, wd), lambda: lm.gated_mlp(x, wg.half(), wu, wd),
                lambda: lm.gated_mlp(x[:, :8], wg, wu, wd), lambda: lm.gated_mlp(x, wg[:8], wu, wd),
                lambda: lm.gated_mlp(x, wg, wu, wd[:, :8]), lambda: lm.gated_mlp(x, wg, wu, wd[0]),
                lambda: lm.gated_mlp(x, wg, wu.cpu(), wd), lambda: lm.gated_mlp(xdna_train.as_cuda(x), wg, wu, wd)):
        with pytest.raises(RuntimeError, match="xdna"):
            bad()
    with pytest.raises(ValueError, match="activation"):
        lm.gated_mlp(x, wg, wu, wd, activation="tanh")
    xg = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(lm.gated_mlp(xg, wg, wu, wd).sum(), [xg], create_graph=True)
    L = _abi.lib()
    need = L.b2_gated_mlp_fwd_workspace_bytes(4, 16, 24, 8)
    st = L.b2_gated_mlp_fwd_bf16(x.data_ptr(), 16, wg.data_ptr(), 16, wu.data_ptr(), 16, wd.data_ptr(), 24, 0,
                                 x.data_ptr(), 8, None, 4, 16, 24, 8, x.data_ptr(), need - 1, None)
    assert st == 5 and b"workspace" in L.b2_last_error()
    assert xdna_train.device_status(0) == 0


@pytest.mark.parametrize("M", [1, 2, 3, 4])
@pytest.mark.parametrize("D,F,E", [(64, 104, 40), (1024, 4096, 256), (512, 1531, 77)])
def test_up_to_four_tokens_round_once(dev, M, D, F, E):
    # h goes on as two bf16 numbers, which leave eps^2 of it; y is rounded once.  fp32 sums add less than 2^-16 of
    # the absolute sums, as above.
    x, wg, wu, wd, dy = make(M, D, F, E, 5)
    with torch.no_grad():
        y = lm.gated_mlp(*(t.to(dev) for t in (x, wg, wu, wd)))
    ref, _ = reference(x, wg, wu, wd, dy, "silu")[0]
    x, wg, wu, wd = (t.double().cuda() for t in (x, wg, wu, wd))
    g, u = x @ wg.t(), x @ wu.t()
    a = g * torch.sigmoid(g)
    eh = 1.2 * 2.0 ** -20 * (u.abs() * (x.abs() @ wg.abs().t()) + a.abs() * (x.abs() @ wu.abs().t()))
    inner = (EPS ** 2 + 2.0 ** -16) * ((a * u).abs() @ wd.abs().t()) + eh @ wd.abs().t()
    err = (xdna_train.as_cuda(y).double() - ref).abs()
    assert (err <= EPS * ref.abs() + 1.01 * inner).all()


def test_few_tokens_keep_infinities(dev):
    # an h beyond bf16's range is an infinity, and what its rounding left is not a NaN
    x = torch.full((1, 8), 2.0 ** 60).bfloat16()
    w = torch.full((8, 8), 2.0 ** 8).bfloat16()
    y = lm.gated_mlp(x.to(dev), w.to(dev), w.to(dev), torch.ones(8, 8).bfloat16().to(dev), activation="relu")
    assert (xdna_train.as_cuda(y) == float("inf")).all()


def test_kept_tensors_are_autograds(dev):
    # what the forward keeps is a saved tensor like any other: hooks see it, it can be moved to the host, a checkpoint
    # makes it again, and it is freed by the backward, not with the graph
    from torch.utils.checkpoint import checkpoint
    M, D, F, E = 300, 64, 1000, 72
    x, wg, wu, wd, dy = (t.to(dev) for t in make(M, D, F, E, 8))
    leaves = [t.requires_grad_() for t in (x, wg, wu, wd)]
    seen = []

    def pack(t):
        seen.append(t.numel())
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        y = lm.gated_mlp(*leaves)
    assert max(seen) >= 4 * M * F
    want = torch.autograd.grad(y, leaves, dy)
    with torch.autograd.graph.save_on_cpu():
        moved = lm.gated_mlp(*leaves)
    again = checkpoint(lambda *a: lm.gated_mlp(*a), *leaves, use_reentrant=False, preserve_rng_state=False)
    for other in (moved, again):
        assert torch.equal(other, y)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(other, leaves, dy), want))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(again, leaves, dy)


def test_kept_tensors_are_freed_by_the_backward(dev):
    M, D, F, E = 1024, 64, 8192, 64
    x, wg, wu, wd, dy = (t.to(dev) for t in make(M, D, F, E, 9))
    leaves = [t.requires_grad_() for t in (x, wg, wu, wd)]
    y = lm.gated_mlp(*leaves)
    before = xdna_train.allocator_stats()["allocated_bytes"]
    torch.autograd.grad(y, leaves, dy)                  # the gradients go at once, y and its graph stay
    assert xdna_train.allocator_stats()["allocated_bytes"] <= before - 8 * M * F


def _decode(saved, M, F):
    """h, P = u act'(g) and A = act(g) of the forward's buffer: 16-bit words h, upper half of P, of A, and the next 8
    bits of both (P's above A's)"""
    words = saved.view(torch.int16).view(M, 4, -1)[:, :, :F].long() & 0xffff
    h, p, a, r = words.unbind(1)
    f32 = lambda bits: (bits - ((bits >> 31) << 32)).int().view(torch.float32).double()  # noqa: E731
    return f32(h << 16), f32((p << 16) | (r & 0xff00)), f32((a << 16) | ((r & 0xff) << 8))


@pytest.mark.parametrize("M,D,F,E", [
    (1, 256, 688, 64), (3, 64, 104, 40), (16, 512, 1531, 64), (24, 1024, 4096, 64),            # few tokens
    (64, 1024, 512, 64), (40, 2045, 300, 33), (129, 2048, 333, 64),                            # split reductions
    (300, 64, 1000, 64), (257, 100, 130, 64), (2048, 128, 1536, 64), (5, 61, 77, 13),          # whole ones
])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_kept_factors_have_sixteen_bits(cuda, M, D, F, E, act):
    # truncated to 16 bits of significand: 2^-15 of themselves.  fp32 sums leave 2^-20 of the absolute sums in g and u
    # (act and act' move by at most 1.2 a unit), the activation's own arithmetic 2^-19.  As bf16 they would be off by
    # up to 2^-7.
    x, wg, wu, wd, _ = (t.to(cuda) for t in make(M, D, F, E, 6))
    L, Fp = _abi.lib(), (F + 7) // 8 * 8
    y = torch.empty(M, E, dtype=torch.bfloat16, device=cuda)
    saved = torch.zeros(M * 4 * Fp, dtype=torch.bfloat16, device=cuda)
    need = L.b2_gated_mlp_fwd_workspace_bytes(M, D, F, E)
    ws = torch.empty(need, dtype=torch.uint8, device=cuda)
    _abi.call("b2_gated_mlp_fwd_bf16", x.data_ptr(), D, wg.data_ptr(), D, wu.data_ptr(), D, wd.data_ptr(), F,
              ["silu", "gelu", "relu"].index(act), y.data_ptr(), E, saved.data_ptr(), M, D, F, E, ws.data_ptr(), need,
              torch.cuda.current_stream().cuda_stream)
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, u = x @ wg.t(), x @ wu.t()
    a = ACT[act](g)
    sig, pdf = torch.sigmoid(g), torch.exp(-g * g / 2) / (2 * torch.pi) ** 0.5
    slope = {"silu": sig * (1 + g * (1 - sig)), "gelu": 0.5 * (1 + torch.erf(g / 2 ** 0.5)) + g * pdf,
             "relu": (g > 0).double()}[act]
    eg, eu = (2.0 ** -20 * (x.abs() @ w.abs().t()) for w in (wg, wu))
    h, P, A = _decode(saved, M, F)
    sure = g.abs() > eg if act == "relu" else torch.ones_like(g, dtype=torch.bool)
    eP = 1.2 * (u.abs() + eu) * eg + slope.abs() * eu + 2.0 ** -19 * u.abs()
    assert ((P - u * slope).abs() <= 2.0 ** -15 * (u * slope).abs() + eP)[sure].all()
    assert ((A - a).abs() <= 2.0 ** -15 * a.abs() + 1.2 * eg + 2.0 ** -19).all()
    eh = a.abs() * eu + (u.abs() + eu) * (1.2 * eg + 2.0 ** -19)
    assert ((h - a * u).abs() <= EPS * (a * u).abs() + 1.01 * eh).all()


@pytest.mark.parametrize("M,F", [(1, 8), (37, 64), (64, 128), (200, 130), (2048, 1536), (64, 1024), (33, 2061)])
def test_backward_takes_all_sixteen_bits(cuda, M, F):
    # x and w_down are unit matrices, so that dh = dy and dw_gate = (dy P)^T, dw_up = (dy A)^T: exact fp32 products of
    # 8 by 16 bits, rounded once to bf16 -- the same bits as torch's.  Whole and split reductions of dh.
    g = torch.Generator().manual_seed(M + F)
    Fp = (F + 7) // 8 * 8
    dy = torch.randn(M, F, generator=g).bfloat16().to(cuda)
    factors = (torch.randn(2, M, F, generator=g).to(cuda).view(torch.int32) & -256).view(torch.float32)
    words = torch.zeros(M, 4, Fp, dtype=torch.int64, device=cuda)
    bits = factors.view(torch.int32).long() & 0xffffffff
    words[:, 1:3, :F] = (bits >> 16).transpose(0, 1)
    words[:, 3, :F] = (bits[0] & 0xff00) | ((bits[1] >> 8) & 0xff)
    saved = (words - ((words >> 15) << 16)).short().contiguous()
    x, wd = (torch.eye(n, dtype=torch.bfloat16, device=cuda) for n in (M, F))
    w = torch.zeros(F, M, dtype=torch.bfloat16, device=cuda)
    out = [torch.full((F, M), 7.0, dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    need = _abi.lib().b2_gated_mlp_bwd_workspace_bytes(M, M, F, F)
    ws = torch.empty(need, dtype=torch.uint8, device=cuda)
    _abi.call("b2_gated_mlp_bwd_bf16", dy.data_ptr(), F, x.data_ptr(), M, w.data_ptr(), M, w.data_ptr(), M,
              wd.data_ptr(), F, 0, saved.data_ptr(), None, out[0].data_ptr(), out[1].data_ptr(), None, M, M, F, F,
              ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    for got, factor in zip(out, factors):
        want = (dy.float() * factor).bfloat16()
        assert torch.equal(got.t(), want)
        assert M * F < 64 or not torch.equal((dy.float() * factor.bfloat16().float()).bfloat16(), want)


@pytest.mark.parametrize("M,D,F,E", [(16, 512, 1024, 512), (64, 512, 1024, 512), (300, 1001, 1300, 999),
                                     (1024, 512, 2048, 512)])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_two_roundings_and_no_more(dev, M, D, F, E, act):
    # y and dw_down carry the rounding of h and their own, dx, dw_gate and dw_up that of dg and du and their own.  One
    # rounding of normally distributed numbers leaves 0.435 eps in the 2-norm (0.39 for significands spread evenly over
    # their logarithm), two independent ones 0.615; a third, of the factors, would make it 0.75, truncated bf16
    # factors more than 1.
    one = torch.randn(1 << 16, generator=torch.Generator().manual_seed(0))
    assert 0.42 * EPS < (one.bfloat16() - one).norm() / one.norm() < 0.45 * EPS
    x, wg, wu, wd, dy = make(M, D, F, E, 7)
    leaves = [t.to(dev).requires_grad_() for t in (x, wg, wu, wd)]
    y = lm.gated_mlp(*leaves, activation=act)
    grads = torch.autograd.grad(y, leaves, dy.to(dev))
    for got, (want, _), what in zip((y, *grads), reference(x, wg, wu, wd, dy, act),
                                    ("y", "dx", "dw_gate", "dw_up", "dw_down")):
        err = (xdna_train.as_cuda(got.detach()).double() - want).norm() / want.norm()
        assert err <= 0.7 * EPS, (what, err.item() / EPS)
