"""Cases of the language-model operators: token embedding, gated feed-forward block, distillation loss.

Every case is one pass through one operator, in its plain form (elementary torch operations in fp32, rounded once at
the end) or, with ``own`` set, through ``xdna_train.lm``.  ``listed`` has fixed cases from a single token to a large
training batch, ``draw`` gives further ones of the same ranges, ``work`` the bytes and operations a pass needs, and
``exact`` the same outputs from the definitions in fp64.

Operators (V: vocabulary, D: model width, F: hidden width):

embedding     y[t] = scale * W[ids[t]];  dW[v] = scale * sum of dy[t] over the tokens with ids[t] == v, in one dense
              gradient (the row of padding_idx stays zero)
gated_mlp     y = (act(x Wg^T) * (x Wu^T)) Wd^T with the gradients of x and the three weights
distill_loss  p = softmax over a row's teacher logits / tau (entries with a negative id are absent), q = softmax of all
              student logits / tau; the row's loss is tau^2 * sum_k p_k (log p_k - log q[id_k]), 0 for a row without
              teacher entries; "mean" divides the weighted sum by the sum of the row weights
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pytorch-xdna2_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import xdna_train
    return xdna_train


def listed():
    return [
        # the next tokens of 16 sequences being generated
        {"name": "embed_step", "op": "embedding", "tokens": 16, "vocab": 32768, "width": 1024, "dtype": "bf16",
         "train": False, "padding": False},
        # a small batch of ragged text with padding, fp32 master weights, sizes that no vector length divides
        {"name": "embed_train_odd", "op": "embedding", "tokens": 3001, "vocab": 50001, "width": 1001, "dtype": "fp32",
         "train": True, "padding": True},
        # a training batch of 16 sequences of 4096 tokens with a large vocabulary
        {"name": "embed_train_large", "op": "embedding", "tokens": 65536, "vocab": 131072, "width": 2048,
         "dtype": "bf16", "train": True, "padding": False},
        # one generated token
        {"name": "mlp_token", "op": "gated_mlp", "tokens": 1, "width": 1024, "hidden": 4096, "act": "silu",
         "train": False},
        # the next tokens of a few sequences, with a hidden width no tile divides
        {"name": "mlp_step_odd", "op": "gated_mlp", "tokens": 19, "width": 2048, "hidden": 5461, "act": "gelu",
         "train": False},
        # a training step at the batch and widths of the package's MLP benchmark
        {"name": "mlp_train", "op": "gated_mlp", "tokens": 512, "width": 1024, "hidden": 4096, "act": "silu",
         "train": True},
        # a ragged training batch: no size is a multiple of a tile or of a 16-byte vector
        {"name": "mlp_train_odd", "op": "gated_mlp", "tokens": 777, "width": 1001, "hidden": 2730, "act": "relu",
         "train": True},
        # two sequences of 4096 tokens through a wide layer
        {"name": "mlp_train_large", "op": "gated_mlp", "tokens": 8192, "width": 4096, "hidden": 12288, "act": "silu",
         "train": True},
        # scoring one token against a teacher's top 8
        {"name": "distill_token", "op": "distill_loss", "rows": 1, "vocab": 32768, "top": 8, "dtype": "bf16",
         "train": False, "tau": 1.0, "pad": 0},
        # a short fp32 batch whose logits are a view of a padded head, rows starting at any alignment
        {"name": "distill_train_odd", "op": "distill_loss", "rows": 301, "vocab": 50001, "top": 20, "dtype": "fp32",
         "train": True, "tau": 2.0, "pad": 15},
        # one sequence of 4096 tokens, prompt tokens masked
        {"name": "distill_train", "op": "distill_loss", "rows": 4096, "vocab": 32768, "top": 32, "dtype": "bf16",
         "train": True, "tau": 1.0, "pad": 0},
        # two sequences of 4096 tokens with a large vocabulary and many teacher entries
        {"name": "distill_train_large", "op": "distill_loss", "rows": 8192, "vocab": 131072, "top": 64,
         "dtype": "bf16", "train": True, "tau": 2.0, "pad": 0},
    ]


def _spread(rng, low, high, step=1):
    """A size between low and high, uniform in its logarithm; three times in four a multiple of `step`."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if step > 1 and rng.random() < 0.75:
        n = max(step, n // step * step)
    return min(max(n, low), high)


def draw(rng):
    op = rng.choice(["embedding", "gated_mlp", "distill_loss"])
    if op == "embedding":
        return {"op": op, "tokens": _spread(rng, 1, 65536), "vocab": _spread(rng, 1000, 131072, 64),
                "width": _spread(rng, 64, 2048, 8), "dtype": rng.choice(["bf16", "bf16", "fp32"]),
                "train": rng.random() < 0.7, "padding": rng.random() < 0.5}
    if op == "gated_mlp":
        return {"op": op, "tokens": _spread(rng, 1, 8192), "width": _spread(rng, 128, 4096, 8),
                "hidden": _spread(rng, 256, 12288, 8), "act": rng.choice(["silu", "gelu", "relu"]),
                "train": rng.random() < 0.6}
    return {"op": op, "rows": _spread(rng, 1, 8192), "vocab": _spread(rng, 1000, 131072, 64),
            "top": _spread(rng, 1, 256), "dtype": rng.choice(["bf16", "bf16", "fp32"]), "train": rng.random() < 0.7,
            "tau": rng.choice([1.0, 2.0, 0.7]), "pad": rng.choice([0, 0, 8, 15])}


# ---- inputs -------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    if case["op"] == "embedding":
        T, V, D, dt = case["tokens"], case["vocab"], case["width"], DTYPES[case["dtype"]]
        # word frequencies fall with the rank: P(id < k) = log(k + 1) / log(V + 1)
        ids = (torch.exp(uniform(T).double() * math.log(V + 1)) - 1).long().clamp_(0, V - 1)
        if case["padding"]:
            ids[uniform(T) < 0.1] = V - 1
        s.update(ids=ids, weight=normal(V, D, std=0.02, dtype=dt), scale=math.sqrt(D),
                 padding_idx=V - 1 if case["padding"] else None)
        if case["train"]:
            s["weight"].requires_grad_()
            s["dy"] = normal(T, D, std=1e-2, dtype=dt)
    elif case["op"] == "gated_mlp":
        M, D, F = case["tokens"], case["width"], case["hidden"]
        s.update(x=normal(M, D), w_gate=normal(F, D, std=D ** -0.5), w_up=normal(F, D, std=D ** -0.5),
                 w_down=normal(D, F, std=F ** -0.5), act=case["act"])
        if case["train"]:
            for k in ("x", "w_gate", "w_up", "w_down"):
                s[k].requires_grad_()
            s["dy"] = normal(M, D, std=1e-2)
    else:
        N, V, K, dt = case["rows"], case["vocab"], case["top"], DTYPES[case["dtype"]]
        # distinct ids: a random start and a random stride that stays within one turn of the vocabulary
        stride = (uniform(N, 1) * (V // K)).long().clamp_(min=1)
        ids = ((uniform(N, 1) * V).long() + torch.arange(K, device="cuda") * stride) % V
        teacher = (8.0 - 3.0 * uniform(N, K).cumsum(1)).to(dt)
        logits = torch.empty(N, V + case["pad"], dtype=dt, device="cuda")
        for a in range(0, N, 1024):  # drawn in blocks of rows: the fp32 normals of all rows would need twice the room
            logits[a:a + 1024] = normal(min(1024, N - a), V + case["pad"], std=2.0, dtype=dt)
        logits = logits[:, :V]
        rows = torch.arange(N, device="cuda").unsqueeze(1)
        logits[rows, ids] += (0.5 * teacher.float() + 3.0).clamp_(min=0.0).to(dt)  # a student that has learned some
        absent = uniform(N, K) < 0.05
        absent[uniform(N) < 0.02] = True  # rows whose teacher kept nothing
        teacher[uniform(N, K) < 0.02] = -math.inf
        if V > 2000:
            logits[:, V - 64:] = -math.inf  # vocabulary slots without a token
            absent |= ids >= V - 64
        s.update(logits=logits, teacher=teacher, ids=ids.masked_fill(absent, -1).int(), tau=case["tau"],
                 weight=(uniform(N) >= 0.15).float() if case["train"] else None)
        if case["train"]:
            s["logits"].requires_grad_()
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    xdna_train, case = _package(), s["case"]
    lm = xdna_train.lm

    def on(*names):  # the tensors on the package's device (the same memory), as leaves where a gradient is wanted
        return [None if s[k] is None else xdna_train.as_xdna(s[k].detach()).requires_grad_(s[k].requires_grad)
                for k in names]

    if case["op"] == "embedding":
        ids, w = on("ids", "weight")
        y = lm.embedding(ids, w, scale=s["scale"], padding_idx=s["padding_idx"])
        if not case["train"]:
            return {"y": y}
        (dw,) = torch.autograd.grad(y, [w], on("dy")[0])
        return {"y": y.detach(), "dw": dw}
    if case["op"] == "gated_mlp":
        leaves = on("x", "w_gate", "w_up", "w_down")
        y = lm.gated_mlp(*leaves, activation=s["act"])
        if not case["train"]:
            return {"y": y}
        dx, dg, du, dd = torch.autograd.grad(y, leaves, on("dy")[0])
        return {"y": y.detach(), "dx": dx, "dw_gate": dg, "dw_up": du, "dw_down": dd}
    z, t, ids, w = on("logits", "teacher", "ids", "weight")
    if not case["train"]:
        return {"loss": lm.distill_loss(z, t, ids, temperature=s["tau"], reduction="none")}
    loss = lm.distill_loss(z, t, ids, temperature=s["tau"], row_weight=w)
    (dz,) = torch.autograd.grad(loss, [z])
    return {"loss": loss.detach(), "dlogits": dz}


@torch.no_grad()
def _plain(s):
    case = s["case"]
    if case["op"] == "embedding":
        w = s["weight"]
        y = (w[s["ids"]].float() * s["scale"]).to(w.dtype)
        if not case["train"]:
            return {"y": y}
        dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
        dw.index_add_(0, s["ids"], s["dy"].float() * s["scale"])
        if s["padding_idx"] is not None:
            dw[s["padding_idx"]] = 0.0
        return {"y": y, "dw": dw.to(w.dtype)}
    if case["op"] == "gated_mlp":
        x, wg, wu, wd = (s[k].float() for k in ("x", "w_gate", "w_up", "w_down"))
        g, u = x @ wg.t(), x @ wu.t()
        if s["act"] == "silu":
            sig = 1.0 / (1.0 + torch.exp(-g))
            a, slope = g * sig, sig * (1.0 + g * (1.0 - sig))
        elif s["act"] == "gelu":
            cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
            a, slope = g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
        else:
            slope = (g > 0).float()
            a = g * slope
        h = a * u
        bf = torch.bfloat16
        y = (h @ wd.t()).to(bf)
        if not case["train"]:
            return {"y": y}
        dy = s["dy"].float()
        dh = dy @ wd
        dg, du = dh * u * slope, dh * a
        return {"y": y, "dx": (dg @ wg + du @ wu).to(bf), "dw_gate": (dg.t() @ x).to(bf),
                "dw_up": (du.t() @ x).to(bf), "dw_down": (dy.t() @ h).to(bf)}
    tau, ids, dt = s["tau"], s["ids"].long(), s["logits"].dtype
    z = s["logits"].float() / tau
    z -= z.amax(1, keepdim=True)
    q = torch.exp(z)
    total = q.sum(1, keepdim=True)
    t = torch.where(ids >= 0, s["teacher"].float() / tau, -math.inf)
    top = t.amax(1, keepdim=True)
    p = torch.exp(t - torch.where(top > -math.inf, top, 0.0))
    mass = p.sum(1, keepdim=True)
    p = p / torch.where(mass > 0, mass, 1.0)
    at = ids.clamp(min=0)
    term = p * (torch.log(p) - (z.gather(1, at) - torch.log(total)))
    rows = tau * tau * torch.where(p > 0, term, 0.0).sum(1)
    if not case["train"]:
        return {"loss": rows}
    w = s["weight"] / s["weight"].sum().clamp(min=1e-30)
    q *= (p.sum(1, keepdim=True) * tau * w.unsqueeze(1)) / total
    q.scatter_add_(1, at, -tau * w.unsqueeze(1) * p)
    return {"loss": (rows * w).sum(), "dlogits": q.to(dt)}


# ---- work ---------------------------------------------------------------------------------------------------------

def work(case):
    if case["op"] == "embedding":
        T, V, D, size = case["tokens"], case["vocab"], case["width"], 2 if case["dtype"] == "bf16" else 4
        k = np.arange(V, dtype=np.float64)
        distinct = float((1.0 - (1.0 - np.log((k + 2) / (k + 1)) / math.log(V + 1)) ** T).sum())
        rows = distinct + T  # rows read and written by the lookup
        if case["train"]:
            rows += T + V    # gradient rows read, dense gradient written
        return {"bytes": rows * D * size + 8 * T, "flops": T * D * (2 if case["train"] else 1)}
    if case["op"] == "gated_mlp":
        M, D, F = case["tokens"], case["width"], case["hidden"]
        if not case["train"]:
            return {"bytes": 2 * (2 * M * D + 3 * D * F), "flops": 6 * M * D * F}
        return {"bytes": 2 * (4 * M * D + 6 * D * F), "flops": 18 * M * D * F}
    N, V, K, size = case["rows"], case["vocab"], case["top"], 2 if case["dtype"] == "bf16" else 4
    if not case["train"]:
        return {"bytes": N * (V * size + K * (size + 4) + 4), "flops": 4 * N * V}
    return {"bytes": N * (2 * V * size + K * (size + 4) + 4) + 4, "flops": 6 * N * V}


# ---- the definitions in fp64 --------------------------------------------------------------------------------------

@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    f8 = torch.float64
    if case["op"] == "embedding":
        ids, scale, w = s["ids"], s["scale"], s["weight"]
        y = w.index_select(0, ids).to(f8).mul_(scale)
        if not case["train"]:
            return {"y": y}
        # tokens grouped by id: the sums of a group are differences of running sums, taken per column block
        order = torch.argsort(ids, stable=True)
        found, counts = torch.unique_consecutive(ids[order], return_counts=True)
        ends = counts.cumsum(0)
        dw = torch.zeros(w.shape, dtype=f8, device=w.device)
        for c in range(0, w.shape[1], 256):
            run_sum = s["dy"][:, c:c + 256][order].to(f8).cumsum(0)[ends - 1]
            dw[found, c:c + 256] = torch.diff(run_sum, dim=0, prepend=torch.zeros_like(run_sum[:1])) * scale
        if s["padding_idx"] is not None:
            dw[s["padding_idx"]] = 0
        return {"y": y, "dw": dw}
    if case["op"] == "gated_mlp":
        leaves = [s[k].detach().to(f8).requires_grad_(case["train"]) for k in ("x", "w_gate", "w_up", "w_down")]
        x, wg, wu, wd = leaves
        with torch.enable_grad():
            g = torch.einsum("md,fd->mf", x, wg)
            act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu}[case["act"]]
            y = torch.einsum("mf,df->md", act(g) * torch.einsum("md,fd->mf", x, wu), wd)
            if not case["train"]:
                return {"y": y}
            grads = torch.autograd.grad(y, leaves, s["dy"].to(f8))
        return dict(zip(("y", "dx", "dw_gate", "dw_up", "dw_down"), (y.detach(),) + grads))
    tau, V = s["tau"], case["vocab"]
    w = None if s["weight"] is None else s["weight"].to(f8) / max(float(s["weight"].sum()), 1e-30)
    losses, grads = [], []
    for a in range(0, case["rows"], 1024):
        ids = s["ids"][a:a + 1024].long()
        kept = ids >= 0
        logq = torch.log_softmax(s["logits"][a:a + 1024].to(f8) / tau, dim=1)
        t = (s["teacher"][a:a + 1024].to(f8) / tau).masked_fill(~kept, -math.inf)
        logp = torch.log_softmax(t, dim=1)
        p = torch.where(logp > -math.inf, logp.exp(), 0.0)  # a row with no entries is NaN there: no probability
        gap = torch.where(p > 0, logp, 0.0) - torch.where(p > 0, logq.gather(1, ids.clamp(min=0)), 0.0)
        losses.append(tau ** 2 * (p * gap).sum(1))
        if case["train"]:
            full = torch.zeros(len(ids), V, dtype=f8, device=ids.device).scatter_add_(1, ids.clamp(min=0), p)
            grads.append(logq.exp_().mul_(p.sum(1, keepdim=True)).sub_(full).mul_(tau * w[a:a + 1024, None]))
    loss = torch.cat(losses)
    if not case["train"]:
        return {"loss": loss}
    return {"loss": (loss * w).sum(), "dlogits": torch.cat(grads)}
