"""Operators of language models on the xdna device: token embedding, the gated
feed-forward block and the distillation loss.

Each function is one differentiable operator with its own sm_100a kernels
(``b2_embedding_*``, ``b2_gated_mlp_*``, ``b2_distill_*`` in
``include/b2.h``).  The reference has
no counterpart.  Their tensors live on one ``xdna`` device
(``xdna_train.as_xdna`` brings a CUDA tensor there without a copy) and the work
runs on its current stream.  On CPU tensors, and with ``set_npu_mode(0)``, the
same formulas run as plain torch operations.

Arguments a kernel does not take are refused with an error; an id outside the
vocabulary can only be seen on the device: it makes the values it touches NaN
and is reported by ``xdna_train.device_status()``.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

__all__ = ["embedding", "gated_mlp", "distill_loss"]

_ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2}
_REDUCTIONS = {"mean": 0, "sum": 1, "none": 2}


_C = None


def _native(t: torch.Tensor):
    """The extension when ``t`` runs on its kernels, else None (plain path)."""
    global _C
    if t.is_cpu:
        return None
    if _C is None:
        from . import device
        device.register_xdna_device()
        _C = device._C
    return _C if _C.npu_mode() > 0 else None


def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
              padding_idx: int | None = None) -> torch.Tensor:
    """``scale * weight[ids]``, shape ``ids.shape + (width,)``.

    ``weight``: ``[vocabulary, width]`` bfloat16 or float32 (rows may be
    strided); ``ids``: int32 or int64.  The gradient of ``weight`` is dense and
    summed in fp32 in a fixed order (the same bits on every run); the row of
    ``padding_idx`` gets none."""
    if padding_idx is not None and not 0 <= padding_idx < weight.shape[0]:
        raise ValueError(f"embedding: padding_idx {padding_idx} is outside the vocabulary of {weight.shape[0]}")
    C = _native(weight)
    if C is None:
        # through an fp32 table, so that the gradient is summed in fp32 and rounded once
        table = weight if weight.dtype == torch.float64 else weight.float()
        return (F.embedding(ids, table, padding_idx) * scale).to(weight.dtype)
    return C.lm_embedding(ids, weight, float(scale), -1 if padding_idx is None else int(padding_idx))


def gated_mlp(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
              activation: str = "silu") -> torch.Tensor:
    """``(act(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T``.

    ``x`` ``[..., D]``, ``w_gate`` and ``w_up`` ``[F, D]``, ``w_down``
    ``[E, F]`` (as ``nn.Linear`` keeps them), all bfloat16; the result is
    ``[..., E]``.  ``activation``: ``"silu"``, ``"gelu"`` (erf form) or
    ``"relu"``.  Sums are fp32; the hidden tensor is rounded to bfloat16
    between the products (of up to four tokens whose rows, and those of
    ``w_gate`` and ``w_up``, are 16-byte aligned, to two bfloat16 numbers), and
    the backward keeps it and the two factors ``act(gate)`` and
    ``up * act'(gate)`` (16 bits of significand): eight bytes a hidden element,
    saved as autograd's tensors.  Inside ``torch.autocast("xdna")`` other
    floating-point arguments are cast first, as for a matrix product."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"gated_mlp: activation must be one of {', '.join(_ACTIVATIONS)}, not {activation!r}")
    C = _native(x)
    if C is None:
        return F.linear(_ACT[activation](F.linear(x, w_gate)) * F.linear(x, w_up), w_down)
    if torch.is_autocast_enabled("xdna"):
        x, w_gate, w_up, w_down = (t.to(torch.bfloat16) for t in (x, w_gate, w_up, w_down))
    return C.lm_gated_mlp(x, w_gate, w_up, w_down, _ACTIVATIONS[activation])


_ACT = {"silu": F.silu, "gelu": F.gelu, "relu": F.relu}


def distill_loss(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_ids: torch.Tensor,
                 temperature: float = 1.0, row_weight: torch.Tensor | None = None,
                 reduction: str = "mean") -> torch.Tensor:
    """Distillation from a teacher's top logits.

    ``logits`` ``[..., V]`` (bfloat16 or float32) are the student's,
    ``teacher_logits`` and ``teacher_ids`` ``[..., K]`` the teacher's largest
    logits and their vocabulary ids (int32 or int64; a negative id marks an
    absent entry; K at most 1024).  With ``p = softmax(teacher_logits / T)``
    over a row's entries and ``q = softmax(logits / T)``, a row's loss is
    ``T**2 * sum(p * (log p - log q[ids]))``, 0 for a row without entries.
    ``row_weight`` ``[...]`` (float32) multiplies the rows; rows of weight 0
    are not read.  ``reduction``: ``"mean"`` (the weighted sum over the sum of
    the weights), ``"sum"`` or ``"none"``.  The loss is float32.

    With a gradient wanted, the pass that computes the loss also writes the
    gradient, so each logit is read once; teacher and weights are constants."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"distill_loss: reduction must be one of {', '.join(_REDUCTIONS)}, not {reduction!r}")
    C = _native(logits)
    if C is None:
        return _plain_distill_loss(logits, teacher_logits, teacher_ids, temperature, row_weight, reduction)
    return C.lm_distill_loss(logits, teacher_logits, teacher_ids, float(temperature), row_weight,
                             _REDUCTIONS[reduction])


def _plain_distill_loss(logits, teacher_logits, teacher_ids, temperature, row_weight, reduction):
    ids = teacher_ids.long()
    if ids.numel() and int(ids.max()) >= logits.shape[-1]:
        raise IndexError("distill_loss: teacher id outside the vocabulary")
    t = (teacher_logits.detach().float() / temperature).masked_fill(ids < 0, float("-inf"))
    has = t.new_zeros(t.shape[:-1] + (1,), dtype=torch.bool)
    if t.shape[-1]:
        has = (t != float("-inf")).any(-1, keepdim=True)  # (a NaN counts: it is not to go unseen)
    logp = torch.log_softmax(t.masked_fill(~has, 0.0), -1)
    p = torch.where(has, logp.exp(), 0.0)
    active = has if row_weight is None else has & (row_weight != 0).unsqueeze(-1)
    z = logits.float().masked_fill(~active, 0.0) / temperature
    logq = torch.log_softmax(z, -1).gather(-1, ids.clamp(min=0))
    keep = (p != 0) & active
    rows = temperature ** 2 * torch.where(keep, p * (logp.masked_fill(~keep, 0.0) - torch.where(keep, logq, 0.0)),
                                          0.0).sum(-1)
    w = torch.ones_like(rows) if row_weight is None else row_weight
    rows = torch.where(w != 0, rows * w, 0.0)
    if reduction == "none":
        return rows
    if reduction == "sum":
        return rows.sum()
    total = w.sum()
    return rows.sum() * torch.where(total != 0, 1.0 / total, 0.0)
