"""Operators on a classifier's logits (kernels: ops/csrc/logit_kernels.hip).

``label_logprobs``: log probability of a given class, entropy and top
alternatives of each row, in one call.  ``PSTrainer.evaluate(entropy=True)``
and the checkpoint evaluator read loss, prec@1, prec@5 and entropy from it; a
teacher's alternatives feed ``distill_loss``.

``distill_loss``: a student's loss against a teacher's top logits, mixed with
the cross entropy of the labels, and its gradient.  With q the softmax of the
teacher's K values at temperature tau (the K alone; entries of one class are
added up) and p_tau the student's over all classes:

    row = weight * tau^2 * sum_c q_c (log q_c - log p_tau_c)
          + (1 - weight) * -log p_1[label]

CUDA (= ROCm) tensors take the HIP kernels, CPU tensors the torch oracle below
(64-bit inside).  Both compute in at least 32 bits and round the gradient once.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from . import ext

# the most alternatives, or teacher's entries, of one row
TOP_MAX = 128

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


class LabelLogprobs(NamedTuple):
    """What ``label_logprobs`` returns; entries that were not asked for are
    None."""

    logprob: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_logprob: Optional[torch.Tensor]
    top_index: Optional[torch.Tensor]


def _rows(logits: torch.Tensor) -> torch.Tensor:
    if logits.dtype not in _FLOATS:
        raise TypeError(f"logits must be fp32, bf16 or fp16, not {logits.dtype}")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("logits must be (..., classes) with a class at least")
    z = logits
    if z.dim() != 2:
        z = z.reshape(math.prod(z.shape[:-1]), z.shape[-1])
    if z.shape[1] > 1 and z.stride(1) != 1:
        z = z.contiguous()
    return z


def _int_rows(t: torch.Tensor, shape, device, name: str) -> torch.Tensor:
    if t.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{name} must be int64 or int32, not {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {tuple(shape)}, not {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, logits on {device}")
    return t.to(torch.int64).contiguous()


def label_logprobs(
    logits: torch.Tensor,
    labels: Optional[torch.Tensor] = None,
    top: int = 0,
    ignore_index: int = -100,
) -> LabelLogprobs:
    """Log probabilities of ``labels``, entropies, and the ``top`` likeliest
    classes of the rows of ``logits`` (..., classes).

    ``labels`` (...), int64 or int32, may be left out.  A label of
    ``ignore_index`` gives 0, any other outside 0..classes-1 gives NaN.
    ``top`` is at most min(classes, 128); equal logits are ordered by class,
    the lowest first, and NaN counts as the greatest.  Classes at -inf have
    probability 0; a row of nothing else gives log probabilities of -inf and
    an entropy of 0; a row with NaN or +inf gives NaN.  Results are fp32 and
    int64 whatever the logits' type, and carry no gradient.  Rows may be
    strided; classes that are not contiguous are copied first.
    """
    z = _rows(logits.detach())
    lead = logits.shape[:-1]
    top = int(top)
    if not 0 <= top <= min(z.shape[1], TOP_MAX):
        raise ValueError(
            f"top must lie in 0..min(classes, {TOP_MAX}), not {top}")
    y = None
    if labels is not None:
        y = _int_rows(labels, lead, logits.device, "labels").reshape(-1)
    if z.is_cuda:
        out = ext().label_logprobs(z, y, top, int(ignore_index))
    else:
        out = _label_logprobs_oracle(z, y, top, int(ignore_index))
    logprob, entropy, top_logprob, top_index = out
    if len(lead) != 1:
        logprob = logprob if logprob is None else logprob.view(lead)
        entropy = entropy.view(lead)
        top_logprob = top_logprob.view(*lead, top)
        top_index = top_index.view(*lead, top)
    if top == 0:
        top_logprob = top_index = None
    return LabelLogprobs(logprob, entropy, top_logprob, top_index)


def distill_loss(
    logits: torch.Tensor,
    teacher_value: torch.Tensor,
    teacher_index: torch.Tensor,
    labels: Optional[torch.Tensor] = None,
    temperature: float = 1.0,
    weight: float = 1.0,
    ignore_index: int = -100,
    reduction: str = "mean",
) -> torch.Tensor:
    """Loss of ``logits`` (..., classes) against a teacher's top logits
    ``teacher_value`` (..., k) at the classes ``teacher_index`` (..., k), with
    ``weight``, and against ``labels`` (...) with ``1 - weight``.

    ``temperature`` lies in 0.01..100.  The values may be logits or log
    probabilities: a constant added to a row changes nothing.  k is at
    most 128; an entry of -inf is absent, and its index is not looked at.  Any
    other index outside 0..classes-1 makes the row NaN, its gradient too, as do
    a value of NaN or +inf and such a label, except ``ignore_index``: that row has
    no loss, no gradient, and is not counted in the mean (of no rows: 0).
    ``labels`` may be given with ``weight=1`` to leave rows out, and has to be
    with any other weight; with ``weight=0`` the teacher is not looked at.
    A teacher's row of absent entries adds nothing, a student's row of -inf
    has loss and gradient 0.  The loss is fp32 (reduction "none": one a row),
    the gradient has the logits' type; the teacher gets none.  The gradient
    cannot be differentiated again.
    """
    z = _rows(logits)
    lead = logits.shape[:-1]
    if teacher_value.dtype not in _FLOATS:
        raise TypeError(
            f"teacher_value must be fp32, bf16 or fp16, not {teacher_value.dtype}")
    if (teacher_value.dim() != logits.dim()
            or teacher_value.shape[:-1] != lead):
        raise ValueError(
            f"teacher_value must be {(*lead, 'k')}, not {tuple(teacher_value.shape)}")
    k = teacher_value.shape[-1]
    if not 1 <= k <= TOP_MAX:
        raise ValueError(f"a teacher's row holds 1..{TOP_MAX} entries, not {k}")
    if teacher_value.device != logits.device:
        raise ValueError(
            f"teacher_value is on {teacher_value.device}, logits on {logits.device}")
    index = _int_rows(teacher_index, teacher_value.shape, logits.device,
                      "teacher_index").view(-1, k)
    value = teacher_value.detach().float().contiguous().view(-1, k)
    temperature, weight = float(temperature), float(weight)
    if not 0.01 <= temperature <= 100.0:
        # tau^2 times what 32 bits lose of a distribution at tau
        raise ValueError(f"temperature must lie in 0.01..100, not {temperature}")
    if not 0.0 <= weight <= 1.0:
        raise ValueError(f"weight must lie in 0..1, not {weight}")
    if labels is None and weight != 1.0:
        raise ValueError("a weight below 1 needs labels")
    if reduction not in _REDUCTIONS:
        raise ValueError(
            f"reduction must be one of {sorted(_REDUCTIONS)}, not {reduction!r}")
    y = None
    if labels is not None:
        y = _int_rows(labels, lead, logits.device, "labels").reshape(-1)
    args = (z, value, index, y, temperature, weight, int(ignore_index),
            _REDUCTIONS[reduction])
    if z.is_cuda:
        loss = ext().distill_loss(*args)
    else:
        loss = _DistillOracle.apply(*args)
    if reduction == "none" and len(lead) != 1:
        loss = loss.view(lead)
    return loss


# ---------------------------------------------------------------------------
# the oracle
# ---------------------------------------------------------------------------
def _log_softmax(z: torch.Tensor) -> torch.Tensor:
    """log softmax in 64 bits; -inf throughout where a row is -inf."""
    z = z.double()
    empty = (z == -math.inf).all(1, keepdim=True)
    out = torch.log_softmax(z.masked_fill(empty, 0.0), 1)
    out = out.masked_fill(empty, -math.inf)
    # +inf and NaN anywhere make the row NaN
    return out + torch.where(z.amax(1, keepdim=True) < math.inf, 0.0, math.nan)


def _times(p: torch.Tensor, log: torch.Tensor) -> torch.Tensor:
    """p * log with 0 * -inf = 0."""
    return torch.where(p == 0.0, torch.zeros_like(p), p * log)


def _label_logprobs_oracle(z, y, top, ignore):
    logp = _log_softmax(z)
    entropy = -_times(logp.exp(), logp).sum(1)
    entropy = torch.where((z == -math.inf).all(1), 0.0, entropy)
    logprob = None
    if y is not None:
        inside = (y >= 0) & (y < z.shape[1])
        logprob = logp.gather(1, torch.where(inside, y, 0)[:, None])[:, 0]
        logprob = torch.where(inside, logprob, math.nan)
        logprob = torch.where(y == ignore, 0.0, logprob).float()
    # a stable sort leaves equal values in the order of their class
    order = torch.where(z.isnan(), math.inf, z.double())
    top_index = torch.stack(
        [z.isnan().double(), order], 0)
    first = torch.sort(top_index[1], dim=1, descending=True, stable=True).indices
    nan_first = torch.sort(top_index[0].gather(1, first), dim=1,
                           descending=True, stable=True).indices
    index = first.gather(1, nan_first)[:, :top].contiguous()
    return logprob, entropy.float(), logp.gather(1, index).float(), index


class _DistillOracle(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, value, index, y, tau, weight, ignore, reduction):
        rows, classes = z.shape
        empty = (z == -math.inf).all(1)
        counted = torch.ones(rows, dtype=torch.bool)
        if y is not None:
            counted = y != ignore
        row = torch.zeros(rows, dtype=torch.float64)
        grad = torch.zeros(rows, classes, dtype=torch.float64)
        if weight > 0.0:
            there = value != -math.inf
            inside = (index >= 0) & (index < classes)
            t = _log_softmax(value.double() / tau)
            q = torch.zeros(rows, classes, dtype=torch.float64)
            q.scatter_add_(1, torch.where(inside & there, index, 0),
                           torch.where(inside & there, t.exp(), 0.0))
            log_p = _log_softmax(z.double() / tau)
            kd = (_times(q, q.log()) - _times(q, log_p)).sum(1)
            bad = torch.where((there & ~inside).any(1), math.nan, 0.0)
            bad = bad + torch.where(t.isnan().any(1), math.nan, 0.0)
            any_q = there.any(1, keepdim=True)
            row += weight * tau * tau * (kd + bad)
            grad += weight * tau * (
                torch.where(any_q, log_p.exp(), 0.0) - q + bad[:, None])
        if y is not None and weight < 1.0:
            inside = (y >= 0) & (y < classes)
            at = torch.where(inside, y, 0)[:, None]
            log_p = _log_softmax(z)
            bad = torch.where(inside, 0.0, math.nan)
            row += (1.0 - weight) * (bad - log_p.gather(1, at)[:, 0])
            grad += (1.0 - weight) * (log_p.exp() + bad[:, None])
            grad.scatter_add_(1, at, torch.full(
                (rows, 1), weight - 1.0, dtype=torch.float64))
        off = ~counted | empty
        row = torch.where(off, 0.0, row)
        grad = torch.where(off[:, None], 0.0, grad)
        ctx.kind = z.dtype
        ctx.save_for_backward(grad)
        ctx.factor = 1.0
        if reduction == 0:
            return row.float()
        if reduction == 1:
            ctx.factor = 1.0 / max(1, int(counted.sum()))
        return (row.sum() * ctx.factor).float()

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, up):
        (grad,) = ctx.saved_tensors
        up = up.double() * ctx.factor
        if up.dim():
            up = up[:, None]
        grad = (grad * up).to(ctx.kind)
        return grad, None, None, None, None, None, None, None
