"""Distillation from a teacher's top logits, on the sm_100a kernels of csrc/distill:

  top_logits          the k largest logits of each row, their columns, and the row's log-sum-exp
  distillation_loss   the loss of a student's logits against such a list, differentiable

With a_i = t_i / tau over the teacher's listed columns c_i, q = softmax(z / tau) of the student's logits z and
q_rest the student's mass on all columns that are not listed:

  p_i  = exp(a_i - L),  L = teacher_lse (then m = 1 - sum p_i is the teacher's mass on the rest), or the
         log-sum-exp of the list itself (then m = 0: the teacher is renormalised over its list)
  KL   = sum_i p_i (log p_i - log q_{c_i}) + m (log m - log q_rest)
  loss = scale (kd_weight tau^2 KL + ce_weight (log sum_j exp z_j - z_target))

tau^2 keeps the gradient's size independent of the temperature (Hinton, Vinyals, Dean 2015, section 2.1).
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch

from ._ext import lib

MAX_TOP = 256
MAX_LIST = 1024
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


class TopLogits(NamedTuple):
    """``values`` (..., k) of the logits' type in descending order, ``ids`` int32 (..., k) their columns,
    ``lse`` fp32 (...) the log-sum-exp of the whole row over the temperature."""
    values: torch.Tensor
    ids: torch.Tensor
    lse: torch.Tensor


class Teacher(NamedTuple):
    """What a student learns from: lists for its (B, T) tokens and how the loss weighs them.  ``ids`` and
    ``values`` (B, T, k), ``lse`` (B, T) or None, as ``top_logits`` gives them at the same ``temperature``."""
    ids: torch.Tensor
    values: torch.Tensor
    lse: torch.Tensor | None = None
    temperature: float = 1.0
    kd_weight: float = 1.0
    ce_weight: float = 0.0

    def rows(self, start: int, end: int, device=None) -> "Teacher":
        """The lists of the sequences [start, end), on ``device``."""
        part = lambda t: None if t is None else t[start:end].to(device or t.device, non_blocking=True)  # noqa: E731
        return self._replace(ids=part(self.ids), values=part(self.values), lse=part(self.lse))


def factor_of(scale, count, reduction: str):
    """The loss' ``scale`` for this reduction over ``count`` targets (a device tensor): a mean's division belongs into it, so
    that a gradient of 16 bits is rounded once, after it."""
    if reduction == "sum":
        return scale
    inverse = count.clamp_min(1).double().reciprocal()
    if scale is None:
        return inverse
    return inverse * (scale.detach().reshape(()) if isinstance(scale, torch.Tensor) else float(scale))


def _rows(logits: torch.Tensor, what: str) -> torch.Tensor:
    """The logits as [N, V] rows with a unit column stride (a view where there is one)."""
    if not logits.is_cuda:
        raise ValueError(f"{what}: the logits must be a CUDA tensor")
    if logits.dtype not in _FLOATS:
        raise TypeError(f"{what}: the logits must be float32, bfloat16 or float16, not {logits.dtype}")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{what}: the logits need at least one column, not {tuple(logits.shape)}")
    if not lib().logits_row_fits(logits.shape[-1], logits.dtype):
        raise ValueError(f"{what}: rows of {logits.shape[-1]} logits exceed the shared memory of a cluster")
    rows = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    return rows if rows.stride(1) == 1 or rows.shape[1] == 1 else rows.contiguous()


@torch.no_grad()
def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0) -> TopLogits:
    """The ``k`` largest logits of each row (1 <= k <= 256), in descending order; equal logits by
    the lower column first; NaN counts as the largest value.  Not differentiable: it prepares a
    teacher's list.  ``lse`` is that of ``logits / temperature``, as ``distillation_loss`` takes it."""
    if not temperature > 0:
        raise ValueError(f"top_logits: the temperature must be positive, not {temperature}")
    rows = _rows(logits, "top_logits")
    if not 1 <= k <= min(MAX_TOP, rows.shape[1]):
        raise ValueError(f"top_logits: k must be between 1 and {min(MAX_TOP, rows.shape[1])}, not {k}")
    values, ids, lse = lib().top_logits(rows, int(k), float(temperature))
    if logits.dim() == 2:
        return TopLogits(values, ids, lse)
    lead = logits.shape[:-1]
    return TopLogits(values.view(*lead, k), ids.view(*lead, k), lse.view(lead))


def _flat(t, *shape):
    """``t`` as a dense tensor of this shape, itself where it is one already."""
    return t if t.shape == shape and t.is_contiguous() else t.reshape(shape).contiguous()


def _list_arguments(rows, teacher_ids, teacher_logits, teacher_lse, targets, ce_weight, scale):
    n = rows.shape[0]
    if teacher_ids.shape != teacher_logits.shape or teacher_ids.dim() < 1:
        raise ValueError(f"distillation_loss: teacher_ids {tuple(teacher_ids.shape)} and teacher_logits "
                         f"{tuple(teacher_logits.shape)} must have the same shape")
    k = teacher_ids.shape[-1]
    if not 1 <= k <= MAX_LIST:
        raise ValueError(f"distillation_loss: the list must have between 1 and {MAX_LIST} entries, not {k}")
    if teacher_ids.numel() != n * k:
        raise ValueError(f"distillation_loss: {teacher_ids.numel() // k} lists for {n} rows of logits")
    if teacher_ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"distillation_loss: teacher_ids must be int32 or int64, not {teacher_ids.dtype}")
    if teacher_logits.dtype not in _FLOATS:
        raise TypeError(f"distillation_loss: teacher_logits must be float32, bfloat16 or float16, not "
                        f"{teacher_logits.dtype}")
    if ce_weight != 0 and targets is None:
        raise ValueError("distillation_loss: the cross-entropy term needs targets")
    for name, value in (("teacher_lse", teacher_lse), ("targets", targets)):
        if value is not None and value.numel() != n:
            raise ValueError(f"distillation_loss: {name} has {value.numel()} elements for {n} rows")
    if teacher_lse is not None:
        teacher_lse = _flat(teacher_lse.detach().float(), n)
    if targets is not None:
        targets = _flat(targets, n)
    if scale is not None:
        if not isinstance(scale, torch.Tensor):
            scale = torch.full((1,), float(scale), device=rows.device)
        if scale.numel() != 1:
            raise ValueError(f"distillation_loss: scale must be one number, not {tuple(scale.shape)}")
        scale = scale.detach().float()
    return _flat(teacher_ids, n, k), _flat(teacher_logits.detach(), n, k), teacher_lse, targets, scale


def distillation_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                      teacher_lse: torch.Tensor | None = None, targets: torch.Tensor | None = None,
                      temperature: float = 1.0, kd_weight: float = 1.0, ce_weight: float = 0.0,
                      scale: torch.Tensor | float | None = None, reduction: str = "sum") -> torch.Tensor:
    """Loss of ``logits`` (..., V) against a teacher's lists, summed over rows or (``reduction="none"``) per row.

    ``teacher_ids`` / ``teacher_logits`` (..., k), 1 <= k <= 1024: columns (int32 or int64) and logits of the
    teacher, distinct columns in any order; an entry with a negative id is absent, and a row without entries
    has no divergence.  An id past the vocabulary is recorded in the status word (``ops._ext.check_status``)
    and counts as absent.  ``teacher_lse`` (...): the log-sum-exp of the teacher's whole row over the same
    temperature (``top_logits(...).lse``); without it the teacher is renormalised over its list.  A row where it is -inf (the
    teacher masked it throughout) has no divergence.
    ``targets`` (...) int64: rows with a negative target (-100) are left out entirely, loss and gradient zero;
    they are required when ``ce_weight`` is not 0.  ``scale`` (a number or a one-element tensor, e.g. one over
    the update's target count) multiplies loss and gradient inside the kernel, before the gradient is rounded
    to the logits' type, so that ``backward()`` has nothing left to do.

    Differentiable with respect to ``logits`` alone, once: the forward forms the gradient in the same pass over the
    logits and keeps it instead of them; the backward multiplies it by the incoming factor in place (fp16 logits are kept as
    well, and a factor other than 1, a loss scaler's for instance, takes another pass over them).  Second derivatives
    and forward-mode tangents are refused (``distillation_loss_reference`` has them).  A teacher's mass outside its
    list at or below 2^-20 counts as none (that is what rounding leaves of 1 - sum p)."""
    if not temperature > 0:
        raise ValueError(f"distillation_loss: the temperature must be positive, not {temperature}")
    if reduction not in ("sum", "none"):
        raise ValueError(f"distillation_loss: reduction must be 'sum' or 'none', not {reduction!r}")
    rows = _rows(logits, "distillation_loss")
    ids, t, teacher_lse, targets, scale = _list_arguments(rows, teacher_ids, teacher_logits, teacher_lse, targets,
                                                          ce_weight, scale)
    loss = lib().distillation(rows, ids, t, teacher_lse, targets, temperature, kd_weight, ce_weight, scale,
                              reduction == "sum")
    return loss if reduction == "sum" or logits.dim() == 2 else loss.view(logits.shape[:-1])


# ------------------------------------------------------------------------------------ plain forms
@torch.no_grad()
def top_logits_reference(logits: torch.Tensor, k: int, temperature: float = 1.0) -> TopLogits:
    """``top_logits`` in plain PyTorch (any device)."""
    values, ids = torch.sort(logits, dim=-1, descending=True, stable=True)
    wide = logits.to(torch.promote_types(logits.dtype, torch.float32))
    return TopLogits(values[..., :k], ids[..., :k].to(torch.int32), torch.logsumexp(wide / temperature, -1))


def distillation_loss_reference(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                                teacher_lse: torch.Tensor | None = None, targets: torch.Tensor | None = None,
                                temperature: float = 1.0, kd_weight: float = 1.0, ce_weight: float = 0.0,
                                scale=None, reduction: str = "sum") -> torch.Tensor:
    """``distillation_loss`` in plain PyTorch: any device, differentiable by autograd, in at least fp32 (an fp64
    student stays fp64).  The definition the kernels are tested against and the CPU path of the model."""
    z = logits.to(torch.promote_types(logits.dtype, torch.float32)).flatten(0, -2)
    n, v = z.shape
    ids = teacher_ids.reshape(n, -1).long()
    there = (ids >= 0) & (ids < v)
    at = torch.where(there, ids, 0)
    a = (teacher_logits.reshape(n, -1).to(z.dtype) / temperature).masked_fill(~there, -math.inf)
    norm = torch.logsumexp(a, 1) if teacher_lse is None else teacher_lse.reshape(n).to(z.dtype)
    some = there.any(1) & (norm != -math.inf)
    a = a.masked_fill(~some[:, None], -math.inf)
    logp = a - torch.where(some, norm, 0)[:, None]
    p = logp.exp()
    logq = torch.log_softmax(z / temperature, 1)
    kl = torch.where(p > 0, p * (logp - logq.gather(1, at)), 0).sum(1)
    if teacher_lse is not None:
        listed = torch.zeros(n, v + 1, dtype=torch.bool, device=z.device)
        listed = listed.scatter_(1, torch.where(there, ids, v), True)[:, :v]
        m = torch.where(some & ~listed.all(1), 1 - p.sum(1), 0)
        counts = m > 2.0 ** -20  # what rounding leaves of 1 - sum p is no mass
        rest = torch.logsumexp(logq.masked_fill(listed, -math.inf), 1)
        kl = kl + torch.where(counts, m * (m.clamp_min(2.0 ** -20).log() - torch.where(counts, rest, 0)), 0)
    loss = kd_weight * temperature ** 2 * kl
    if targets is not None:
        y = targets.reshape(n)
        live = (y >= 0) & (y < v)
        if ce_weight:
            ce = torch.log_softmax(z, 1).gather(1, torch.where(live, y, 0)[:, None]).squeeze(1)
            loss = loss - ce_weight * ce
        loss = torch.where(live, loss, 0)
    elif ce_weight:
        raise ValueError("distillation_loss: the cross-entropy term needs targets")
    if scale is not None:
        loss = loss * scale
    return loss.sum() if reduction == "sum" else loss.view(logits.shape[:-1])
