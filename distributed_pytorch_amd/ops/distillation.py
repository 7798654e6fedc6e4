"""Distillation from a teacher's top logits, mixed with the cross-entropy of hard labels.

The reference trains on hard labels only (``nn.CrossEntropyLoss``, reference min_DDP.py:75,100).  A teacher's answer for a
token is stored as its K largest logits with their classes; the student learns their softmax:

    p = softmax(t / tau) over the K entries       q = softmax(z / tau), q1 = softmax(z) over all classes
    loss_r = (1 - a) tau^2 sum_k p_k (log p_k - log q[id_k])  -  a log q1[target]        (a = hard_weight, tau = temperature)

``topk_distillation`` takes the student's logits, ``projection_topk_distillation`` the input and the weight of the
vocabulary projection (the logits then exist only inside the op, in float32 whatever the tensors' type, so that the loss is as exact as that
of float32 logits).  On gfx950 the loss and the gradient of the logits come out of one kernel that reads each row
once.  An entry whose id is negative or not below ``n_classes``, or whose logit is ``-inf``, is absent; entries may come
in any order, and entries of one class add up.  No gradient reaches the teacher.  Rows whose target is ``ignore_index`` count for nothing and may hold
anything; a row without entries keeps its hard term.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from .. import _ext
from . import gemm
from .cross_entropy import _want_target_check, check_targets_in_range


class DistillResult(NamedTuple):
    loss: torch.Tensor      # scalar (mean / sum) or [N] (reduction='none'), float32
    correct: torch.Tensor   # bool [N]: the student's largest logit is the target (without targets: the teacher's first choice)
    metrics: torch.Tensor   # float32 [4]: loss sum, correct count, counted rows, mean loss


class _TopKDistillation(torch.autograd.Function):
    """Mean and sum: the forward also writes the gradient for a unit upstream gradient, so that the logits are read once
    for both; the backward scales it where the upstream gradient is another one (told apart on the device).  That
    gradient is handed over by the first backward; a second one through a retained graph computes it again.

    Not so in fp16: divided by the number of rows, most of that gradient is below the type's smallest value, and the upstream gradient -- a loss
    scale -- would come too late.  The backward then computes it from the logits with the upstream gradient as a factor ahead of the rounding."""

    @staticmethod
    def forward(ctx, logits, ids, teacher, targets, cfg):
        reduction, ignore_index, n_classes, temperature, hard_weight = cfg
        C = _ext.C()
        ctx.set_materialize_grads(False)  # (of the two by-products: zeros that nobody reads)
        mean = reduction == "mean"
        ctx.cfg = cfg
        ctx.needs = ctx.needs_input_grad[0]
        fused = ctx.needs and reduction != "none" and logits.dtype != torch.float16
        loss, row_loss, correct, metrics, scale, stats, dlogits = C.distill_forward(
            logits, ids, teacher, targets, n_classes, ignore_index, temperature, hard_weight, mean, "new" if fused else "none")
        ctx.dlogits, ctx.scale = dlogits, scale
        ctx.save_for_backward(logits, ids, teacher, targets, stats)
        ctx.mark_non_differentiable(correct, metrics)
        return (row_loss if reduction == "none" else loss), correct, metrics

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _dcorrect, _dmetrics):
        if dloss is None:
            return (None,) * 5
        C = _ext.C()
        g = dloss.detach().to(torch.float32).contiguous()
        logits, ids, teacher, targets, stats = ctx.saved_tensors
        if ctx.dlogits is not None:
            d, ctx.dlogits = ctx.dlogits, None
            C.distill_apply_upstream(d, g)
            return d, None, None, None, None
        reduction, ignore_index, n_classes, temperature, hard_weight = ctx.cfg
        if stats is None:
            stats = C.distill_forward(logits, ids, teacher, targets, n_classes, ignore_index, temperature, hard_weight, reduction == "mean", "none")[5]
        d = C.distill_backward(logits, ids, teacher, targets, stats, ctx.scale, g, n_classes, ignore_index, temperature, hard_weight, reduction == "mean")
        return d, None, None, None, None


class _ProjectionTopKDistillation(torch.autograd.Function):
    """Vocabulary projection and loss as one node, whose backward is two matrix products of the logits' gradient (see
    ``cross_entropy._ProjectionXent``).  The logits are float32 whatever the tensors' type, as the loss is: in fp32 the kernel that computes the
    loss overwrites them with their gradient, in bf16 it writes the gradient beside them and they go.  In fp16 they stay and the
    backward computes their gradient, for the reason given above."""

    @staticmethod
    def forward(ctx, x2, weight, ids, teacher, targets, cfg, impl, grad):
        reduction, ignore_index, n_classes, temperature, hard_weight = cfg
        ctx.set_materialize_grads(False)
        C = _ext.C()
        args = (ids, teacher, targets, n_classes, ignore_index, temperature, hard_weight, reduction == "mean")
        half = x2.dtype == torch.float16
        impl = "strict" if impl == "native" else impl
        if impl == "strict" and x2.dtype != torch.float32:
            loss, correct, metrics, scale, stats, logits, dlogits = C.projection_distill_forward(
                x2, weight, *args, "none" if not grad else "logits" if half else "gradient")
        else:
            logits = gemm.nt(x2, weight, None, impl)
            loss, _, correct, metrics, scale, stats, dlogits = C.distill_forward(logits, *args, "inplace" if grad and not half else "none")
        if grad and half:
            ctx.save_for_backward(x2, weight, logits, ids, teacher, targets, scale, stats)
        elif grad:
            ctx.save_for_backward(x2, weight, dlogits)  # for a unit upstream gradient
        ctx.impl, ctx.half, ctx.cfg = impl, half, cfg
        ctx.mark_non_differentiable(correct, metrics)
        return loss, correct, metrics

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _dcorrect, _dmetrics):
        if dloss is None:
            return (None,) * 8
        g = dloss.detach().to(torch.float32).reshape(())
        C = _ext.C()
        if ctx.half:
            x2, weight, logits, ids, teacher, targets, scale, stats = ctx.saved_tensors
            reduction, ignore_index, n_classes, temperature, hard_weight = ctx.cfg
            dlogits = C.distill_backward(logits, ids, teacher, targets, stats, scale, g, n_classes, ignore_index, temperature, hard_weight,
                                         reduction == "mean", weight.shape[0] if logits.dtype == torch.float32 else 0)
        else:
            x2, weight, dlogits = ctx.saved_tensors
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dx = gemm.nn(dlogits, weight, ctx.impl)
            if not ctx.half:
                C.distill_apply_upstream(dx, g)
        if ctx.needs_input_grad[1]:
            dw = gemm.weight_grad(dlogits, x2, weight, ctx.impl)
            if not ctx.half:
                C.distill_apply_upstream(dw, g)
        return dx, dw, None, None, None, None, None, None


def _check(N: int, n_classes: int, width: int, ids, teacher, targets, temperature: float, hard_weight: float, reduction: str, allowed) -> None:
    if reduction not in allowed:
        raise ValueError(f"reduction must be {' | '.join(allowed)}, got {reduction}")
    if not 1e-12 <= temperature <= 1e12:  # (float32 holds its reciprocal, and its square times any number of rows)
        raise ValueError(f"temperature must lie in 1e-12 .. 1e12, got {temperature}")
    if not 0.0 <= hard_weight <= 1.0:
        raise ValueError(f"hard_weight must lie in [0, 1], got {hard_weight}")
    if hard_weight > 0 and targets is None:
        raise ValueError("hard_weight > 0 needs targets")
    if not 1 <= n_classes <= width:
        raise ValueError(f"n_classes must lie in 1 .. {width}, got {n_classes}")
    if ids.dim() != 2 or ids.shape != teacher.shape or ids.shape[0] != N or ids.shape[1] < 1:
        raise ValueError(f"teacher_ids and teacher_logits must both be [{N}, K], got {tuple(ids.shape)} and {tuple(teacher.shape)}")
    if ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"teacher_ids must be int64 or int32, got {ids.dtype}")
    if not teacher.is_floating_point():
        raise ValueError(f"teacher_logits must be floating point, got {teacher.dtype}")
    if targets is not None and (targets.shape != (N,) or targets.dtype != torch.int64):
        raise ValueError(f"targets must be int64 [{N}], got {targets.dtype} {tuple(targets.shape)}")


def _check_ids(ids: torch.Tensor, n_classes: int) -> None:
    if bool((ids >= n_classes).any()):
        raise IndexError(f"teacher id {int(ids[ids >= n_classes][0])} is out of bounds (classes 0..{n_classes - 1}, negative = no entry)")


def _composed(logits, ids, teacher, targets, cfg) -> DistillResult:
    """The same loss out of stock operators (CPU tensors)."""
    reduction, ignore_index, n_classes, temperature, hard_weight = cfg
    z = logits[:, :n_classes]
    z = z if z.dtype == torch.float64 else z.float()
    N = z.shape[0]
    counted = torch.ones(N, dtype=torch.bool, device=z.device) if targets is None else targets != ignore_index
    live = counted if targets is None else counted & (targets >= 0) & (targets < n_classes)
    z = torch.where(live.unsqueeze(1), z, z.new_zeros(()))  # an ignored row may hold anything
    row = z.new_zeros(N)
    t = teacher.detach().to(z.dtype)
    there = (ids >= 0) & (ids < n_classes) & (t != float("-inf"))
    if hard_weight < 1:
        at = torch.where(there, ids, 0).long()
        # Divided by the temperature as differences to the largest, which the type's lowest value survives; a finite stand-in for "absent" keeps
        # rows without entries out of inf - inf.
        top = torch.where(there, t, float("-inf")).amax(1, keepdim=True)
        top = torch.where(there.any(1, keepdim=True), top, 0.0)
        log_p = torch.log_softmax(torch.where(there, (t - top) / temperature, t.new_full((), torch.finfo(t.dtype).min)), 1)
        p = torch.where(there, log_p.exp(), 0.0)
        term = p * (log_p - torch.log_softmax(z / temperature, 1).gather(1, at))
        row = row + (1 - hard_weight) * temperature ** 2 * torch.where(p > 0, term, 0.0).sum(1)
    if hard_weight > 0:
        row = row + hard_weight * F.cross_entropy(z, torch.where(live, targets, 0), reduction="none")
    row = torch.where(live, row, 0.0)
    best = z.argmax(1)
    if targets is not None:
        correct = (best == targets) & live
    else:
        first = torch.where(there, t, float("-inf")).argmax(1, keepdim=True)
        correct = (best == ids.gather(1, first).squeeze(1)) & there.any(1)
    n = counted.sum().clamp(min=1)
    metrics = torch.stack([row.sum(), correct.sum().to(row.dtype), counted.sum().to(row.dtype), row.sum() / n]).detach().float()
    loss = row.sum() / n if reduction == "mean" else (row.sum() if reduction == "sum" else row)
    return DistillResult(loss, correct, metrics)


def topk_distillation(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, targets: Optional[torch.Tensor] = None,
                      temperature: float = 1.0, hard_weight: float = 0.0, reduction: str = "mean", ignore_index: int = -100,
                      n_classes: Optional[int] = None, check_targets: Optional[bool] = None) -> DistillResult:
    """Distillation loss of ``logits[N, C]`` against a teacher's entries ``teacher_ids[N, K]`` / ``teacher_logits[N, K]``
    (on the GPU K <= 1024 and C <= 2 ** 20), see the module's description.

    ``targets[N]`` give the hard term (weight ``hard_weight``) and mark ignored rows; the mean is taken over rows whose
    target is not ``ignore_index`` (over all rows without targets).  ``n_classes`` < C marks trailing columns as padding:
    they take no part and get zero gradient.  ``temperature`` lies in 1e-12 .. 1e12, and logits divided by it are taken to stay below 2 ** 24
    in size, beyond which float32 tells no neighbouring ones apart.  ``check_targets`` (or ``DIST_CHECK_TARGETS=1``) raises ``IndexError`` for
    a target or a teacher id beyond the classes, at the price of a host synchronisation.
    """
    if logits.dim() != 2:
        raise ValueError("topk_distillation expects logits of shape [N, C]")
    nc = logits.shape[1] if n_classes is None else int(n_classes)
    _check(logits.shape[0], nc, logits.shape[1], teacher_ids, teacher_logits, targets, temperature, hard_weight, reduction, ("mean", "sum", "none"))
    if _want_target_check(check_targets):
        _check_ids(teacher_ids, nc)
        if targets is not None:
            check_targets_in_range(targets, nc, ignore_index)
    cfg = (reduction, ignore_index, nc, float(temperature), float(hard_weight))
    if not logits.is_cuda:
        return _composed(logits, teacher_ids, teacher_logits, targets, cfg)
    logits = logits if logits.is_contiguous() and logits.data_ptr() % 16 == 0 else logits.clone(memory_format=torch.contiguous_format)
    teacher = teacher_logits.detach()
    teacher = teacher if teacher.dtype in (torch.float32, torch.bfloat16, torch.float16) else teacher.float()
    loss, correct, metrics = _TopKDistillation.apply(logits, teacher_ids.contiguous(), teacher.contiguous(),
                                                     None if targets is None else targets.contiguous(), cfg)
    return DistillResult(loss, correct, metrics)


def projection_topk_distillation(x: torch.Tensor, weight: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                                 targets: Optional[torch.Tensor] = None, temperature: float = 1.0, hard_weight: float = 0.0,
                                 reduction: str = "mean", ignore_index: int = -100, n_classes: Optional[int] = None, impl: str = "native",
                                 check_targets: Optional[bool] = None) -> DistillResult:
    """``topk_distillation`` of the logits ``x @ weight.T`` (``x``: [..., K_in], ``weight``: [C, K_in]; the teacher's tensors
    are [..., K] and ``targets`` [...] over the same leading dimensions).  reduction: mean | sum.  Ignored rows of ``x`` may hold anything
    finite (the weight's gradient is a product with all of ``x``).

    bf16 training keeps the logits' gradient (2 bytes each) until the backward, beside some rows of float32 logits in passing (8 GiB at
    most); fp16 training keeps the float32 logits.  ``impl="library"`` takes the vendor's products, for comparisons: logits rounded to the tensors'
    type, and the loss with them.
    """
    if impl not in ("native", "library"):
        raise ValueError(f"impl must be native | library, got {impl}")
    x2 = x.reshape(-1, x.shape[-1])
    ids = teacher_ids.reshape(-1, teacher_ids.shape[-1])
    teacher = teacher_logits.reshape(-1, teacher_logits.shape[-1])
    t1 = None if targets is None else targets.reshape(-1)
    nc = weight.shape[0] if n_classes is None else int(n_classes)
    _check(x2.shape[0], nc, weight.shape[0], ids, teacher, t1, temperature, hard_weight, reduction, ("mean", "sum"))
    if _want_target_check(check_targets):
        _check_ids(ids, nc)
        if t1 is not None:
            check_targets_in_range(t1, nc, ignore_index)
    if not (x2.is_cuda and x2.dtype == weight.dtype and x2.dtype in (torch.float32, torch.bfloat16, torch.float16)):
        return topk_distillation(F.linear(x2, weight), ids, teacher, t1, temperature, hard_weight, reduction, ignore_index, nc, check_targets=False)
    cfg = (reduction, ignore_index, nc, float(temperature), float(hard_weight))
    teacher = teacher.detach()
    teacher = teacher if teacher.dtype in (torch.float32, torch.bfloat16, torch.float16) else teacher.float()
    loss, correct, metrics = _ProjectionTopKDistillation.apply(x2.contiguous(), weight.contiguous(), ids.contiguous(), teacher.contiguous(),
                                                               None if t1 is None else t1.contiguous(), cfg, impl,
                                                               torch.is_grad_enabled() and (x2.requires_grad or weight.requires_grad))
    return DistillResult(loss, correct, metrics)


class TopKDistillation(nn.Module):
    """Criterion around ``topk_distillation``; after a call, ``last_correct`` / ``last_metrics`` hold the by-products."""

    def __init__(self, temperature: float = 1.0, hard_weight: float = 0.0, reduction: str = "mean", ignore_index: int = -100,
                 n_classes: Optional[int] = None, check_targets: Optional[bool] = None):
        super().__init__()
        self.temperature, self.hard_weight, self.reduction = temperature, hard_weight, reduction
        self.ignore_index, self.n_classes, self.check_targets = ignore_index, n_classes, check_targets
        self.last_correct: Optional[torch.Tensor] = None
        self.last_metrics: Optional[torch.Tensor] = None

    def forward(self, logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                targets: Optional[torch.Tensor] = None) -> torch.Tensor:
        K = teacher_ids.shape[-1]
        r = topk_distillation(logits.reshape(-1, logits.shape[-1]), teacher_ids.reshape(-1, K), teacher_logits.reshape(-1, K),
                              None if targets is None else targets.reshape(-1), self.temperature, self.hard_weight, self.reduction,
                              self.ignore_index, self.n_classes, self.check_targets)
        self.last_correct, self.last_metrics = r.correct, r.metrics
        return r.loss
