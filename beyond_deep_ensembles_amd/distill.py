"""Distilling an ensemble (or any teacher) into one model from the teacher's top logits.

A teacher's answer is kept per row as its ``k`` largest logits, their classes, and ``rest``, the log-sum of what it gives the
other classes (``topk_logits``, ``DeepEnsemble.predict_topk``); the student's loss is the KL divergence between the two
distributions over those ``k`` classes and "any other class" (``distillation_loss``), computed together with its gradient in
one pass over the student's logits.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from .lookup import _backend
from .ops import BdeKernelError, DTYPE_CODES


class TopLogits(NamedTuple):
    values: torch.Tensor        # [..., k], the logits' type, falling
    indices: torch.Tensor       # [..., k], int64
    rest: torch.Tensor          # [...], float32: log sum over the other classes of exp(logit / temperature)


def _logit_rows(logits, name="logits"):
    if logits.dim() < 1 or logits.shape[-1] < 1 or logits.dtype not in DTYPE_CODES:
        raise BdeKernelError(f"{name}: expected a float32 / bfloat16 / float16 [..., V] tensor, got {logits.dtype} {tuple(logits.shape)}")
    rows = logits.reshape(-1, logits.shape[-1])
    if (rows.shape[1] > 1 and rows.stride(1) != 1) or (rows.shape[0] > 1 and rows.stride(0) < rows.shape[1]):
        rows = rows.contiguous()
    return rows


def _dense(t, shape):
    """Contiguous with the strides that go with it (one element or none may carry any)."""
    t = t.reshape(shape).contiguous()
    return t if t.dim() == 0 or t.stride(-1) == 1 else t.clone(memory_format=torch.contiguous_format)


def _temperature(t) -> float:
    t = float(t)
    if not 0.0 < t < float("inf"):
        raise ValueError(f"temperature: a positive number expected, got {t}")
    return t


def topk_logits(logits: torch.Tensor, k: int, *, temperature: float = 1.0, _ops=None) -> TopLogits:
    """The ``k`` largest logits of every row in falling order (the lower class ahead among equals, a NaN above every number)
    with their classes, and the log-sum of the others at ``temperature``.  Log-probabilities are logits.  No gradient."""
    temperature = _temperature(temperature)
    k = int(k)
    _ops, native = _backend(_ops)
    if native is not None:
        return TopLogits(*native.topk_logits(logits, k, temperature))
    rows = _logit_rows(logits.detach())
    n, v = rows.shape
    if not 1 <= k <= min(v, 256) or v > 262144 or n >= 2 ** 31:
        raise BdeKernelError(f"topk_logits: 1 <= k <= min(V, 256), V <= 262144 and fewer than 2^31 rows supported, got k={k}, V={v}, {n} rows")
    shape = logits.shape[:-1]
    values = torch.empty((n, k), dtype=rows.dtype, device=rows.device)
    indices = torch.empty((n, k), dtype=torch.int64, device=rows.device)
    rest = torch.empty(n, dtype=torch.float32, device=rows.device)
    _ops.topk_logits(rows, k, values, indices, rest, temperature=temperature)
    return TopLogits(values.view(shape + (k,)), indices.view(shape + (k,)), rest.view(shape))


def _capturing(t) -> bool:
    return t.is_cuda and torch.cuda.is_current_stream_capturing()


class _Distill(torch.autograd.Function):
    """Under ``sum`` / ``mean`` the forward writes the gradient for d objective / d loss = 1 in the pass that computes the loss;
    the backward returns that buffer after a launch that leaves it alone where the value IS 1 and recomputes it from the logits
    where it is not (one rounding either way).  Later backward passes of a retained graph, and passes that are captured -- a
    graph may be replayed without the one that holds the forward --, compute into a buffer of their own."""

    @staticmethod
    def forward(ctx, logits, values, indices, rest, weight, reduction, scale, temperature, ops):
        z = logits.detach()
        n = z.shape[0]
        loss_rows = torch.empty(n, dtype=torch.float32, device=z.device)
        loss = inv = grad = None
        if reduction != "none":
            loss = torch.empty((), dtype=torch.float32, device=z.device)
            if ctx.needs_input_grad[0] and not _capturing(z):
                grad = torch.empty(z.shape, dtype=z.dtype, device=z.device)
        if reduction == "mean" and weight is not None:
            inv = torch.empty((), dtype=torch.float32, device=z.device)
        ops.distill_fwd(z, values, indices, rest, weight, loss_rows, loss=loss, grad=grad, inv_weight=inv, reduction=reduction, scale=scale,
                        temperature=temperature)
        ctx.save_for_backward(logits, values, indices, rest, weight, inv)
        ctx.meta = (reduction, scale, temperature, ops)
        ctx.unit_grad = grad
        return loss_rows if reduction == "none" else loss

    @staticmethod
    @once_differentiable          # the kernels produce plain tensors: no double backward
    def backward(ctx, g):
        logits, values, indices, rest, weight, inv = ctx.saved_tensors
        reduction, scale, temperature, ops = ctx.meta
        z = logits.detach()
        grad, ctx.unit_grad = ctx.unit_grad, None
        ready = grad is not None and not _capturing(z)
        if not ready:
            grad = torch.empty(z.shape, dtype=z.dtype, device=z.device)
        ops.distill_bwd(z, values, indices, rest, weight, _dense(g, g.shape), grad, inv_weight=inv, mean=reduction == "mean", skip_if_one=ready,
                        scale=scale, temperature=temperature)
        return (grad,) + (None,) * 8


def distillation_loss(logits: torch.Tensor, values: torch.Tensor, indices: torch.Tensor, rest: Optional[torch.Tensor] = None, *,
                      temperature: float = 1.0, weight: Optional[torch.Tensor] = None, scale: float = 1.0, reduction: str = "mean",
                      _ops=None) -> torch.Tensor:
    """KL divergence from a teacher's top logits to the student's ``logits`` [..., V], float32.

    ``values`` / ``indices`` [..., K] and ``rest`` [...] are what ``topk_logits`` gives at the same ``temperature``: the teacher's
    distribution over its K classes and all others together.  Without ``rest`` the list is all there is.  Entries whose index
    is outside [0, V) are not used (pad short lists with -1); entries of one class add up.  ``weight`` [...]: a factor per row --
    a row of weight 0 (padding) contributes nothing whatever it holds, as does one about which the teacher says nothing.
    ``reduction``: "none" (a loss per row), "sum", "mean" (over the sum of the weights; 0 if that is 0).  ``scale`` multiplies
    the loss: fold constant factors (alpha * temperature ** 2, a loss scale) in here, so that the gradient leaves the forward
    pass finished.  The gradient goes to ``logits`` alone, in their type."""
    if reduction not in ("none", "sum", "mean"):
        raise ValueError(f"reduction: 'none', 'sum' or 'mean', not {reduction!r}")
    temperature = _temperature(temperature)
    _ops, native = _backend(_ops)
    if native is not None:
        return native.distillation_loss(logits, values, indices, rest, weight, _ops.REDUCTION[reduction], scale, temperature)
    rows = _logit_rows(logits)
    n, v = rows.shape
    lead = tuple(logits.shape[:-1])
    if values.dim() < 1 or tuple(values.shape[:-1]) != lead or indices.shape != values.shape:
        raise BdeKernelError(f"distillation_loss: values and indices of shape {lead + ('K',)} expected, got {tuple(values.shape)} and "
                             f"{tuple(indices.shape)}")
    k = values.shape[-1]
    if not 1 <= k <= 1024 or not 1 <= v <= 262144 or n >= 2 ** 31:
        raise BdeKernelError(f"distillation_loss: 1 <= K <= 1024, 1 <= V <= 262144 and fewer than 2^31 rows supported, got K={k}, V={v}, "
                             f"{n} rows")
    for name, t in (("rest", rest), ("weight", weight)):
        if t is not None and tuple(t.shape) != lead:
            raise BdeKernelError(f"{name}: expected shape {lead}, got {tuple(t.shape)}")
    for name, t in (("values", values), ("rest", rest), ("weight", weight)):
        if t is not None and t.requires_grad:
            raise BdeKernelError(f"{name}: the teacher's side and the weights are constants of this loss (no gradient); detach them")
    flat = [_dense(values, (n, k)), _dense(indices, (n, k))] + [None if t is None else _dense(t, (n,)) for t in (rest, weight)]
    loss = _Distill.apply(rows, *flat, reduction, float(scale), temperature, _ops)
    return loss.view(lead) if reduction == "none" else loss
