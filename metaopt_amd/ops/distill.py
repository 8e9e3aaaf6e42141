"""Distillation from a teacher's top logits for the population LM: the loss beside
:func:`.lm.cross_entropy` for trials that learn from a teacher as well as from labels -- a HIP
kernel (csrc/lm_distill.hip) behind an autograd Function, with a PyTorch reference of the same math
(the CPU backend)."""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .heads import _call, _no_tangents, _once, _p, _same
from .lm import _hip, _ScaledGrad

c_void_p, c_int, c_float, c_int64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_int64

_lib.register_signatures({
    "mopt_distill": ([c_void_p, c_int64] + [c_void_p] * 9 + [c_int] * 6 + [c_float] * 3 + [c_void_p],
                     c_int),
})

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
#: most teacher entries of a row
MAX_TOP = 1024


def distill_ref(logits, labels, top_values, top_index, rows_per_trial, temperature=1.0, alpha=0.5):
    """Per-trial sums of :func:`distill_loss`'s rows in (at least) fp32."""
    f = torch.promote_types(logits.dtype, torch.float32)
    x = logits.to(f)
    R, V = x.shape

    def rows(t):
        return (t.to(f).repeat_interleave(rows_per_trial) if torch.is_tensor(t) else
                torch.full((R,), float(t), dtype=f, device=x.device))[:, None]
    tau, a = rows(temperature), rows(alpha)
    y, index = labels.long()[:, None], top_index.long()
    hard, soft = (y >= 0) & (y < V), (index >= 0) & (index < V)
    t = torch.where(soft, top_values.to(f) / tau, torch.full((), -float("inf"), dtype=f, device=x.device))
    some = (t > -float("inf")).any(1, keepdim=True)
    q = torch.where(some, t, torch.zeros_like(t)).softmax(1) * soft * some
    ce = -x.log_softmax(1).gather(1, torch.where(hard, y, torch.zeros_like(y)))
    lp = (x / tau).log_softmax(1).gather(1, torch.where(soft, index, torch.zeros_like(index)))
    zero = torch.zeros((), dtype=f, device=x.device)
    kl = torch.where(q > 0, q * (torch.where(q > 0, q, torch.ones_like(q)).log() - lp), zero)
    loss = (torch.where(hard & (a != 1), (1 - a) * ce, zero).squeeze(1)
            + torch.where(some & (a != 0), a * tau * tau * kl.sum(1, keepdim=True), zero).squeeze(1))
    return loss.view(-1, rows_per_trial).sum(1)


def _launch(logits, labels, top, index, tau, alpha, rows_per_trial, scale, weight, grad, want_loss):
    R, V = logits.shape
    P = R // rows_per_trial
    loss = rows = None
    if want_loss:
        rows = torch.empty(R, dtype=torch.float32, device=logits.device)
        loss = torch.empty(P, dtype=torch.float32, device=logits.device)
    tensor = torch.is_tensor
    _call(logits, "mopt_distill", _p(logits), logits.stride(0), _p(labels), _p(top), _p(index),
          _p(tau) if tensor(tau) else None, _p(alpha) if tensor(alpha) else None, _p(weight), _p(rows),
          _p(loss), _p(grad), R, rows_per_trial, V, top.shape[1], _TYPES[top.dtype],
          _TYPES[logits.dtype], 1.0 if tensor(tau) else tau, 0.0 if tensor(alpha) else alpha, scale)
    return loss


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, top, index, tau, alpha, rows_per_trial, scale, unit, inplace):
        ctx.unit = unit
        if unit:       # one pass over the logits: the loss and its gradient
            grad = logits if inplace else torch.empty(logits.shape, dtype=logits.dtype,
                                                      device=logits.device)
            loss = _launch(logits, labels, top, index, tau, alpha, rows_per_trial, scale, None, grad,
                           True)
            if inplace:                # (who else kept the logits for a backward has to know)
                torch.autograd.graph.increment_version(logits)
            ctx.save_for_backward(grad)
            return loss
        mixed = [t for t in (tau, alpha) if torch.is_tensor(t)]
        ctx.save_for_backward(logits, labels, top, index, *mixed)
        ctx.meta = (tau if not torch.is_tensor(tau) else None,
                    alpha if not torch.is_tensor(alpha) else None, rows_per_trial, scale)
        return _launch(logits, labels, top, index, tau, alpha, rows_per_trial, scale, None, None, True)

    @_once
    def backward(ctx, dloss):
        if ctx.unit:
            (grad,) = ctx.saved_tensors
        else:
            logits, labels, top, index, *mixed = ctx.saved_tensors
            tau, alpha, rows_per_trial, scale = ctx.meta
            tau = mixed.pop(0) if tau is None else tau
            alpha = mixed.pop(0) if alpha is None else alpha
            grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
            _launch(logits, labels, top, index, tau, alpha, rows_per_trial, scale,
                    dloss.float().contiguous(), grad, False)
        return (grad,) + (None,) * 9


def _mix(name, v, P, like, low, high):
    if torch.is_tensor(v):
        if v.dtype != torch.float32 or tuple(v.shape) != (P,) or not v.is_contiguous():
            raise ValueError(f"{name} must be a number or a contiguous float32 tensor of {P} values, "
                             "one a trial")
        if v.requires_grad:
            raise ValueError(f"{name} has no gradient here: detach it")
        _same(like, name, v)
        return v
    v = float(v)
    if not low <= v <= high:
        raise ValueError(f"{name} {v} is outside [{low}, {high}]")
    return v


def distill_loss(logits, labels, top_values, top_index, rows_per_trial, temperature=1.0, alpha=0.5,
                 grad_scale=1.0, unit_weights=False, inplace=False):
    """Per-trial SUM ``[P]`` (fp32) over the rows of ``logits`` ``[R, V]`` of

    ``(1 - alpha) CE(labels) + alpha temperature^2 KL(teacher || student)``,

    the teacher being the softmax of its top logits ``top_values`` ``[R, K]`` / ``temperature`` at
    the vocabulary indices ``top_index`` (int32 ``[R, K]``) and nothing elsewhere, the student the
    softmax of ``logits / temperature`` over the whole vocabulary.

    Entries with an index outside ``[0, V)`` are absent (rows with fewer than K); equal indices of a
    row add up; a row without any has no teacher term, a label outside ``[0, V)`` (int32 ``[R]``) no
    cross-entropy.  ``temperature`` (> 0) and ``alpha`` (in [0, 1]) are numbers or fp32 ``[P]``
    tensors, one value a trial.  logits: bf16, fp16 or fp32; top_values any of these.

    ``grad_scale`` multiplies the gradient (``1 / rows_per_trial``: mean-loss gradients).
    ``unit_weights=True`` promises that the result is differentiated through ``loss.sum()`` only:
    the gradient comes out of the forward pass (one read of the logits, one write) and takes the
    logits' place with ``inplace=True`` (a write in place to autograd: an operation that kept the
    logits for its own backward refuses it).  Without it the backward reads the logits again."""
    if logits.dim() != 2 or not logits.is_floating_point():
        raise ValueError("logits are [rows, vocabulary]")
    R, V = logits.shape
    if V < 1 or rows_per_trial < 1 or R % rows_per_trial:
        raise ValueError(f"{R} rows of {V} logits are not whole trials of {rows_per_trial} rows")
    if labels.dtype != torch.int32 or tuple(labels.shape) != (R,):
        raise ValueError(f"labels must be int32 [{R}]")
    if top_index.dim() != 2 or top_index.shape[0] != R or top_index.dtype != torch.int32:
        raise ValueError(f"top_index must be int32 [{R}, K]")
    if top_values.shape != top_index.shape or not top_values.is_floating_point():
        raise ValueError("top_values and top_index are of one shape")
    if top_index.shape[1] > MAX_TOP:
        raise ValueError(f"{top_index.shape[1]} teacher entries a row: at most {MAX_TOP}")
    if top_values.requires_grad:
        raise ValueError("the teacher has no gradient here: detach top_values")
    if inplace and not unit_weights:
        raise ValueError("inplace needs unit_weights: the backward reads the logits again")
    _same(logits, "labels top_values top_index", labels, top_values, top_index)
    P = R // rows_per_trial
    tau = _mix("temperature", temperature, P, logits, 1e-6, 1e6)
    alpha = _mix("alpha", alpha, P, logits, 0.0, 1.0)
    if not _hip(logits, "distill"):
        loss = distill_ref(logits, labels, top_values, top_index, rows_per_trial, tau, alpha)
        return loss if grad_scale == 1.0 else _ScaledGrad.apply(loss, grad_scale)
    for name, t in (("logits", logits), ("top_values", top_values)):
        if t.dtype not in _TYPES:
            raise ValueError(f"distill_loss on a GPU takes bfloat16, float16 or float32 {name}, not "
                             f"{t.dtype}")
    _no_tangents("distill_loss", logits, top_values, *(t for t in (tau, alpha) if torch.is_tensor(t)))
    if R == 0:
        return logits.new_zeros(P, dtype=torch.float32) + 0.0 * logits.sum()
    need = torch.is_grad_enabled() and logits.requires_grad
    if inplace and need and (logits.is_leaf or not logits.is_contiguous()):
        raise ValueError("inplace overwrites the logits: not those of a leaf or a strided view")
    # rows are read at any element's alignment; only their elements have to lie together
    logits = logits if logits.stride(1) == 1 or V == 1 else logits.contiguous()
    labels, top_values, top_index = (t.contiguous() for t in (labels, top_values, top_index))
    if need:
        return _Distill.apply(logits, labels, top_values, top_index, tau, alpha, int(rows_per_trial),
                              float(grad_scale), bool(unit_weights), bool(inplace))
    return _launch(logits, labels, top_values, top_index, tau, alpha, int(rows_per_trial),
                   float(grad_scale), None, None, True)
