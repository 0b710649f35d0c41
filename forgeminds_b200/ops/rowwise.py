"""Autograd wrappers of the row kernels LayerNorm, rotary positions, distillation from top logits and expert routing
(GPU only; :mod:`forgeminds_b200.kernels` checks arguments and picks the PyTorch path elsewhere).

Calls that need no gradient go straight to the kernels; the Functions keep what their backward kernels read: row
statistics instead of normalised values, the choice and its weights instead of scores.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import require
from .functional import BF16, bf16_of, gemm

F32 = torch.float32


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _rows2(x: torch.Tensor) -> torch.Tensor:
    """``[rows, d]`` with contiguous rows: a view where the strides allow it (rows may be apart), else a copy."""
    x2 = x.reshape(-1, x.shape[-1])
    return x2 if x2.shape[1] <= 1 or x2.stride(1) == 1 else x2.contiguous()


# ------------------------------------------------------------------------------ LayerNorm
def _gain(x, w, b):
    """Detached weight and bias in one type that the kernels take: fp32, or the input's."""
    ws = [t.detach() for t in (w, b) if t is not None]
    if not ws:
        return None, None
    dt = ws[0].dtype
    if any(t.dtype != dt for t in ws) or dt not in (F32, x.dtype):
        dt = F32
    it = iter(t.to(dt).contiguous() for t in ws)
    return next(it) if w is not None else None, next(it) if b is not None else None


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, eps):
        x2 = _rows2(x)
        wd, bd = _gain(x, w, b)
        y, _, stats = require().layernorm_fwd(x2, None, wd, bd, eps, True)
        ctx.save_for_backward(x2, wd, stats)
        ctx.w_fp32 = all(t is None or t.dtype == F32 for t in (wd, bd))
        ctx.types = tuple(None if t is None else t.dtype for t in (w, b))
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x2, wd, stats = ctx.saved_tensors
        dx, dw, db = require().layernorm_bwd(_rows2(dy), x2, wd, stats, None, ctx.needs_input_grad[1],
                                             ctx.needs_input_grad[2], ctx.w_fp32)
        return dx.view(dy.shape), _as(dw, ctx.types[0]), _as(db, ctx.types[1]), None


def _as(t, dtype):
    return t if t is None or t.dtype == dtype else t.to(dtype)


def layer_norm(x, w, b, eps):
    if _wants_grad(x, w, b):
        return _LayerNorm.apply(x, w, b, eps)
    return require().layernorm_fwd(_rows2(x), None, *_gain(x, w, b), eps, False)[0].view(x.shape)


class _AddLayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, w, b, eps):
        ctx.set_materialize_grads(False)
        wd, bd = _gain(x, w, b)
        y, total, stats = require().layernorm_fwd(_rows2(x), _rows2(delta), wd, bd, eps, True)
        ctx.save_for_backward(total, wd, stats)
        ctx.w_fp32 = all(t is None or t.dtype == F32 for t in (wd, bd))
        ctx.types = tuple(None if t is None else t.dtype for t in (w, b))
        ctx.x_shape = x.shape
        return total.view(x.shape), y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, gsum, gy):
        if gy is None:                                  # only the sum was used
            return gsum, gsum, None, None, None
        total, wd, stats = ctx.saved_tensors
        dx, dw, db = require().layernorm_bwd(_rows2(gy), total, wd, stats, None if gsum is None else _rows2(gsum),
                                             ctx.needs_input_grad[2], ctx.needs_input_grad[3], ctx.w_fp32)
        dx = dx.view(ctx.x_shape)
        return dx, dx, _as(dw, ctx.types[0]), _as(db, ctx.types[1]), None


def add_layer_norm(x, delta, w, b, eps):
    """``(x + delta, layer_norm(x + delta))`` from one pass over the row."""
    if _wants_grad(x, delta, w, b):
        return _AddLayerNorm.apply(x, delta, w, b, eps)
    y, total, _ = require().layernorm_fwd(_rows2(x), _rows2(delta), *_gain(x, w, b), eps, False)
    return total.view(x.shape), y.view(x.shape)


# ------------------------------------------------------------------------------ rotary positions
def _heads(x):
    return x if x.shape[3] <= 1 or x.stride(3) == 1 else x.contiguous()


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, interleaved):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(cos, sin, positions)
        ctx.interleaved = interleaved
        qo, ko = require().rotary(_heads(q), None if k is None else _heads(k), cos, sin, positions, interleaved, 1.0)
        return qo if k is None else (qo, ko)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk=None):
        cos, sin, positions = ctx.saved_tensors
        first, second = (gq, gk) if gq is not None else (gk, None)
        if first is None:
            return (None,) * 6
        a, b = require().rotary(_heads(first), None if second is None else _heads(second), cos, sin, positions,
                                ctx.interleaved, -1.0)      # the inverse rotation
        dq, dk = (a, b) if gq is not None else (None, a)
        return dq, dk, None, None, None, None


def rotary(q, k, cos, sin, positions, interleaved):
    if _wants_grad(q, k):
        return _Rotary.apply(q, k, cos, sin, positions, interleaved)
    qo, ko = require().rotary(_heads(q), None if k is None else _heads(k), cos, sin, positions, interleaved, 1.0)
    return qo if k is None else (qo, ko)


# ------------------------------------------------------------------------------ distillation from top logits
class _KLTopK(torch.autograd.Function):
    """The forward pass also leaves the gradient for an upstream gradient of 1, while the row is in the caches; the
    first backward pass hands that tensor out after a kernel has redone the rows whose upstream gradient is another
    number (it is compared on the device). A second one, or one inside a graph capture, computes it anew: a captured
    backward may be replayed with other values."""

    @staticmethod
    def forward(ctx, student, values, index, lse, tau, reduction):
        s2 = _rows2(student)
        ready = ctx.needs_input_grad[0] and not torch.cuda.is_current_stream_capturing()
        loss, rows, stats, grad, ws = require().kl_topk_fwd(s2, values, index, lse, tau, reduction != "none",
                                                           reduction == "mean", None, ready, False)
        ctx.save_for_backward(s2, values, index, lse, stats, ws if reduction == "mean" else None)
        ctx.ready, ctx.tau, ctx.shape = grad, tau, student.shape
        return rows.view(student.shape[:-1]) if reduction == "none" else loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        s2, values, index, lse, stats, count = ctx.saved_tensors
        ready = None if torch.cuda.is_current_stream_capturing() else ctx.ready
        ctx.ready = None
        up = g.to(F32).reshape(-1).contiguous() if g.dim() else g.to(F32)
        grad = require().kl_topk_bwd(s2, values, index, lse, stats, ctx.tau, count, up, ready)
        return grad.view(ctx.shape), None, None, None, None, None


def kl_topk(student, values, index, lse, tau, reduction):
    if _wants_grad(student):
        return _KLTopK.apply(student, values, index, lse, tau, reduction)
    loss, rows, *_ = require().kl_topk_fwd(_rows2(student), values, index, lse, tau, reduction != "none",
                                           reduction == "mean", None, False, False)
    return rows.view(student.shape[:-1]) if reduction == "none" else loss


class _LinearKLTopK(torch.autograd.Function):
    """Mean top-logit KL of ``h @ W.T`` without fp32 logits: each chunk of bf16 logits becomes its gradient in place;
    the two gradient products run once in the backward pass, scaled by the incoming gradient on the device."""

    @staticmethod
    def forward(ctx, h, weight, values, index, lse, tau, count, chunk):
        C = require()
        w = bf16_of(weight)
        h2 = h.reshape(-1, h.shape[-1]).contiguous()
        n, V = h2.shape[0], w.shape[0]
        need = any(ctx.needs_input_grad[:2])
        logits = torch.empty((n if need else min(n, chunk), V), dtype=BF16, device=h.device)
        parts = []
        for lo in range(0, n, chunk):
            hi = min(n, lo + chunk)
            part = logits[lo:hi] if need else logits[: hi - lo]
            gemm(h2[lo:hi], w, out=part)
            parts.append(C.kl_topk_fwd(part, values[lo:hi], index[lo:hi], None if lse is None else lse[lo:hi], tau, True,
                                       True, count, need, True)[0])
        ctx.save_for_backward(h2, w, logits if need else None)
        ctx.weight, ctx.h_shape = weight, h.shape
        return torch.stack(parts).sum()

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        h2, w, dlogits = ctx.saved_tensors
        weight = ctx.weight
        g32 = g.to(F32).reshape(1).contiguous()
        dh = dw = None
        if ctx.needs_input_grad[0]:
            dh = gemm(dlogits, w, b_mn=True, alpha_dev=g32).view(ctx.h_shape)
        if ctx.needs_input_grad[1]:
            main = getattr(weight, "_fm_main_grad", None)
            if main is not None:
                gemm(dlogits, h2, a_mn=True, b_mn=True, out=main, c=main, beta=1.0, alpha_dev=g32, allow_split=True)
            else:
                dw = _as(gemm(dlogits, h2, a_mn=True, b_mn=True, out_dtype=F32, alpha_dev=g32, allow_split=True), weight.dtype)
        return dh, dw, None, None, None, None, None, None


def linear_kl_topk(h, weight, values, index, lse, tau, count, chunk):
    """``h`` bf16 ``[.., d]``, ``weight [V, d]``; ``count`` (device int32 ``[1]``): the rows that the mean is over."""
    return _LinearKLTopK.apply(h, weight, values, index, lse, tau, count, chunk)


# ------------------------------------------------------------------------------ routing to experts
class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, k, cfg, need_aux, aux_coef, z_coef):
        softmax, groups, top_groups, best, renorm, scale = cfg
        ctx.set_materialize_grads(False)
        w, idx, counts, aux = require().route_fwd(logits, bias, k, softmax, groups, top_groups, best, renorm, scale, need_aux,
                                                  aux_coef, z_coef)
        ctx.save_for_backward(logits, w, idx, counts)
        ctx.how = (softmax, renorm, scale, aux_coef, z_coef)
        ctx.mark_non_differentiable(idx, counts)
        return w, idx, counts, aux

    @staticmethod
    @once_differentiable
    def backward(ctx, dw, _didx, _dcounts, daux):
        if dw is None and daux is None:
            return (None,) * 7
        logits, w, idx, counts = ctx.saved_tensors
        dw = None if dw is None else dw.to(F32).contiguous()
        daux = None if daux is None else daux.to(F32).reshape(1)
        return require().route_bwd(logits, w, idx, counts, dw, daux, *ctx.how), None, None, None, None, None, None


def route(logits, bias, k, softmax, groups, top_groups, best, renorm, scale, aux_coef, z_coef):
    """``logits [N, E]`` -> ``(weights fp32 [N, k], idx int32 [N, k], counts int32 [E], aux fp32 or None)``."""
    cfg = (softmax, groups, top_groups, best, renorm, scale)
    need_aux = aux_coef != 0.0 or z_coef != 0.0
    rows = _rows2(logits)
    if _wants_grad(logits):
        return _Route.apply(rows, bias, k, cfg, need_aux, aux_coef, z_coef)
    return tuple(require().route_fwd(rows, bias, k, *cfg, need_aux, aux_coef, z_coef))
