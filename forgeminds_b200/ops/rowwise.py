"""Output head and distillation from a teacher's top logits in one Function (GPU only; ``fm.kernels.kl_topk_distill_loss``
checks arguments and picks the PyTorch path elsewhere).

The row operators themselves (``layer_norm``, ``rotary_qk``, ``kl_topk``, ``route``) are differentiable as they come out of
the extension: their autograd nodes are C++ (``csrc/bindings_rows.cpp``), which keeps what their backward kernels read: row
statistics instead of normalised values, the choice and its weights instead of scores.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import require
from .functional import BF16, bf16_of, gemm

F32 = torch.float32


class _LinearKLTopK(torch.autograd.Function):
    """Mean top-logit KL of ``h @ W.T`` without fp32 logits: each chunk of bf16 logits becomes its gradient in place;
    the two gradient products run once in the backward pass, scaled by the incoming gradient on the device. ``need``:
    whether there will be one (``ctx.needs_input_grad`` says so of a Parameter under ``no_grad`` too); all ``n`` rows are
    held until then, and ``chunk`` of them otherwise."""

    @staticmethod
    def forward(ctx, h, weight, values, index, lse, tau, count, chunk, need):
        C = require()
        w = bf16_of(weight)
        h2 = h.reshape(-1, h.shape[-1]).contiguous()
        n, V = h2.shape[0], w.shape[0]
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
                dw = gemm(dlogits, h2, a_mn=True, b_mn=True, out_dtype=F32, alpha_dev=g32, allow_split=True)
                dw = dw if dw.dtype == weight.dtype else dw.to(weight.dtype)
        return dh, dw, None, None, None, None, None, None, None


def linear_kl_topk(h, weight, values, index, lse, tau, count, chunk):
    """``h`` bf16 ``[.., d]``, ``weight [V, d]``; ``count`` (device int32 ``[1]``): the rows that the mean is over."""
    need = torch.is_grad_enabled() and (h.requires_grad or weight.requires_grad)
    return _LinearKLTopK.apply(h, weight, values, index, lse, tau, count, chunk, need)
