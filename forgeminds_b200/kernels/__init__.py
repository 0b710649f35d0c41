"""Fused kernels with a functional interface.

Each function replaces an eager PyTorch expression, keeps its autograd contract and picks one of
two implementations per call:

* the hand-written sm_100a kernel (CUDA tensors of a supported dtype on a compute-capability-10
  device, backend not forced to ``"fallback"``), or
* the PyTorch statement in :mod:`forgeminds_b200.kernels.reference` (CPU, other dtypes, while
  ``torch.compile`` traces).

``stats()`` reports how often each path ran and why. Public names follow the reference's
``forgemind/kernels/__init__.py:42-48``.

    import forgeminds_b200 as fm
    y = fm.kernels.rms_norm(x, w, 1e-6)
    xn, y = fm.kernels.add_rms_norm(x, delta, w)
    y = fm.kernels.swiglu(gate, up);  y = fm.kernels.swiglu_split(gate_up)
    y = fm.kernels.qk_norm_rope(q, w, cos, sin)
    loss = fm.kernels.kl_distill_loss(hs, ht, w, teacher_head)
    y = fm.kernels.layer_norm(x, w, b);  xn, y = fm.kernels.add_layer_norm(x, delta, w, b)
    cos, sin = fm.kernels.rotary_tables(n, head_dim);  q, k = fm.kernels.rotary_qk(q, k, cos, sin)
    weights, idx, counts, aux = fm.kernels.route_experts(logits, k, score="sigmoid", bias=bias)
    loss = fm.kernels.kl_topk_logits(student_logits, teacher_values, teacher_index)
    fm.kernels.enable(model); fm.kernels.patch(model.norm); fm.kernels.revert(model)
"""
from __future__ import annotations

import math

import torch

from . import reference as _ref
from ._state import (HAS_NATIVE, HAS_TRITON, fast_ok, get_backend, reset_stats, set_backend, stats, tracing,
                     use_custom_ops)

__all__ = [
    "HAS_TRITON", "HAS_NATIVE", "set_backend", "get_backend", "stats", "reset_stats",
    "rms_norm", "add_rms_norm", "qk_norm_rope", "swiglu", "swiglu_split",
    "kl_div_logits", "kl_div", "kl_distill_loss", "distill_kl",
    "newton_schulz", "topk", "softmax",
    "layer_norm", "add_layer_norm", "rotary", "rotary_qk", "rotary_tables", "route_experts",
    "kl_topk_logits", "kl_topk_distill_loss",
    "enable", "patch", "revert", "available", "use_custom_ops",
]

MAX_K = 512


def available() -> bool:
    """True when the CUDA kernels can run on this machine."""
    from .. import ops
    return ops.available()


def _fn():
    from ..ops import functional
    return functional


# ------------------------------------------------------------------------------ norms
def _use_ops() -> bool:
    """Whether the public functions go through the ``torch.library`` forms (``kernels/_ops.py``)."""
    from . import _ops
    return use_custom_ops() or _ops.env_default()


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """``x * rsqrt(mean(x^2) + eps) * w`` over the last dimension."""
    if _use_ops():
        from . import _ops
        return _ops.rms_norm_op(x, w, float(eps))
    return _rms_norm_eager(x, w, eps)


def _rms_norm_eager(x, w, eps=1e-6):
    if x.shape[-1] % 8 == 0 and x.shape[-1] <= 16384 and fast_ok(x, w):
        return _fn().rms_norm(x, w, eps)
    return _ref.rms_norm(x, w, eps)


def add_rms_norm(x: torch.Tensor, delta: torch.Tensor, w: torch.Tensor, eps: float = 1e-6):
    """Residual add and norm in one pass: returns ``(x + delta, rms_norm(x + delta, w))``."""
    if _use_ops() and x.shape == delta.shape:
        from . import _ops
        return _ops.add_rms_norm_op(x, delta, w, float(eps))
    return _add_rms_norm_eager(x, delta, w, eps)


def _add_rms_norm_eager(x, delta, w, eps=1e-6):
    if x.shape == delta.shape and x.shape[-1] % 8 == 0 and x.shape[-1] <= 16384 and fast_ok(x, delta, w):
        return _fn().add_rms_norm(x, delta, w, eps)
    return _ref.add_rms_norm(x, delta, w, eps)


class _QKNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, cos, sin, eps):
        from .. import ops
        y, rstd = ops.require().qk_norm_rope_fwd(x.contiguous(), w.detach().contiguous(), cos, sin, eps)
        ctx.save_for_backward(x, w.detach(), cos, sin, rstd)
        ctx.w_dtype = w.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        from .. import ops
        x, w, cos, sin, rstd = ctx.saved_tensors
        dx, dw = ops.require().qk_norm_rope_bwd(dy.contiguous(), x.contiguous(), w.contiguous(), cos, sin, rstd)
        return dx, dw.to(ctx.w_dtype), None, None, None


def _rope_table(t: torch.Tensor, T: int, half: int):
    """Accepts [T, hd/2] or the broadcastable [1, T, 1, hd/2]; returns contiguous fp32 [T, hd/2]."""
    if t.numel() != T * half:
        return None
    return t.reshape(T, half).to(torch.float32).contiguous()


def qk_norm_rope(x: torch.Tensor, w: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                 eps: float = 1e-6) -> torch.Tensor:
    """Per-head RMSNorm over the head dimension of ``x [B,T,H,D]``, then half-split RoPE."""
    if x.dim() == 4 and x.shape[-1] % 16 == 0 and x.shape[-1] <= 128 and fast_ok(x, w):
        T, half = x.shape[1], x.shape[-1] // 2
        c, s = _rope_table(cos, T, half), _rope_table(sin, T, half)
        if c is not None and s is not None and w.dtype in (x.dtype, torch.float32):
            return _QKNormRope.apply(x, w, c, s, eps)
    return _ref.qk_norm_rope(x, w, cos, sin, eps)


# ------------------------------------------------------------------------------ SwiGLU
def swiglu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """``silu(gate) * up`` for two tensors of the same shape (no broadcasting: a mismatch is almost
    always a wiring mistake and would silently multiply the cost)."""
    if gate.shape != up.shape:
        raise ValueError(f"swiglu needs gate and up of one shape, got {tuple(gate.shape)} and {tuple(up.shape)}")
    if _use_ops() and gate.shape == up.shape and gate.dtype == up.dtype:
        from . import _ops
        return _ops.swiglu_op(gate, up)
    return _swiglu_eager(gate, up)


def _swiglu_eager(gate, up):
    if gate.shape == up.shape and gate.shape[-1] % 8 == 0 and gate.dtype == up.dtype and fast_ok(gate, up):
        return _fn().swiglu(gate, up)
    return _ref.swiglu(gate, up)


def swiglu_split(x: torch.Tensor) -> torch.Tensor:
    """``silu(x[..., :h]) * x[..., h:]`` for the output of a fused gate|up projection."""
    if x.shape[-1] % 2:
        raise ValueError(f"swiglu_split halves the last dimension into gate and up; it is odd here: {tuple(x.shape)}")
    if x.shape[-1] % 16 == 0 and fast_ok(x):
        return _fn().swiglu_split(x)
    return _ref.swiglu_split(x)


# ------------------------------------------------------------------------------ KL
class _KLDiv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, student, teacher, reduction, reuse):
        from .. import ops
        V = student.shape[-1]
        rows = student.numel() // V
        scale = 1.0 / rows if reduction == "mean" else 1.0
        need = student.requires_grad
        row_loss, grad = ops.require().kl_fwd_bwd(student.contiguous(), teacher.contiguous(), scale, need,
                                                  bool(reuse and need))
        ctx.save_for_backward(grad if need else None)
        ctx.shape = student.shape
        ctx.reduction = reduction
        if reduction == "none":
            return row_loss.view(student.shape[:-1])
        total = row_loss.sum()
        return total * scale if reduction == "mean" else total

    @staticmethod
    def backward(ctx, g):
        (grad,) = ctx.saved_tensors
        if grad is None:
            return None, None, None, None
        if ctx.reduction == "none":
            grad = grad.view(ctx.shape) * g.unsqueeze(-1).to(grad.dtype)
        else:
            grad = grad.view(ctx.shape) * g.to(grad.dtype)
        return grad, None, None, None


def kl_div_logits(student: torch.Tensor, teacher: torch.Tensor, reduction: str = "mean",
                  grad_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``KL(softmax(teacher) || softmax(student))`` over the last dim; the teacher is a constant."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction must be mean|sum|none, got {reduction!r}")
    if (student.shape == teacher.shape and student.shape[-1] > 0 and student.dtype == teacher.dtype
            and fast_ok(student, teacher)):
        return _KLDiv.apply(student, teacher.detach(), reduction, False)
    return _ref.kl_div_logits(student, teacher.detach(), reduction)[0]


def kl_distill_loss(hs: torch.Tensor, ht: torch.Tensor, w: torch.Tensor, teacher_head,
                    chunk: int = 4096) -> torch.Tensor:
    """Mean KL of ``softmax(teacher_head(ht)) || softmax(hs @ w.T)``; the teacher runs without grad."""
    if not fast_ok(hs, ht):
        return _ref.kl_distill_loss(hs, ht, w, teacher_head, chunk)
    s2 = hs.reshape(-1, hs.shape[-1])
    t2 = ht.reshape(-1, ht.shape[-1])
    rows = s2.shape[0]
    total = None
    for lo in range(0, rows, chunk):
        hi = min(rows, lo + chunk)
        with torch.no_grad():
            t_logits = teacher_head(t2[lo:hi]).detach()
        s_logits = s2[lo:hi] @ w.t()
        if s_logits.dtype != t_logits.dtype:
            t_logits = t_logits.to(s_logits.dtype)
        part = _KLDiv.apply(s_logits, t_logits, "sum", True)
        total = part if total is None else total + part
    return total / rows


kl_div = kl_div_logits
distill_kl = kl_distill_loss


# ------------------------------------------------------------------------------ Newton-Schulz
def newton_schulz(g: torch.Tensor, steps: int = 5, dtype: torch.dtype | None = None,
                  fused: bool = True) -> torch.Tensor:
    """Quintic Newton-Schulz orthogonalisation of ``g [..., m, n]`` (not differentiable).

    The result has the compute dtype: fp32 for fp32 inputs, bf16 otherwise, or ``dtype``.
    On the GPU the three products of an iteration run on the tcgen05 GEMM with the polynomial
    folded into their epilogues (``alpha * A B^T + beta * C``)."""
    if g.ndim < 2:
        raise ValueError(f"newton_schulz needs ndim >= 2 (a matrix), got shape {tuple(g.shape)}")
    if steps < 1:
        raise ValueError(f"steps must be >= 1, got {steps}")
    if dtype is not None and dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError(f"dtype must be float32/float16/bfloat16, got {dtype}")
    with torch.no_grad():
        work = dtype if dtype is not None else (torch.float32 if g.dtype == torch.float32 else torch.bfloat16)
        if fused and work == torch.bfloat16 and g.numel() > 0 and not tracing() and fast_ok(g):
            from ..ops.newton_schulz import newton_schulz_bf16
            out = newton_schulz_bf16(g, steps)
            if out is not None:
                return out
        return _ref.newton_schulz(g, steps, dtype)


# ------------------------------------------------------------------------------ top-k / softmax
def topk(x: torch.Tensor, k: int, dim: int = -1, sorted: bool = True):
    """``torch.topk`` over the last dim with a fixed tie rule: values descending, NaN largest, equal
    values in ascending index order."""
    if x.dim() < 1:
        raise ValueError(f"topk needs ndim >= 1, got shape {tuple(x.shape)}")
    if dim not in (-1, x.dim() - 1):
        return torch.topk(x, k, dim=dim, sorted=True)
    n = x.shape[-1]
    if k < 1 or k > n:
        raise RuntimeError(f"selected index k out of range (got {k} vs {n})")
    if tracing():
        return torch.topk(x, k, dim=-1, sorted=True)
    if k <= MAX_K and x.numel() < 2 ** 31 and fast_ok(x):
        return _fn().topk_lastdim(x, k)
    if x.is_floating_point() and not x.requires_grad:
        return _ref.topk(x, k)
    return torch.topk(x, k, dim=-1, sorted=True)


def softmax(x: torch.Tensor, dim: int = -1, dtype: torch.dtype | None = None) -> torch.Tensor:
    """``torch.softmax`` over the last dim (other dims use torch)."""
    if x.dim() < 1:
        raise ValueError(f"softmax needs ndim >= 1, got shape {tuple(x.shape)}")
    if dim not in (-1, x.dim() - 1):
        return torch.softmax(x, dim=dim, dtype=dtype)
    if dtype is not None and dtype != x.dtype:
        x = x.to(dtype)
    if not tracing() and x.numel() < 2 ** 31 and fast_ok(x):
        return _fn().softmax_lastdim(x)
    return torch.softmax(x, dim=-1)


# ------------------------------------------------------------------------------ LayerNorm
# The kernels' path of the functions below goes straight to the extension: its C++ side checks the arguments (ValueError, as
# here) and holds the autograd nodes. SMALL: sizes within which every limit of the kernels holds.
SMALL = 2 ** 24


def _rw():
    from ..ops import rowwise
    return rowwise


def _ext():
    from .. import ops
    return ops._mod or ops.require()


def _one_device(name: str, first: torch.Tensor, *others) -> None:
    device = first.device
    for t in others:
        if t is not None and t.device != device:
            raise ValueError(f"{name}: tensors on {device} and {t.device}")


def _check_layer_norm(name: str, x, w, b) -> None:
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name} normalises the last dimension; the input is {tuple(x.shape)}")
    if not x.is_floating_point():
        raise ValueError(f"{name} needs floating-point input, got {x.dtype}")
    for what, t in (("weight", w), ("bias", b)):
        if t is not None and tuple(t.shape) != (x.shape[-1],):
            raise ValueError(f"{name}: {what} {tuple(t.shape)} does not fit rows of {x.shape[-1]}")
    _one_device(name, x, w, b)


_MOST_ROWS = 2 ** 31 - 2 ** 16        # rows that the kernels number in 31 bits


def _ln_fast(x, *rest) -> bool:
    return (x.numel() < SMALL or (x.shape[-1] <= 2 ** 24 and x.numel() // x.shape[-1] < _MOST_ROWS)) and fast_ok(x, *rest)


def layer_norm(x: torch.Tensor, w: torch.Tensor | None = None, b: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * w + b`` over the last dimension (``var`` is the mean square deviation); ``w`` and
    ``b`` are fp32 or of ``x``'s type and may each be left out. Statistics and the gradients of ``w`` and ``b`` are summed
    in fp32, in an order that does not change from run to run."""
    if _ln_fast(x, w, b):
        return _ext().layer_norm(x, w, b, eps)
    _check_layer_norm("layer_norm", x, w, b)
    return _ref.layer_norm(x, w, b, eps)


def add_layer_norm(x: torch.Tensor, delta: torch.Tensor, w: torch.Tensor | None = None, b: torch.Tensor | None = None,
                   eps: float = 1e-5):
    """Residual add and norm in one pass: returns ``(x + delta, layer_norm(x + delta, w, b))``. The norm is that of the sum
    as it is stored in ``x``'s type."""
    if _ln_fast(x, delta, w, b):
        return _ext().add_layer_norm(x, delta, w, b, eps)
    _check_layer_norm("add_layer_norm", x, w, b)
    if x.shape != delta.shape or x.dtype != delta.dtype:
        raise ValueError(f"add_layer_norm needs two tensors of one shape and type, got {tuple(x.shape)} {x.dtype} and "
                         f"{tuple(delta.shape)} {delta.dtype}")
    _one_device("add_layer_norm", x, delta)
    return _ref.add_layer_norm(x, delta, w, b, eps)


# ------------------------------------------------------------------------------ rotary positions
def rotary_tables(n: int, dim: int, theta: float = 10000.0, *, scaling: str | None = None, factor: float = 1.0,
                  trained: int | None = None, fast_turns: float = 32.0, slow_turns: float = 1.0,
                  attention_factor: float | None = None, device=None) -> tuple[torch.Tensor, torch.Tensor]:
    """``cos, sin`` (fp32 ``[n, dim / 2]``) of ``position * theta^(-2i / dim)``, angles taken in 64 bits: in 32 a far
    position is off by whole degrees. ``scaling`` stretches a context by ``factor``:

    * ``"linear"``: every speed divided by ``factor``;
    * ``"ntk"``: ``theta * factor^(dim / (dim - 2))``, which leaves the fastest pair and divides the slowest by ``factor``;
    * ``"yarn"``: pairs that turn more than ``fast_turns`` times within the ``trained`` positions keep their speed, those
      that turn less than ``slow_turns`` times are divided by ``factor``, a ramp over the turns in between; cos and sin are
      multiplied by ``attention_factor`` (default ``0.1 ln(factor) + 1``).
    """
    if n < 1 or dim < 2 or dim % 2:
        raise ValueError(f"rotary_tables needs n >= 1 positions and an even number of rotated values, got {n} and {dim}")
    if not theta > 0 or not factor >= 1:
        raise ValueError(f"theta must be positive and factor at least 1, got {theta} and {factor}")
    if scaling not in (None, "none", "linear", "ntk", "yarn"):
        raise ValueError(f"scaling must be linear|ntk|yarn or None, got {scaling!r}")
    i = torch.arange(0, dim, 2, dtype=torch.float64, device=device)
    gain = 1.0 if attention_factor is None else float(attention_factor)
    if scaling == "ntk":
        theta = theta * factor ** (dim / max(1, dim - 2))
    freq = float(theta) ** (-i / dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        if trained is None or trained < 1 or not fast_turns > slow_turns:
            raise ValueError("yarn needs the number of trained positions and fast_turns > slow_turns")
        keep = ((trained * freq / (2 * math.pi) - slow_turns) / (fast_turns - slow_turns)).clamp(0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
        if attention_factor is None:
            gain = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(n, dtype=torch.float64, device=device).unsqueeze(1) * freq
    return (angle.cos() * gain).to(torch.float32), (angle.sin() * gain).to(torch.float32)


def _rotary_args(name, x, k, cos, sin, positions):
    for t in (x, k):
        if t is not None and (t.dim() != 4 or not t.is_floating_point()):
            raise ValueError(f"{name} needs floating-point [batch, tokens, heads, head_dim], got {tuple(t.shape)} {t.dtype}")
    B, T, _, D = x.shape
    if k is not None and ((k.shape[0], k.shape[1], k.shape[3]) != (B, T, D) or k.dtype != x.dtype):
        raise ValueError(f"{name}: q {tuple(x.shape)} {x.dtype} and k {tuple(k.shape)} {k.dtype} differ in more than their heads")
    _one_device(name, x, k, cos, sin, positions)
    if cos.requires_grad or sin.requires_grad:
        raise ValueError(f"{name}: the tables are constants, but one of them requires a gradient")
    if cos.dim() == 4 and cos.shape[0] == 1 and cos.shape[2] == 1:      # [1, T, 1, R/2], as models keep them to broadcast
        cos, sin = cos[0, :, 0], sin.reshape(sin.shape[1], sin.shape[-1]) if sin.dim() == 4 else sin
    if cos.dim() != 2 or cos.shape != sin.shape:
        raise ValueError(f"{name}: cos and sin must be [positions, rotated / 2], got {tuple(cos.shape)} and {tuple(sin.shape)}")
    if 2 * cos.shape[1] > D:
        raise ValueError(f"{name}: tables for {2 * cos.shape[1]} values of heads of {D}")
    if positions is None:
        if T > cos.shape[0]:
            raise ValueError(f"{name}: tables of {cos.shape[0]} positions for sequences of {T} tokens")
    else:
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{name}: positions must be int32 or int64, got {positions.dtype}")
        if tuple(positions.shape) not in ((T,), (B, T), (1, T)):
            raise ValueError(f"{name}: positions {tuple(positions.shape)} for {B} sequences of {T} tokens")
        if cos.shape[0] < 1:
            raise ValueError(f"{name}: empty tables")
    return cos, sin


def _rotary(name, x, k, cos, sin, positions, interleaved):
    if cos.shape[-1:] != (0,) and _rotary_small(x, k) and fast_ok(x, k):
        if k is None:
            return _ext().rotary_one(x, cos, sin, positions, interleaved)
        return _ext().rotary_qk(x, k, cos, sin, positions, interleaved)
    cos, sin = _rotary_args(name, x, k, cos, sin, positions)
    if k is None:
        return _ref.rotary(x, cos, sin, positions, interleaved)
    return _ref.rotary(x, cos, sin, positions, interleaved), _ref.rotary(k, cos, sin, positions, interleaved)


def _rotary_small(x, k) -> bool:
    if 0 < x.numel() < 2 ** 16:
        return True
    heads = x.shape[2] + (0 if k is None else k.shape[2]) if x.dim() == 4 and (k is None or k.dim() == 4) else 0
    return 0 < heads <= 2 ** 24 and 0 < x.shape[3] <= 2 ** 16 and 0 < x.shape[0] * x.shape[1] < 2 ** 31


def rotary(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor | None = None,
           interleaved: bool = False) -> torch.Tensor:
    """Rotary positions for ``x [batch, tokens, heads, head_dim]`` (any strides; the result is contiguous). See
    :func:`rotary_qk`, which serves queries and keys in one launch."""
    return _rotary("rotary", x, None, cos, sin, positions, interleaved)


def rotary_qk(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor | None = None,
              interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """``(u, v) = (a cos - b sin, a sin + b cos)`` for the pairs ``(i, i + R/2)``, or with ``interleaved`` ``(2i, 2i + 1)``,
    of the first ``R`` values of every head; the values behind them are copied. ``cos, sin [positions, R/2]`` (also
    ``[1, positions, 1, R/2]``, see :func:`rotary_tables`) are constants. Row ``t`` of a sequence takes table row ``t``, or
    ``positions[t]`` / ``positions[b, t]``: a negative one (padding) leaves the heads as they are, one past the table makes
    their rotated values NaN. Queries and keys may be views of one projection's output."""
    return _rotary("rotary_qk", q, k, cos, sin, positions, interleaved)


# ------------------------------------------------------------------------------ distillation from top logits
def _kl_topk_args(name, rows_shape, vocab, values, index, temperature, lse):
    if not 1e-20 <= temperature <= 1e20:
        raise ValueError(f"{name}: temperature must be from 1e-20 to 1e20, got {temperature}")
    if index.dtype not in (torch.int32, torch.int64) or not values.is_floating_point():
        raise ValueError(f"{name}: teacher_values must be floating-point and teacher_index int32 or int64, got {values.dtype} "
                         f"and {index.dtype}")
    shape = index.shape
    if len(shape) < 1 or shape[-1] < 1 or shape != values.shape or shape[:-1] != rows_shape:
        raise ValueError(f"{name}: teacher_values {tuple(values.shape)} and teacher_index {tuple(index.shape)} for rows "
                         f"{tuple(rows_shape)}")
    if vocab < 1:
        raise ValueError(f"{name}: no logits")
    if index.dim() != 2:
        values, index = values.reshape(-1, index.shape[-1]), index.reshape(-1, index.shape[-1])
    if values.requires_grad:
        values = values.detach()
    if lse is not None:
        if lse.shape != rows_shape or not lse.is_floating_point():
            raise ValueError(f"{name}: teacher_lse {tuple(lse.shape)} {lse.dtype} for rows {tuple(rows_shape)}")
        lse = lse.detach().reshape(-1)
    return values, index, lse


def _kl_topk_native(values, index, lse):
    """The teacher's side as the kernels take it: one piece, bf16 or fp32, int64."""
    if values.dtype not in (torch.float32, torch.bfloat16):
        values = values.to(torch.float32)
    if index.dtype != torch.int64:
        index = index.to(torch.int64)
    return values.contiguous(), index.contiguous(), None if lse is None else lse.to(torch.float32).contiguous()


def kl_topk_logits(student: torch.Tensor, teacher_values: torch.Tensor, teacher_index: torch.Tensor, *,
                   temperature: float = 1.0, reduction: str = "mean", teacher_lse: torch.Tensor | None = None) -> torch.Tensor:
    """Distillation from a teacher's ``K`` largest logits: ``sum_k p_k (log p_k - log softmax(student / temperature)[i_k])``
    per row of ``student [.., V]``, with ``teacher_values, teacher_index [.., K]`` (what ``topk`` of its logits gave).

    ``p`` is the softmax of the kept ``teacher_values / temperature``; with ``teacher_lse`` (the logsumexp of ALL teacher
    logits over ``temperature``) it is their share of the whole distribution. The loss is not multiplied by
    ``temperature^2`` (temperatures from 1e-20 to 1e20). The teacher is a constant. A slot whose index lies outside
    ``[0, V)`` (-1 for padding) or whose value is ``-inf`` does not count; a row without slots that count has neither loss
    nor gradient, and ``"mean"`` is over the other rows. An index that stands twice counts twice."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction must be mean|sum|none, got {reduction!r}")
    if _kl_small(student, teacher_index) and fast_ok(student):
        return _ext().kl_topk(student, teacher_values, teacher_index, teacher_lse, temperature, _REDUCTIONS[reduction])
    if student.dim() < 1 or not student.is_floating_point():
        raise ValueError(f"kl_topk_logits: student must be floating-point [.., V], got {tuple(student.shape)} {student.dtype}")
    V = student.shape[-1]
    _one_device("kl_topk_logits", student, teacher_values, teacher_index, teacher_lse)
    values, index, lse = _kl_topk_args("kl_topk_logits", student.shape[:-1], V, teacher_values, teacher_index, temperature, teacher_lse)
    rows = _ref.kl_topk(student.reshape(-1, V), values, index, lse, temperature)
    if reduction == "none":
        return rows.view(student.shape[:-1])
    if reduction == "sum":
        return rows.sum()
    return rows.sum() / _ref.kl_topk_counts(values, index, V).any(dim=-1).sum().clamp(min=1)


def _wide_sum(t: torch.Tensor) -> torch.Tensor:
    return (t if t.dtype == torch.float64 else t.float()).sum()


def _kl_small(student: torch.Tensor, index: torch.Tensor) -> bool:
    return student.dim() > 0 and index.dim() > 0 and index.shape[-1] <= _KL_MAX_KEEP and \
        (student.numel() < SMALL or (student.shape[-1] <= 2 ** 24 and student.numel() // student.shape[-1] < _MOST_ROWS))


_REDUCTIONS = {"mean": 0, "sum": 1, "none": 2}
_KL_MAX_KEEP = 1024          # FMB_KL_MAX_KEEP: more kept logits than this take the PyTorch path


def kl_topk_distill_loss(hs: torch.Tensor, w: torch.Tensor, teacher_values: torch.Tensor, teacher_index: torch.Tensor, *,
                         temperature: float = 1.0, teacher_lse: torch.Tensor | None = None, chunk: int = 4096) -> torch.Tensor:
    """Mean :func:`kl_topk_logits` of the student logits ``hs @ w.T``, which are made ``chunk`` rows at a time. Without
    gradients no more than that exists of them. In training all rows are held until the backward pass: once, as bf16 logits
    that become their gradient in place and are scaled inside the two gradient products, for bf16 ``hs`` on the GPU and a head
    whose two sizes are multiples of 8; otherwise the logits and a gradient of each chunk, which is made again in the
    backward pass because the mean is taken behind it."""
    if hs.dim() < 1 or w.dim() != 2 or hs.shape[-1] != w.shape[1]:
        raise ValueError(f"kl_topk_distill_loss: hidden states {tuple(hs.shape)} and head {tuple(w.shape)}")
    if chunk < 1:
        raise ValueError(f"chunk must be >= 1, got {chunk}")
    V = w.shape[0]
    _one_device("kl_topk_distill_loss", hs, w, teacher_values, teacher_index, teacher_lse)
    values, index, lse = _kl_topk_args("kl_topk_distill_loss", hs.shape[:-1], V, teacher_values, teacher_index, temperature,
                                       teacher_lse)
    s2 = hs.reshape(-1, hs.shape[-1])
    n = s2.shape[0]
    native = V <= 2 ** 24 and index.shape[1] <= _KL_MAX_KEEP and n < _MOST_ROWS and fast_ok(hs)
    if native:
        values, index, lse = _kl_topk_native(values, index, lse)
    counts = _ref.kl_topk_counts(values, index, V).any(dim=-1).sum().clamp(min=1)
    if native and n and hs.dtype == torch.bfloat16 and V % 8 == 0 and hs.shape[-1] % 8 == 0 and w.dtype in (torch.float32, torch.bfloat16):
        return _rw().linear_kl_topk(s2, w, values, index, lse, float(temperature), counts.to(torch.int32).reshape(1), int(chunk))
    total = _wide_sum(s2) if n == 0 else None          # no rows: 0, still a function of hs
    for lo in range(0, n, chunk):
        part = slice(lo, lo + chunk)
        logits = s2[part] @ w.to(s2.dtype).t()
        some = None if lse is None else lse[part]
        rows = _ext().kl_topk(logits, values[part], index[part], some, float(temperature), _REDUCTIONS["sum"]) if native else \
            _ref.kl_topk(logits, values[part], index[part], some, temperature).sum()
        total = rows if total is None else total + rows
    return total / counts


# ------------------------------------------------------------------------------ routing to experts
ROUTE_MAX_EXPERTS, ROUTE_MAX_K, ROUTE_MAX_GROUPS = 512, 32, 32


def check_route(E: int, k: int, score: str, n_groups: int, top_groups: int, group_best: int) -> None:
    """Raises ``ValueError`` for a choice of ``k`` of ``E`` experts that :func:`route_experts` refuses."""
    if score not in ("softmax", "sigmoid"):
        raise ValueError(f"score must be softmax|sigmoid, got {score!r}")
    if n_groups < 1 or E % n_groups or not 1 <= top_groups <= n_groups or group_best not in (1, 2):
        raise ValueError(f"{E} experts in {n_groups} groups of which {top_groups} are kept by their {group_best} best: the "
                         "groups must be equal, 1 <= top_groups <= n_groups, group_best 1 or 2")
    if not 1 <= k <= E // n_groups * top_groups:
        raise ValueError(f"k must be from 1 to the {E // n_groups * top_groups} experts of the kept groups, got {k}")


def route_experts(logits: torch.Tensor, k: int, *, score: str = "softmax", bias: torch.Tensor | None = None, n_groups: int = 1,
                  top_groups: int = 1, group_best: int = 2, renormalise: bool = True, scale: float = 1.0,
                  aux_coef: float = 0.0, z_coef: float = 0.0):
    """Routing of ``logits [tokens, experts]``: ``(weights fp32 [tokens, k], idx int32 [tokens, k], counts int32 [experts],
    aux)``, differentiable in the weights and ``aux``.

    Scores are ``softmax`` or ``sigmoid`` of the logits. Chosen are the ``k`` experts with the largest score plus ``bias``
    (``[experts]``, a constant that balances the load and does not enter the weights), in falling order, equal ones by
    ascending number; the order is that of the exact scores, as far as 64 bits tell them apart. With ``n_groups`` > 1 (equal groups of neighbours) only the
    ``top_groups`` groups with the largest sum of their ``group_best`` (1 or 2) largest biased scores are chosen from.
    Weights are the chosen scores, divided by their sum with ``renormalise``, times ``scale``. ``counts`` are the tokens each
    expert got. ``aux`` is ``aux_coef * E * sum_e load_e * mean(share_e) + z_coef * mean(logsumexp^2)`` with ``share`` the
    scores over their sum and ``load`` the part of all choices that fell on an expert (a constant), or None when both
    coefficients are 0. A token whose logits are all ``-inf`` has scores of 0; weights of chosen scores that are all 0 are 0."""
    if logits.dim() != 2 or not logits.is_floating_point() or logits.shape[1] < 1:
        raise ValueError(f"route_experts needs floating-point [tokens, experts], got {tuple(logits.shape)} {logits.dtype}")
    N, E = logits.shape
    check_route(E, k, score, n_groups, top_groups, group_best)
    args = (n_groups, top_groups, group_best, bool(renormalise), scale, aux_coef, z_coef)
    if E <= ROUTE_MAX_EXPERTS and k <= ROUTE_MAX_K and n_groups <= ROUTE_MAX_GROUPS and N * k < _MOST_ROWS and fast_ok(logits):
        return _ext().route(logits, bias, k, score == "softmax", *args)
    if bias is not None:
        if tuple(bias.shape) != (E,) or not bias.is_floating_point():
            raise ValueError(f"route_experts: bias {tuple(bias.shape)} {bias.dtype} for {E} experts")
        _one_device("route_experts", logits, bias)
        bias = bias.detach()
    return _ref.route_experts(logits, int(k), score == "softmax", bias, *args)


from .apply import enable, patch, revert  # noqa: E402  (needs the functions above)
