"""Plain-PyTorch statements of every kernel in this package.

They fix the semantics the CUDA kernels must match -- accumulate in fp32 (fp64 inputs stay fp64),
round once when storing, output dtype equals input dtype -- and are the CPU path of the public
functions. Counterpart of the reference's ``forgemind/kernels/_fallback.py:15-109``.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

NS_COEFFS = (3.4445, -4.7750, 2.0315)


def _wide(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype in (torch.float32, torch.float64) else t.float()


def rms_norm(x, w, eps: float = 1e-6):
    xf = _wide(x)
    inv = torch.rsqrt(xf.square().mean(dim=-1, keepdim=True) + eps)
    return (xf * inv * _wide(w)).to(x.dtype)


def add_rms_norm(x, delta, w, eps: float = 1e-6):
    summed = x + delta
    return summed, rms_norm(summed, w, eps)


def rotate_half_split(y, cos, sin):
    a, b = y.chunk(2, dim=-1)
    return torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)


def qk_norm_rope(x, w, cos, sin, eps: float = 1e-6):
    """Per-head RMSNorm over the head dim of ``x [B,T,H,D]`` followed by half-split rotation."""
    xf = _wide(x)
    inv = torch.rsqrt(xf.square().mean(dim=-1, keepdim=True) + eps)
    return rotate_half_split(xf * inv * _wide(w), cos, sin).to(x.dtype)


def swiglu(gate, up):
    return (F.silu(_wide(gate)) * _wide(up)).to(gate.dtype)


def swiglu_split(x):
    h = x.shape[-1] // 2
    return swiglu(x[..., :h], x[..., h:])


def kl_div_logits(student, teacher, reduction: str = "mean"):
    """``KL(softmax(teacher) || softmax(student))`` over the last dim and its gradient with respect
    to the student logits (already scaled for the chosen reduction)."""
    log_s = torch.log_softmax(_wide(student), dim=-1)
    log_t = torch.log_softmax(_wide(teacher), dim=-1)
    p_t = log_t.exp()
    rows = (p_t * (log_t - log_s)).sum(dim=-1)
    if reduction == "none":
        loss, scale = rows, 1.0
    elif reduction == "sum":
        loss, scale = rows.sum(), 1.0
    else:
        scale = 1.0 / max(1, rows.numel())
        loss = rows.sum() * scale
    return loss, ((log_s.exp() - p_t) * scale).to(student.dtype)


def kl_distill_loss(hs, ht, w, teacher_head, chunk: int = 4096):
    """Mean KL of ``softmax(teacher_head(ht)) || softmax(hs @ w.T)``; gradients reach ``hs`` and ``w``
    only. Student logits exist one chunk of rows at a time."""
    s2 = hs.reshape(-1, hs.shape[-1])
    t2 = ht.reshape(-1, ht.shape[-1])
    rows = s2.shape[0]
    total = None
    for lo in range(0, rows, chunk):
        hi = min(rows, lo + chunk)
        with torch.no_grad():
            t_logits = teacher_head(t2[lo:hi]).detach()
        part = kl_div_logits(s2[lo:hi] @ w.t(), t_logits, "sum")[0]
        total = part if total is None else total + part
    return total / rows


def newton_schulz(g, steps: int = 5, dtype=None):
    """Quintic Newton-Schulz orthogonalisation of ``g [..., m, n]`` (Gram matrix on the short side,
    Frobenius pre-scaling; coefficients 3.4445, -4.7750, 2.0315)."""
    a, b, c = NS_COEFFS
    shape = g.shape
    work = torch.float32 if g.dtype == torch.float32 else torch.bfloat16
    if dtype is not None:
        work = dtype
    x = g.reshape(-1, shape[-2], shape[-1])
    flip = shape[-2] > shape[-1]
    if flip:
        x = x.mT
    x = x.to(work)
    x = x / (x.norm(dim=(-2, -1), keepdim=True) + 1e-7)
    for _ in range(steps):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    if flip:
        x = x.mT
    return x.reshape(shape)


def topk(x, k: int):
    """Top-k of the last dim: values descending, NaN largest, equal values by ascending index."""
    xf = x.float() if x.dtype in (torch.float16, torch.bfloat16) else x
    key = torch.where(torch.isnan(xf), torch.full_like(xf, float("inf")), xf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :k]
    return torch.gather(x, -1, order), order


def softmax(x):
    return torch.softmax(x, dim=-1)


# ------------------------------------------------------------------------------ LayerNorm
def layer_norm(x, w=None, b=None, eps: float = 1e-5):
    xf = _wide(x)
    centred = xf - xf.mean(dim=-1, keepdim=True)
    y = centred * torch.rsqrt(centred.square().mean(dim=-1, keepdim=True) + eps)
    if w is not None:
        y = y * _wide(w)
    if b is not None:
        y = y + _wide(b)
    return y.to(x.dtype)


def add_layer_norm(x, delta, w=None, b=None, eps: float = 1e-5):
    summed = x + delta
    return summed, layer_norm(summed, w, b, eps)


# ------------------------------------------------------------------------------ rotary positions
def rotary(x, cos, sin, positions=None, interleaved: bool = False):
    """Rotation of the first ``2 * cos.shape[-1]`` values of each head of ``x [B, T, H, D]`` by the angles of table row
    ``position``: a negative position leaves the head as it is, one past the table gives NaN."""
    T, R = x.shape[1], 2 * cos.shape[-1]
    stay = None
    if positions is None:
        c, s = cos[:T], sin[:T]
    else:
        at = positions.clamp(0, max(cos.shape[0] - 1, 0)).long()
        stay, past = (positions < 0).unsqueeze(-1), (positions >= cos.shape[0]).unsqueeze(-1)
        c = cos[at].masked_fill(stay, 1.0).masked_fill(past, float("nan"))
        s = sin[at].masked_fill(stay, 0.0).masked_fill(past, float("nan"))
    c, s = c.unsqueeze(-2), s.unsqueeze(-2)
    xf = _wide(x)
    a, b = (xf[..., 0:R:2], xf[..., 1:R:2]) if interleaved else (xf[..., : R // 2], xf[..., R // 2: R])
    u, v = a * c - b * s, a * s + b * c
    turned = torch.stack((u, v), dim=-1).flatten(-2) if interleaved else torch.cat((u, v), dim=-1)
    if stay is not None:
        turned = torch.where(stay.unsqueeze(-2), xf[..., :R], turned)      # infinities too
    return torch.cat((turned, xf[..., R:]), dim=-1).to(x.dtype)


# ------------------------------------------------------------------------------ distillation from top logits
def kl_topk_counts(values, index, vocab: int):
    """Which slots count: an index inside the vocabulary and a teacher logit that is not ``-inf``."""
    return (index >= 0) & (index < vocab) & (values != float("-inf"))


def kl_topk(student, values, index, lse=None, temperature: float = 1.0):
    """Per-row ``sum_k p_k (log p_k - log q[index_k])`` (fp32, or fp64 for fp64 logits) of 2-D inputs."""
    held = kl_topk_counts(values, index, student.shape[-1])
    has = held.any(dim=-1, keepdim=True)
    z = _wide(student)
    # differences before they are scaled: a large logit over tau is rounded to more than the exponent can bear, or overflows
    z = ((z - z.detach().amax(dim=-1, keepdim=True)) / temperature).masked_fill(~has, 0.0)
    t = values.to(z.dtype).masked_fill(~held, float("-inf"))
    if lse is None:
        logp = torch.log_softmax(((t - t.amax(dim=-1, keepdim=True)) / temperature).masked_fill(~has, 0.0), dim=-1)
    else:
        logp = t / temperature - lse.to(z.dtype).unsqueeze(-1)
    p = logp.exp().masked_fill(~held, 0.0)
    logq = torch.log_softmax(z, dim=-1).gather(-1, index.masked_fill(~held, 0))
    return torch.where(held & (p != 0), p * (logp - logq), torch.zeros_like(p)).sum(dim=-1)


# ------------------------------------------------------------------------------ routing to experts
def route_experts(logits, k: int, softmax: bool = True, bias=None, groups: int = 1, top_groups: int = 1, best: int = 2,
                  renorm: bool = True, scale: float = 1.0, aux_coef: float = 0.0, z_coef: float = 0.0):
    """``(weights [N, k], idx int32 [N, k], counts int32 [E], aux or None)``. The choice is made in 64 bits: neighbours in
    the order of scores may differ by less than 32 bits hold."""
    N, E = logits.shape
    with torch.no_grad():
        z = logits.double()
        if softmax:
            pick = torch.softmax(z.masked_fill((z == float("-inf")).all(dim=-1, keepdim=True), 0.0), dim=-1)
            pick = pick.masked_fill((z == float("-inf")).all(dim=-1, keepdim=True), 0.0)
        else:
            pick = torch.sigmoid(z)
        score = pick
        pick = pick if bias is None else pick + bias.double()
        order = z if bias is None else pick           # without a bias the logits have the scores' order
        largest = lambda t: torch.nan_to_num(t, nan=float("inf"), posinf=float("inf"), neginf=float("-inf"))  # noqa: E731
        order, pick = largest(order), largest(pick)
        shut = torch.zeros_like(order, dtype=torch.bool)
        if groups > 1:
            each = pick.view(N, groups, -1)
            top = each.sort(dim=-1, descending=True, stable=True).indices[..., :best]
            # scores and biases are added apart: the same ones in another order are equal
            score = score.view_as(each).gather(-1, top).sum(dim=-1)
            if bias is not None:
                score = score + bias.double().view(1, groups, -1).expand_as(each).gather(-1, top).sum(dim=-1)
            score = largest(score)
            out = score.sort(dim=-1, descending=True, stable=True).indices[:, top_groups:]
            shut = torch.zeros_like(score, dtype=torch.bool).scatter_(-1, out, True)
            shut = shut.unsqueeze(-1).expand_as(each).reshape(N, E)
        rank = order.sort(dim=-1, descending=True, stable=True).indices
        open_first = shut.gather(-1, rank).to(torch.uint8).sort(dim=-1, stable=True).indices      # shut ones to the end
        idx = rank.gather(-1, open_first)[:, :k]
        counts = torch.zeros(E, dtype=torch.int32, device=logits.device)
        counts.scatter_add_(0, idx.reshape(-1), torch.ones(N * k, dtype=torch.int32, device=logits.device))
    zf = _wide(logits)
    dead = (zf == float("-inf")).all(dim=-1, keepdim=True)
    zf = zf.masked_fill(dead, 0.0)
    probs = torch.softmax(zf, dim=-1).masked_fill(dead, 0.0)
    if renorm:      # shares of the chosen alone, from the logarithms of their scores: they may vanish in fp32 and still have shares
        at = zf.gather(-1, idx)
        logs = at if softmax else F.logsigmoid(at)
        none = dead | (logs == float("-inf")).all(dim=-1, keepdim=True)
        weights = torch.softmax(logs.masked_fill(none, 0.0), dim=-1).masked_fill(none, 0.0)
    else:
        weights = probs.gather(-1, idx) if softmax else torch.sigmoid(zf).masked_fill(dead, 0.0).gather(-1, idx)
    aux = None
    if aux_coef or z_coef:
        share = probs
        if not softmax:
            scores = torch.sigmoid(zf).masked_fill(dead, 0.0)
            total = scores.sum(dim=-1, keepdim=True)
            share = scores / torch.where(total == 0, torch.ones_like(total), total)
        load = counts.to(zf.dtype) / max(1, N * k)
        lse = torch.logsumexp(zf, dim=-1).masked_fill(dead.squeeze(-1), 0.0)
        n = max(1, N)
        aux = aux_coef * E * (load * (share.sum(dim=0) / n)).sum() + z_coef * lse.square().sum() / n
    return weights * scale, idx.to(torch.int32), counts, aux
