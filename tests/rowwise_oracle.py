"""The definitions of LayerNorm, rotary positions, top-logit distillation and expert routing in 64 bits, written from
their formulas, and the bounds that fp32 arithmetic with one rounding at the end has to keep."""
import torch

U32 = 2.0 ** -24


def half_step(dtype) -> float:
    """Largest relative error of one rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


def within(out, exact, slack):
    """``out`` is ``exact`` up to ``slack`` (an absolute error per element of the arithmetic before the last rounding) and one
    rounding to ``out``'s type. Returns the worst excess over the bound (at most 0 when all is well)."""
    assert out.shape == exact.shape, (out.shape, exact.shape)
    o, e = out.double(), exact.double()
    same = (o == e) | (torch.isnan(o) & torch.isnan(e))
    slack = torch.as_tensor(slack, dtype=torch.float64, device=e.device).expand_as(e)
    smallest = torch.finfo(out.dtype).smallest_normal          # below it a rounding is no longer relative
    bound = half_step(out.dtype) * (e.abs() + slack) + slack + smallest
    excess = torch.where(same, torch.full_like(e, -1.0), (o - e).abs() - bound)
    excess = torch.where(torch.isnan(excess), torch.full_like(e, float("inf")), excess)
    return float(excess.max()) if excess.numel() else -1.0


def layer_norm(x, w, b, eps, dy=None, ds=None):
    """``dict(y, dx, dw, db)`` and the bounds of fp32 arithmetic for each, of 2-D ``x``."""
    x = x.double()
    d = x.shape[1]
    w64 = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.double()
    b64 = torch.zeros(d, dtype=torch.float64, device=x.device) if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    r = ((x - mean).square().mean(1, keepdim=True) + eps).rsqrt()
    xh = (x - mean) * r
    out, off = {"y": xh * w64 + b64}, {}
    # mean: a sum of d values in chains of at most 64 and trees, so 80 units of the values' size; the variance likewise,
    # which moves r by half of that; a handful of roundings more for each element
    size = x.abs().amax(1, keepdim=True)
    exh = U32 * (100 * size * r + 100 * xh.abs())
    off["y"] = exh * w64.abs() + 4 * U32 * (xh * w64).abs() + 2 * U32 * b64.abs()
    if dy is not None:
        dy = dy.double()
        g = dy * w64
        m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
        out["dx"] = r * (g - m1 - xh * m2)
        a1, a2 = g.abs().mean(1, keepdim=True), (g * xh).abs().mean(1, keepdim=True)
        eg = 4 * U32 * g.abs() + 100 * U32 * a1 + exh * m2.abs() + xh.abs() * (100 * U32 * a2 + (g.abs() * exh).mean(1, keepdim=True))
        off["dx"] = r * eg + 110 * U32 * (r * (g.abs() + a1 + xh.abs() * a2))
        if ds is not None:
            out["dx"] = out["dx"] + ds.double()
            off["dx"] = off["dx"] + 2 * U32 * (out["dx"].abs() + ds.double().abs())
        rows = x.shape[0]
        out["dw"], out["db"] = (dy * xh).sum(0), dy.sum(0)
        off["dw"] = (rows + 64) * U32 * (dy * xh).abs().sum(0) + (dy.abs() * exh).sum(0)
        off["db"] = (rows + 64) * U32 * dy.abs().sum(0)
    return out, off


def rotary(x, cos, sin, positions, interleaved, sign=1.0):
    """Rotation of ``x [B, T, H, D]`` pair by pair, and its bound."""
    B, T, H, D = x.shape
    L, half = cos.shape
    y = x.double().clone()
    off = torch.zeros_like(y)
    pos = torch.arange(T, device=x.device) if positions is None else positions
    pos = pos.expand(B, T)
    inside = ((pos >= 0) & (pos < L))[:, :, None]
    at = pos.clamp(0, L - 1).long()
    for i in range(half):
        p, q = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = cos.double()[at, i][:, :, None], sign * sin.double()[at, i][:, :, None]
        a, b = x.double()[..., p], x.double()[..., q]
        u, v = a * c - b * s, a * s + b * c
        y[..., p], y[..., q] = torch.where(inside, u, a), torch.where(inside, v, b)
        size = 3 * U32 * ((a * c).abs() + (b * s).abs() + (a * s).abs() + (b * c).abs())
        off[..., p], off[..., q] = torch.where(inside, size, 0.0), torch.where(inside, size, 0.0)
        nan = (pos >= L)[:, :, None].expand(B, T, H)
        y[..., p] = y[..., p].masked_fill(nan, float("nan"))
        y[..., q] = y[..., q].masked_fill(nan, float("nan"))
    return y, off


def kl_topk(student, values, index, tau, lse=None, reduction="mean", upstream=1.0):
    """``(loss, gradient, bound of the loss, bound of the gradient)`` of 2-D inputs; ``upstream`` one number or ``[rows]``."""
    rows, V = student.shape
    x = student.double() / tau
    held = (index >= 0) & (index < V) & (values != float("-inf"))
    at = index.clamp(0, V - 1)
    at = torch.where(held, at, torch.zeros_like(at))
    has = held.any(1)
    t = torch.where(held, values.double() / tau, torch.full_like(values, float("-inf"), dtype=torch.float64))
    base = torch.logsumexp(torch.where(has[:, None], t, torch.zeros_like(t)), 1) if lse is None else lse.double()
    logp = t - base[:, None]
    p = torch.where(held, logp.exp(), torch.zeros_like(t))
    high = x.amax(1, keepdim=True)
    e = (x - high).exp()
    total = e.sum(1, keepdim=True)
    logq = x - high - total.log()
    q = e / total
    lq = logq.gather(1, at)
    row = torch.where(held & (p > 0), p * (logp - lq), torch.zeros_like(p)).sum(1)
    n = max(1, int(has.sum())) if reduction == "mean" else 1
    scale = (torch.as_tensor(upstream, dtype=torch.float64, device=x.device).reshape(-1, 1) / (n * tau)).expand(rows, 1)
    want = torch.zeros_like(x).scatter_add_(1, at, p)
    mass = p.sum(1, keepdim=True)
    grad = torch.where(has[:, None], (q * mass - want) * scale, torch.zeros_like(x))
    # 2^x to 2^-22; its argument z log2(e) / tau is off by a unit of its own size; sums in chains of V / 512 values
    fine = torch.isfinite(x)
    span = torch.where(fine & torch.isfinite(high), (high - x).abs(), torch.zeros_like(x))
    big = torch.where(torch.isfinite(high), high.abs(), torch.zeros_like(high))
    rq = 2.0 ** -21 + U32 * (V / 512 + 64 + 4 * (span + big))
    tt = torch.where(held, (values.double() / tau).abs(), torch.zeros_like(p)).amax(1, keepdim=True)
    if lse is not None:
        tt = torch.maximum(tt, lse.double().abs()[:, None])
    rp = U32 * (16 + index.shape[1] + 4 * tt)
    off_grad = torch.where(has[:, None], scale.abs() * ((rq + rp) * q * mass + rp * want + 4 * U32 * (q * mass + want)),
                           torch.zeros_like(x))
    each = torch.where(held & (p > 0), p * (rp * (1 + (logp - lq).abs()) + U32 * (16 + V / 512 + 8 * (tt + big + lq.abs()))
                                            + 2.0 ** -21), torch.zeros_like(p)).sum(1)
    off_row = each + 40 * U32 * torch.where(held & (p > 0), (p * (logp - lq)).abs(), torch.zeros_like(p)).sum(1)
    if reduction == "none":
        return row, grad, off_row, off_grad
    loss = row.sum() / n
    off_loss = (off_row.sum() + (rows / 512 + 40) * U32 * row.abs().sum()) / n
    return loss, grad, off_loss, off_grad


def route(logits, k, score, bias, groups, top_groups, best, renorm, scale, dw=None, aux_coef=0.0, z_coef=0.0, daux=0.0):
    """``dict(weights, idx, counts, aux, grad)``; finite logits."""
    z = logits.double()
    N, E = z.shape
    lse = torch.logsumexp(z, 1, keepdim=True)
    soft = (z - lse).exp()
    s = soft if score == "softmax" else 1 / (1 + (-z).exp())
    c = s if bias is None else s + bias.double()
    order = z.clone() if bias is None else c.clone()
    if groups > 1:
        size = E // groups
        extra = torch.zeros(E, dtype=z.dtype, device=z.device) if bias is None else bias.double()
        rows, scores, extra = c.tolist(), s.tolist(), extra.tolist()
        for t in range(N):
            marks = []
            for g in range(groups):
                top = sorted(range(g * size, (g + 1) * size), key=lambda e: (-rows[t][e], e))[:best]
                # scores and biases apart: the same ones in another order are equal, as they are in exact arithmetic
                marks.append((-(sum(scores[t][e] for e in top) + sum(extra[e] for e in top)), g))
            for _, g in sorted(marks)[top_groups:]:
                order[t, g * size:(g + 1) * size] = -float("inf")
    idx = torch.tensor([sorted(range(E), key=lambda e: (-o[e], e))[:k] for o in order.tolist()], dtype=torch.int64).reshape(N, k)
    idx = idx.to(z.device)
    chosen = s.gather(1, idx)
    total = chosen.sum(1, keepdim=True)
    w = chosen / total if renorm else chosen
    counts = torch.bincount(idx.reshape(-1), minlength=E)
    share, load = s / s.sum(1, keepdim=True), counts.double() / max(1, N * k)
    out = {"weights": w * scale, "idx": idx, "counts": counts,
           "aux": aux_coef * E * (load * share.mean(0)).sum() + z_coef * lse.square().mean()}
    if dw is not None:
        d = dw.double() * scale
        ds = torch.zeros_like(s).scatter_(1, idx, (d - (d * w).sum(1, keepdim=True)) / total if renorm else d)
        dp = daux * aux_coef * E / max(1, N) * load
        ds = ds + (dp - (share * dp).sum(1, keepdim=True)) / s.sum(1, keepdim=True)
        dz = s * (ds - (s * ds).sum(1, keepdim=True)) if score == "softmax" else ds * s * (1 - s)
        out["grad"] = dz + daux * z_coef * 2 / max(1, N) * lse * soft
    return out
