"""What is measured of the operators that a student model's training step is made of: LayerNorm, rotary positions,
routing to experts and distillation from a teacher's stored top logits.

``run`` computes them in their plain form (elementary torch operations in 32 bits, routing scores in 64 because
neighbours in an order of scores may differ by less than 32 bits hold), or, with ``own``, through ``fm.kernels``.
"""
import math

import numpy as np
import torch

own = False

F32, F64 = torch.float32, torch.float64
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp32": 4}
LN_EPS = 1e-5


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token for each of a handful of sequences goes through a norm: latency
        dict(name="layer_norm_tokens", op="layer_norm", rows=8, dim=1024, dtype="bf16", wdtype="bf16", add=False,
             train=False, affine=True, pitch=0),
        # the norm of a 1024-wide block over a micro-batch of 4 x 2048 tokens, forward and backward
        dict(name="layer_norm_train", op="layer_norm", rows=8192, dim=1024, dtype="bf16", wdtype="fp32", add=False,
             train=True, affine=True, pitch=0),
        # residual add and norm of a 4096-wide block over 8 x 2048 tokens, forward and backward: the largest
        dict(name="add_layer_norm_train", op="layer_norm", rows=16384, dim=4096, dtype="bf16", wdtype="fp32", add=True,
             train=True, affine=True, pitch=0),
        # one new token for each of 64 sequences at positions far out on a scaled table, 32 / 8 heads of 128: latency
        dict(name="rotary_tokens", op="rotary", batch=64, seq=1, hq=32, hk=8, dim=128, rot=128, interleaved=False,
             dtype="bf16", train=False, positions="far", table=131072, scaling="yarn", packed=True),
        # q and k of a block as views of one q|k|v product, 4 x 2048 tokens, 16 / 4 heads of 64, with gradients
        dict(name="rotary_train", op="rotary", batch=4, seq=2048, hq=16, hk=4, dim=64, rot=64, interleaved=False,
             dtype="bf16", train=True, positions="rows", table=2048, scaling="none", packed=True),
        # a long prompt with documents packed into it, neighbouring pairs, half of each head rotated: the largest
        dict(name="rotary_long", op="rotary", batch=1, seq=65536, hq=32, hk=8, dim=128, rot=64, interleaved=True,
             dtype="bf16", train=False, positions="documents", table=65536, scaling="linear", packed=False),
        # a small fp32 batch of 64 tokens against 16 kept logits, loss and gradient
        dict(name="kl_topk_small", op="kl_topk", rows=64, vocab=32000, keep=16, dtype="fp32", tdtype="fp32", tau=1.0,
             norm="kept", train=True, holes=0.0),
        # a micro-batch of 4 x 2048 tokens over a 32000-word vocabulary, 64 kept logits, loss and gradient
        dict(name="kl_topk_train", op="kl_topk", rows=8192, vocab=32000, keep=64, dtype="bf16", tdtype="bf16", tau=2.0,
             norm="kept", train=True, holes=0.05),
        # a wide vocabulary of odd size, the teacher's normaliser stored beside its logits: the largest
        dict(name="kl_topk_wide", op="kl_topk", rows=4096, vocab=128259, keep=128, dtype="bf16", tdtype="fp32", tau=1.0,
             norm="full", train=True, holes=0.02),
        # the tokens of one decoding step, 64 experts, 6 of them: latency
        dict(name="route_tokens", op="route", tokens=32, experts=64, k=6, score="softmax", bias=False, groups=1, top_groups=1,
             best=1, renorm=True, dtype="bf16", train=False, aux=False),
        # a micro-batch of 4 x 2048 tokens over 8 experts, 2 of them, balance and z terms, gradients
        dict(name="route_train", op="route", tokens=8192, experts=8, k=2, score="softmax", bias=False, groups=1, top_groups=1,
             best=1, renorm=True, dtype="bf16", train=True, aux=True),
        # 32 x 2048 tokens over 256 experts in 8 groups, sigmoid scores with a balance bias, gradients: the largest
        dict(name="route_groups_train", op="route", tokens=65536, experts=256, k=8, score="sigmoid", bias=True, groups=8,
             top_groups=4, best=2, renorm=True, dtype="fp32", train=True, aux=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("layer_norm", "rotary", "kl_topk", "route"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    if op == "layer_norm":
        dim = _log(rng, 64, 16384)
        if rng.random() < 0.6:                      # most widths are whole vectors, some are not
            dim = max(64, dim // 8 * 8)
        most = 16384 * 4096 // (2 if dtype == "fp32" else 1)
        rows = _log(rng, 1, min(65536, most // dim))
        return dict(op=op, rows=rows, dim=dim, dtype=dtype, wdtype=rng.choice((dtype, "fp32")), add=rng.random() < 0.4,
                    train=rng.random() < 0.7, affine=rng.random() < 0.85, pitch=rng.choice((0, 0, 0, 8, 24)))
    if op == "rotary":
        dim = rng.choice((32, 64, 64, 80, 96, 128, 128, 192, 256))
        rot = dim if rng.random() < 0.6 else max(2, rng.randrange(1, dim // 2 + 1) * 2)
        hk = rng.choice((1, 2, 4, 8))
        hq = hk * rng.choice((1, 2, 4, 7, 8))
        batch = _log(rng, 1, 64)
        most = 65536 * 40 * 128 // (2 if dtype == "fp32" else 1) // 2
        seq = _log(rng, 1, max(1, min(65536, most // (batch * (hq + hk) * dim))))
        return dict(op=op, batch=batch, seq=seq, hq=hq, hk=hk, dim=dim, rot=rot, interleaved=rng.random() < 0.5, dtype=dtype,
                    train=rng.random() < 0.5, positions=rng.choice(("rows", "far", "documents")),
                    table=max(seq, _log(rng, 1024, 262144)), scaling=rng.choice(("none", "linear", "ntk", "yarn")),
                    packed=rng.random() < 0.6)
    if op == "kl_topk":
        vocab = _log(rng, 1000, 160000)
        if rng.random() < 0.6:
            vocab = vocab // 8 * 8
        keep = _log(rng, 1, 256)
        most = 4096 * 128259 // (2 if dtype == "fp32" else 1)
        return dict(op=op, rows=_log(rng, 1, min(16384, most // vocab)), vocab=vocab, keep=keep, dtype=dtype,
                    tdtype=rng.choice(("bf16", "fp32")), tau=rng.choice((1.0, 1.0, 2.0, 4.0)), norm=rng.choice(("kept", "kept", "full")),
                    train=rng.random() < 0.8, holes=rng.choice((0.0, 0.03, 0.3)))
    groups = rng.choice((1, 1, 2, 4, 8))
    experts = groups * _log(rng, 4 if groups > 1 else 8, 512 // groups if groups > 1 else 384)
    top_groups = groups if groups == 1 else rng.randrange(1, groups + 1)
    k = rng.randrange(1, min(16, experts // groups * top_groups) + 1)
    return dict(op=op, tokens=_log(rng, 1, min(65536, 65536 * 256 // experts)), experts=experts, k=k,
                score=rng.choice(("softmax", "sigmoid")), bias=rng.random() < 0.5, groups=groups, top_groups=top_groups,
                best=rng.choice((1, 2)), renorm=rng.random() < 0.7, dtype=dtype, train=rng.random() < 0.6, aux=rng.random() < 0.5)


def work(case):
    c = case
    if c["op"] == "layer_norm":
        n, es = c["rows"] * c["dim"], SIZE[c["dtype"]]
        w = 2 * c["dim"] * SIZE[c["wdtype"]] if c["affine"] else 0
        tensors = (4 if c["add"] else 2)                               # forward: x (, delta) in, y (, sum) out
        byte, flops = tensors * n * es + w, n * (10 if c["affine"] else 8)
        if c["train"]:                                                 # dy (, d sum) in, dx out; gradients of w and b out
            byte += ((3 if c["add"] else 2) * n) * es + w              # the row itself is counted once, with the forward
            flops += n * (14 if c["affine"] else 9)
        return {"bytes": byte, "flops": flops}
    if c["op"] == "rotary":
        tok = c["batch"] * c["seq"]
        n = tok * (c["hq"] + c["hk"]) * c["dim"]
        lines = c["seq"] if c["positions"] == "rows" else min(tok, c["table"])
        byte = 2 * n * SIZE[c["dtype"]] + lines * c["rot"] * 4 + (0 if c["positions"] == "rows" else 8 * tok)
        flops = tok * (c["hq"] + c["hk"]) * c["rot"] * 3
        return {"bytes": byte * (2 if c["train"] else 1), "flops": flops * (2 if c["train"] else 1)}
    if c["op"] == "kl_topk":
        n, es = c["rows"] * c["vocab"], SIZE[c["dtype"]]
        byte = n * es * (2 if c["train"] else 1) + c["rows"] * c["keep"] * (SIZE[c["tdtype"]] + 8) + 4 * c["rows"]
        return {"bytes": byte, "flops": n * (7 if c["train"] else 4)}
    n, es = c["tokens"] * c["experts"], SIZE[c["dtype"]]
    byte = n * es + c["tokens"] * c["k"] * 8 + c["experts"] * 8
    flops = n * (8 + c["k"])
    if c["train"]:
        byte += n * es + c["tokens"] * c["k"] * 4
        flops += n * 8
    return {"bytes": byte, "flops": flops}


# ------------------------------------------------------------------------------------------ inputs
def _inv_freq(rot, theta, scaling, factor, trained):
    """Rotation speeds in 64 bits and the factor on cos and sin, for a context stretched by ``factor``."""
    i = torch.arange(0, rot, 2, dtype=F64)
    if scaling == "ntk":
        theta = theta * factor ** (rot / max(1, rot - 2))
    freq = theta ** (-i / rot)
    if scaling == "linear":
        return freq / factor, 1.0
    if scaling == "yarn":
        turns = trained * freq / (2 * math.pi)            # whole turns within the trained context: over 32 kept, under 1 stretched
        mix = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return freq * mix + freq / factor * (1 - mix), 0.1 * math.log(factor) + 1.0
    return freq, 1.0


def _tables(case, device):
    factor = 1.0 if case["scaling"] == "none" else max(2.0, case["table"] / 8192)
    freq, gain = _inv_freq(case["rot"], 10000.0, case["scaling"], factor, 8192)
    angle = torch.arange(case["table"], dtype=F64, device=device)[:, None] * freq.to(device)
    return (angle.cos() * gain).to(F32), (angle.sin() * gain).to(F32)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    c, dt = case, DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    s = {"case": dict(c)}
    if c["op"] == "layer_norm":
        rows, dim = c["rows"], c["dim"]
        lift = 1.0 + 4.0 * (torch.rand(dim, device=dev, generator=g) < 0.01)        # a few strong channels, as trained models have

        def stream(scale, offset=0.0):
            wide = torch.empty(rows, dim + c["pitch"], device=dev, dtype=dt)
            wide[:, :dim] = normal(rows, dim) * scale * lift + offset
            return wide[:, :dim]

        s["x"] = stream(1.0, 0.3).requires_grad_(c["train"])
        if c["add"]:
            s["delta"] = stream(0.5).requires_grad_(c["train"])
            s["ds"] = stream(0.02) if c["train"] else None
        if c["train"]:
            s["dy"] = stream(0.02)
        s["w"] = s["b"] = None
        if c["affine"]:
            wdt = DTYPES[c["wdtype"]]
            s["w"] = (1.0 + 0.2 * normal(dim)).to(wdt).requires_grad_(c["train"])
            s["b"] = (0.1 * normal(dim)).to(wdt).requires_grad_(c["train"])
    elif c["op"] == "rotary":
        B, T, hq, hk, D = c["batch"], c["seq"], c["hq"], c["hk"], c["dim"]
        if c["packed"]:                                                             # views of one q|k|v product
            qkv = normal(B, T, (hq + 2 * hk) * D).to(dt)
            q = qkv[..., : hq * D].unflatten(-1, (hq, D))
            k = qkv[..., hq * D: (hq + hk) * D].unflatten(-1, (hk, D))
        else:
            q, k = normal(B, T, hq, D).to(dt), normal(B, T, hk, D).to(dt)
        s["q"], s["k"] = q.detach().requires_grad_(c["train"]), k.detach().requires_grad_(c["train"])
        if c["train"]:
            s["gq"], s["gk"] = (normal(B, T, hq, D) * 0.02).to(dt), (normal(B, T, hk, D) * 0.02).to(dt)
        s["cos"], s["sin"] = _tables(c, dev)
        s["positions"] = None
        if c["positions"] == "far":                                                 # sequences that have already run for long
            start = torch.randint(0, c["table"] - T + 1, (B, 1), device=dev, generator=g)
            s["positions"] = start + torch.arange(T, device=dev)
        elif c["positions"] == "documents":                                         # counting starts again at each document
            cut = (torch.rand(B, T, device=dev, generator=g) < 1 / 700).cumsum(-1)
            at = torch.arange(T, device=dev).expand(B, T)
            first = torch.full((B, T + 1), T, device=dev).scatter_reduce(1, cut, at, "amin")
            s["positions"] = at - first.gather(1, cut)
    elif c["op"] == "kl_topk":
        rows, V, K = c["rows"], c["vocab"], c["keep"]
        base = normal(rows, V)
        teacher = base * 2.0 + 1.5 * normal(rows, V)
        values, index = teacher.topk(K, dim=-1)
        s["lse"] = None
        if c["norm"] == "full":
            s["lse"] = torch.logsumexp(teacher / c["tau"], dim=-1)
        del teacher
        s["student"] = base.mul_(2.0).add_(normal(rows, V)).to(dt).requires_grad_(c["train"])
        if c["holes"]:                                   # rows of padding, and rows that kept fewer than K
            whole = torch.rand(rows, 1, device=dev, generator=g) < c["holes"]
            tail = (torch.rand(rows, 1, device=dev, generator=g) < c["holes"]) & (torch.arange(K, device=dev) >= max(1, K // 2))
            index = index.masked_fill(whole | tail, -1)
        s["values"], s["index"] = values.to(DTYPES[c["tdtype"]]), index
    else:
        N, E = c["tokens"], c["experts"]
        s["logits"] = (normal(N, E) + 0.5 * normal(E)).to(dt).requires_grad_(c["train"])
        s["bias"] = 0.02 * normal(E) if c["bias"] else None
        s["coefs"] = (1e-2, 1e-3) if c["aux"] else (0.0, 0.0)
        if c["train"]:
            s["dw"] = 0.02 * normal(N, c["k"])
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(state):
    step = {"layer_norm": _layer_norm, "rotary": _rotary, "kl_topk": _kl_topk, "route": _route}[state["case"]["op"]]
    if own:
        return _OWN[state["case"]["op"]](state)
    with torch.no_grad():
        return step(state)


def _layer_norm(s):
    c = s["case"]
    dt = s["x"].dtype
    x = s["x"].float()
    out = {}
    if c["add"]:
        out["sum"] = (x + s["delta"].float()).to(dt)
        x = out["sum"].float()                            # the norm is that of the sum as it is stored
    centred = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + LN_EPS)
    xh = centred * rstd
    out["y"] = (xh * s["w"].float() + s["b"].float() if c["affine"] else xh).to(dt)
    if c["train"]:
        dy = s["dy"].float()
        g = dy * s["w"].float() if c["affine"] else dy
        dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
        if c["add"]:
            dx = dx + s["ds"].float()
        out["dx"] = dx.to(dt)
        if c["affine"]:
            out["dw"], out["db"] = (dy * xh).sum(0).to(s["w"].dtype), dy.sum(0).to(s["b"].dtype)
    return out


def _turn(x, cos, sin, interleaved):
    """Rotation of the first ``2 * cos.shape[-1]`` values of each head; ``cos``, ``sin`` ``[B or 1, T, 1, R/2]``."""
    R = 2 * cos.shape[-1]
    xf = x.float()
    a, b = (xf[..., 0:R:2], xf[..., 1:R:2]) if interleaved else (xf[..., : R // 2], xf[..., R // 2: R])
    u, v = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((turned, xf[..., R:]), -1).to(x.dtype)


def _rotary(s):
    c, pos = s["case"], s["positions"]
    if pos is None:
        cos, sin = s["cos"][None, : c["seq"], None], s["sin"][None, : c["seq"], None]
    else:
        cos, sin = s["cos"][pos][:, :, None], s["sin"][pos][:, :, None]
    out = {"q": _turn(s["q"], cos, sin, c["interleaved"]), "k": _turn(s["k"], cos, sin, c["interleaved"])}
    if c["train"]:
        out["dq"], out["dk"] = _turn(s["gq"], cos, -sin, c["interleaved"]), _turn(s["gk"], cos, -sin, c["interleaved"])
    return out


def _kl_topk(s):
    c, tau = s["case"], s["case"]["tau"]
    z = s["student"].float() / tau
    held = s["index"] >= 0
    at = s["index"].clamp(min=0)
    t = (s["values"].float() / tau).masked_fill(~held, -math.inf)
    has = held.any(-1)
    if c["norm"] == "full":
        logp = t - s["lse"][:, None]
    else:
        top = t.amax(-1, keepdim=True).masked_fill(~has[:, None], 0.0)
        logp = t - (top + (t - top).exp().sum(-1, keepdim=True).log())
    p = logp.exp().masked_fill(~held, 0.0)
    top = z.amax(-1, keepdim=True)
    e = (z - top).exp()
    total = e.sum(-1, keepdim=True)
    logq = z.gather(-1, at) - top - total.log()
    each = torch.where(held, p * (logp - logq), 0.0).sum(-1)
    n = has.sum().clamp(min=1).float()
    out = {"loss": each.sum() / n}
    if c["train"]:
        g = (e / total) * p.sum(-1, keepdim=True)
        g = g.scatter_add(-1, at, -p) / (n * tau)
        out["grad"] = g.to(s["student"].dtype)
    return out


def _route(s):
    c = s["case"]
    E, k, (aux_coef, z_coef) = c["experts"], c["k"], s["coefs"]
    z = s["logits"].double()
    N = z.shape[0]
    lse = torch.logsumexp(z, -1, keepdim=True)
    soft = (z - lse).exp()
    score = soft if c["score"] == "softmax" else torch.sigmoid(z)
    pick = score if s["bias"] is None else score + s["bias"].double()
    if c["groups"] > 1:
        each = pick.view(N, c["groups"], -1)
        best = each.sort(dim=-1, descending=True).values[..., : c["best"]].sum(-1)
        kept = best.sort(dim=-1, descending=True, stable=True).indices[:, : c["top_groups"]]
        open_ = torch.zeros_like(best, dtype=torch.bool).scatter_(-1, kept, True)
        pick = each.masked_fill(~open_[..., None], -math.inf).view(N, E)
    idx = pick.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    chosen = score.gather(-1, idx)
    total = chosen.sum(-1, keepdim=True)
    weights = chosen / total if c["renorm"] else chosen
    ones = torch.ones(N * k, dtype=torch.int32, device=z.device)
    counts = torch.zeros(E, dtype=torch.int32, device=z.device).scatter_add_(0, idx.reshape(-1), ones)
    out = {"weights": weights.float(), "idx": idx.to(torch.int32), "counts": counts}
    norm = score.sum(-1, keepdim=True)
    share, load = score / norm, counts.double() / (N * k)
    if c["aux"]:
        out["aux"] = (aux_coef * E * (load * share.mean(0)).sum() + z_coef * (lse * lse).mean()).float()
    if c["train"]:
        dw = s["dw"].double()
        ds = torch.zeros_like(score)
        ds.scatter_(-1, idx, (dw - (dw * weights).sum(-1, keepdim=True)) / total if c["renorm"] else dw)
        dz = torch.zeros_like(score)
        if c["aux"]:
            dp = aux_coef * E / N * load
            ds = ds + (dp - (share * dp).sum(-1, keepdim=True)) / norm
            dz = z_coef * 2 / N * lse * soft
        if c["score"] == "softmax":
            dz = dz + score * (ds - (score * ds).sum(-1, keepdim=True))
        else:
            dz = dz + ds * score * (1 - score)
        out["grad"] = dz.to(s["logits"].dtype)
    return out


# ------------------------------------------------------------------------------------------ the framework's calls
def _own_layer_norm(s):
    from forgeminds_b200 import kernels as K
    c = s["case"]
    if c["add"]:
        total, y = K.add_layer_norm(s["x"], s["delta"], s["w"], s["b"], LN_EPS)
        out = {"sum": total.detach(), "y": y.detach()}
    else:
        y = K.layer_norm(s["x"], s["w"], s["b"], LN_EPS)
        out = {"y": y.detach()}
    if c["train"]:
        leaves = [s["x"]] + ([s["w"], s["b"]] if c["affine"] else [])
        grads = torch.autograd.grad((total, y), leaves, (s["ds"], s["dy"])) if c["add"] else \
            torch.autograd.grad(y, leaves, s["dy"])
        out["dx"] = grads[0]
        if c["affine"]:
            out["dw"], out["db"] = grads[1:]
    return out


def _own_rotary(s):
    from forgeminds_b200 import kernels as K
    c = s["case"]
    q, k = K.rotary_qk(s["q"], s["k"], s["cos"], s["sin"], positions=s["positions"], interleaved=c["interleaved"])
    out = {"q": q.detach(), "k": k.detach()}
    if c["train"]:
        out["dq"], out["dk"] = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"]))
    return out


def _own_kl_topk(s):
    from forgeminds_b200 import kernels as K
    c = s["case"]
    loss = K.kl_topk_logits(s["student"], s["values"], s["index"], temperature=c["tau"], teacher_lse=s["lse"])
    out = {"loss": loss.detach()}
    if c["train"]:
        (out["grad"],) = torch.autograd.grad(loss, s["student"])
    return out


def _own_route(s):
    from forgeminds_b200 import kernels as K
    c = s["case"]
    w, idx, counts, aux = K.route_experts(s["logits"], c["k"], score=c["score"], bias=s["bias"], n_groups=c["groups"],
                                          top_groups=c["top_groups"], group_best=c["best"], renormalise=c["renorm"],
                                          aux_coef=s["coefs"][0], z_coef=s["coefs"][1])
    out = {"weights": w.detach(), "idx": idx, "counts": counts}
    if c["aux"]:
        out["aux"] = aux.detach()
    if c["train"]:
        if c["aux"]:
            (out["grad"],) = torch.autograd.grad((w, aux), s["logits"], (s["dw"], torch.ones_like(aux)))
        else:
            (out["grad"],) = torch.autograd.grad(w, s["logits"], s["dw"])
    return out


_OWN = {"layer_norm": _own_layer_norm, "rotary": _own_rotary, "kl_topk": _own_kl_topk, "route": _own_route}


# ------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        return {"layer_norm": _exact_layer_norm, "rotary": _exact_rotary, "kl_topk": _exact_kl_topk,
                "route": _exact_route}[case["op"]](s)


def _exact_layer_norm(s):
    c, out = s["case"], {}
    x = s["x"].double()
    if c["add"]:
        out["sum"] = x + s["delta"].double()
        x = (s["x"].float() + s["delta"].float()).to(s["x"].dtype).double()
    var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    sd = (var + LN_EPS).sqrt()
    xh = (x - mean) / sd
    w = s["w"].double() if c["affine"] else torch.ones((), dtype=F64, device=x.device)
    out["y"] = xh * w + s["b"].double() if c["affine"] else xh
    if c["train"]:
        dy, d = s["dy"].double(), x.shape[-1]
        g = dy * w
        dx = (d * g - g.sum(-1, keepdim=True) - xh * (xh * g).sum(-1, keepdim=True)) / (d * sd)
        out["dx"] = dx + s["ds"].double() if c["add"] else dx
        if c["affine"]:
            out["dw"], out["db"] = torch.einsum("nd,nd->d", dy, xh), torch.einsum("nd->d", dy)
    return out


def _exact_rotary(s):
    c = s["case"]
    B, T, R = c["batch"], c["seq"], c["rot"]
    pos = torch.arange(T, device=s["q"].device).expand(B, T) if s["positions"] is None else s["positions"]
    unit = torch.complex(s["cos"].double(), s["sin"].double())[pos.reshape(-1)].view(B, T, 1, R // 2)

    def turn(x, factor):
        y = x.double().clone()
        first, second = (slice(0, R, 2), slice(1, R, 2)) if c["interleaved"] else (slice(0, R // 2), slice(R // 2, R))
        z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * factor
        y[..., first], y[..., second] = z.real, z.imag
        return y

    out = {"q": turn(s["q"], unit), "k": turn(s["k"], unit)}
    if c["train"]:
        out["dq"], out["dk"] = turn(s["gq"], unit.conj()), turn(s["gk"], unit.conj())
    return out


def _exact_kl_topk(s):
    c = s["case"]
    rows, V = s["student"].shape
    grad = torch.zeros(rows, V, dtype=F64, device="cuda") if c["train"] else None
    live = (s["index"] >= 0).any(-1)
    n = max(1, int(live.sum()))
    total = 0.0
    for lo in range(0, rows, 512):
        some = slice(lo, lo + 512)
        held, at = s["index"][some] >= 0, s["index"][some].clamp(min=0)
        t = (s["values"][some].double() / c["tau"]).masked_fill(~held, -1e300)
        base = s["lse"][some, None].double() if c["norm"] == "full" else torch.logsumexp(t, -1, keepdim=True)
        p = torch.where(held, (t - base).exp(), 0.0)
        logq = torch.log_softmax(s["student"][some].double() / c["tau"], -1)
        total += float((torch.special.xlogy(p, p) - p * logq.gather(-1, at)).sum())
        if c["train"]:
            want = torch.zeros_like(logq).scatter_add_(-1, at, p)
            grad[some] = (logq.exp() * p.sum(-1, keepdim=True) - want) / (n * c["tau"])
    out = {"loss": torch.tensor(total / n, dtype=F64, device="cuda")}
    if c["train"]:
        out["grad"] = grad
    return out


def _exact_route(s):
    c = s["case"]
    z = s["logits"].detach().float().cpu().numpy().astype(np.float64)
    N, E = z.shape
    k, (aux_coef, z_coef) = c["k"], s["coefs"]
    high = z.max(1, keepdims=True)
    e = np.exp(z - high)
    mass = e.sum(1, keepdims=True)
    soft, lse = e / mass, np.log(mass) + high
    score = soft if c["score"] == "softmax" else 1.0 / (1.0 + np.exp(-z))
    pick = score + (0.0 if s["bias"] is None else s["bias"].cpu().numpy().astype(np.float64))
    if c["groups"] > 1:
        each = pick.reshape(N, c["groups"], -1)
        best = -np.sort(-each, axis=2)[:, :, : c["best"]].sum(2)
        out_of = np.argsort(-best, axis=1, kind="stable")[:, c["top_groups"]:]
        shut = np.zeros(best.shape, bool)
        np.put_along_axis(shut, out_of, True, 1)
        pick = np.where(np.repeat(shut, E // c["groups"], 1), -np.inf, pick)
    idx = np.argsort(-pick, axis=1, kind="stable")[:, :k]
    chosen = np.take_along_axis(score, idx, 1)
    weights = chosen / chosen.sum(1, keepdims=True) if c["renorm"] else chosen
    counts = np.bincount(idx.ravel(), minlength=E)
    norm = score.sum(1, keepdims=True)
    load = counts / (N * k)
    out = {"weights": weights, "idx": None, "counts": None}
    if c["aux"]:
        out["aux"] = np.float64(aux_coef * E * (load * (score / norm).mean(0)).sum() + z_coef * (lse ** 2).mean())
    if c["train"]:
        dw = s["dw"].cpu().numpy().astype(np.float64)
        part = (dw - (dw * weights).sum(1, keepdims=True)) / chosen.sum(1, keepdims=True) if c["renorm"] else dw
        ds = np.zeros((N, E))
        np.put_along_axis(ds, idx, part, 1)
        if c["aux"]:
            dp = aux_coef * E / N * load
            ds += (dp - (score * dp).sum(1, keepdims=True) / norm) / norm
        dz = score * (ds - (score * ds).sum(1, keepdims=True)) if c["score"] == "softmax" else ds * score * (1 - score)
        out["grad"] = dz + z_coef * 2 / N * lse * soft
    return out
