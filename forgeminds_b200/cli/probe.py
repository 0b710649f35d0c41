"""Awkward-shape probe: every public kernel at shapes that hit its tail paths, forward and backward,
against the PyTorch statement of the same op.

``python -m forgeminds_b200.cli probe [--device cuda|cpu] [--json]``

Shapes on purpose: row counts that are not a multiple of the rows a block handles, widths that are not a
power of two (but keep the kernels' 8-element alignment), the split SwiGLU layout, a vocabulary that does
not fit one pass of the KL kernel, a top-k with k close to the width, a ragged attention sequence and a
matrix product whose sizes are not multiples of the tile. On a B200 the sm_100a kernels run and the device
status word (bounded waits, and the address checks of the debug build when ``FORGEMINDS_DEBUG_SO=1`` loads
it) is read after every case; on a CPU box the same cases run through the dispatcher's PyTorch path, which
checks the dispatcher, the shape guards and the autograd contract of every op.

Exit 0 when every case matches its reference and the status word stayed clear, 1 otherwise. This is the
counterpart of the reference's ``tools/tilelens_probe.py`` (which drives its Triton kernels through an
interpreter-based sanitizer): the bounds checks here are compiled into the debug library instead.
"""
from __future__ import annotations

import argparse
import json
import math
import sys

import torch


def _cases(dev, dt):
    """``(name, fn(inputs) -> tensor or tuple, reference fn, inputs, tolerance)``"""
    from .. import kernels as K
    from ..kernels import reference as R
    g = torch.Generator(device="cpu").manual_seed(11)

    def rnd(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g) * scale).to(device=dev, dtype=dtype)

    T, hd = 37, 48
    ang = torch.outer(torch.arange(T, dtype=torch.float32), 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float32) / hd))
    cos, sin = ang.cos().to(dev)[None, :, None, :], ang.sin().to(dev)[None, :, None, :]
    kept, kept_at = rnd(65, 5001, dtype=torch.float32).topk(9, dim=-1)
    bias, groups = rnd(40, scale=0.1, dtype=torch.float32), dict(score="sigmoid", n_groups=5, top_groups=3)
    out = [
        ("rms_norm 1003x1032", lambda a: K.rms_norm(a[0], a[1], 1e-6), lambda a: R.rms_norm(a[0], a[1], 1e-6),
         [rnd(1003, 1032), rnd(1032, dtype=torch.float32)], 3e-2),
        ("add_rms_norm 517x200", lambda a: K.add_rms_norm(a[0], a[1], a[2]), lambda a: R.add_rms_norm(a[0], a[1], a[2]),
         [rnd(517, 200), rnd(517, 200), rnd(200, dtype=torch.float32)], 3e-2),
        ("swiglu 333x1416", lambda a: K.swiglu(a[0], a[1]), lambda a: R.swiglu(a[0], a[1]),
         [rnd(333, 1416), rnd(333, 1416)], 3e-2),
        ("swiglu_split 129x(2x712)", lambda a: K.swiglu_split(a[0]), lambda a: R.swiglu_split(a[0]), [rnd(129, 1424)], 3e-2),
        ("qk_norm_rope 3x37x5x48", lambda a: K.qk_norm_rope(a[0], a[1], cos, sin),
         lambda a: R.qk_norm_rope(a[0], a[1], cos, sin), [rnd(3, T, 5, hd), rnd(hd, dtype=torch.float32)], 4e-2),
        ("softmax 77x136", lambda a: K.softmax(a[0]), lambda a: R.softmax(a[0]), [rnd(77, 136)], 2e-2),
        ("kl_div_logits 65x5000", lambda a: K.kl_div_logits(a[0], a[1].detach()),       # the teacher is a constant
         lambda a: R.kl_div_logits(a[0], a[1].detach())[0],
         [rnd(65, 5000), rnd(65, 5000)], 3e-2),
        ("layer_norm 1003x1030", lambda a: K.layer_norm(*a), lambda a: R.layer_norm(*a),
         [rnd(1003, 1030), rnd(1030, dtype=torch.float32), rnd(1030, dtype=torch.float32)], 3e-2),
        ("add_layer_norm 517x2056", lambda a: K.add_layer_norm(*a), lambda a: R.add_layer_norm(*a),
         [rnd(517, 2056), rnd(517, 2056), rnd(2056, dtype=torch.float32), rnd(2056, dtype=torch.float32)], 3e-2),
        ("rotary 3x37x5x48, 20 of 48 interleaved", lambda a: K.rotary(a[0], cos[0, :, 0, :10], sin[0, :, 0, :10], None, True),
         lambda a: R.rotary(a[0], cos[0, :, 0, :10], sin[0, :, 0, :10], None, True), [rnd(3, T, 5, hd)], 2e-2),
        ("kl_topk_logits 65x5001", lambda a: K.kl_topk_logits(a[0], kept, kept_at),
         lambda a: R.kl_topk(a[0], kept, kept_at).mean(), [rnd(65, 5001)], 3e-2),
        ("route_experts 61x40, 3 of 5 groups", lambda a: K.route_experts(a[0], 6, bias=bias, **groups)[0],
         lambda a: R.route_experts(a[0], 6, False, bias, 5, 3)[0], [rnd(61, 40)], 2e-2),
    ]
    return out


def _flat(v):
    return [t for t in (v if isinstance(v, (tuple, list)) else (v,)) if torch.is_tensor(t)]


def _rel(a, b):
    a, b = a.detach().float(), b.detach().float()
    return float((a - b).norm() / b.norm().clamp(min=1e-6))


def _status(dev):
    """Device status word (0 = clear) on a CUDA box with the native library; None elsewhere."""
    if dev.type != "cuda":
        return None
    from .. import ops
    if not ops.available():
        return None
    word = ops.status_word(dev)
    code = int(word.item())
    word.zero_()
    return code


def run(dev, dt):
    rows = []
    for name, fn, ref, inputs, tol in _cases(dev, dt):
        row = {"case": name, "ok": True, "status": None}
        try:
            ins = [t.clone().requires_grad_(t.is_floating_point()) for t in inputs]
            rin = [t.detach().float().requires_grad_(t.is_floating_point()) for t in inputs]
            got, want = _flat(fn(ins)), _flat(ref(rin))
            row["fwd"] = max(_rel(g, w) for g, w in zip(got, want))
            seeds = [torch.randn(w.shape, generator=torch.Generator().manual_seed(5)).to(w.device) for w in want]
            torch.autograd.backward(got, [s.to(g.dtype) for s, g in zip(seeds, got)])
            torch.autograd.backward(want, [s.to(w.dtype) for s, w in zip(seeds, want)])
            row["bwd"] = max(_rel(a.grad, b.grad) for a, b in zip(ins, rin) if a.grad is not None and b.grad is not None)
            row["ok"] = row["fwd"] < tol and row["bwd"] < 2 * tol
        except Exception as e:                                    # noqa: BLE001 - the probe reports, it does not stop
            row["ok"], row["error"] = False, f"{type(e).__name__}: {e}"
        row["status"] = _status(dev)
        if row["status"]:
            row["ok"] = False
        rows.append(row)
    rows += _selection_cases(dev, dt)
    if dev.type == "cuda":
        rows += _tensor_core_cases(dev)
    return rows


def _selection_cases(dev, dt):
    from .. import kernels as K
    from ..kernels import reference as R
    g = torch.Generator(device="cpu").manual_seed(3)
    x = torch.randn(61, 72, generator=g).to(device=dev, dtype=dt)
    rows = []
    for k in (1, 7, 70):
        row = {"case": f"topk 61x72 k={k}", "ok": True, "status": None}
        try:
            v, i = K.topk(x, k)
            rv, ri = R.topk(x, k)
            row["fwd"] = float((v.float() - rv.float()).abs().max())
            # ties may be ordered differently: compare the selected values, and the indices through a gather
            row["ok"] = row["fwd"] == 0.0 and bool(torch.equal(x.gather(-1, i.long()), v))
        except Exception as e:                                    # noqa: BLE001
            row["ok"], row["error"] = False, f"{type(e).__name__}: {e}"
        row["status"] = _status(dev)
        rows.append(row)
    return rows


def _tensor_core_cases(dev):
    """Products and attention at sizes that are not multiples of their tiles (B200 only)."""
    from .. import ops
    if not ops.available():
        return []
    from ..ops import functional as Fn
    g = torch.Generator(device="cpu").manual_seed(9)
    rows = []
    for m, n, k in ((1000, 264, 520), (130, 1032, 72), (8, 8, 8)):
        row = {"case": f"gemm {m}x{n}x{k}", "ok": True}
        try:
            a = torch.randn(m, k, generator=g).to(dev, torch.bfloat16)
            b = torch.randn(n, k, generator=g).to(dev, torch.bfloat16)
            y = Fn.gemm(a, b)
            row["fwd"] = _rel(y, a.float() @ b.float().t())
            row["ok"] = row["fwd"] < 1e-2
        except Exception as e:                                    # noqa: BLE001
            row["ok"], row["error"] = False, f"{type(e).__name__}: {e}"
        row["status"] = _status(dev)
        row["ok"] = row["ok"] and not row["status"]
        rows.append(row)
    for B, T, hq, hkv, hd in ((1, 203, 4, 2, 64), (2, 131, 6, 2, 80), (1, 300, 4, 1, 128)):
        row = {"case": f"attention B{B} T{T} {hq}/{hkv} hd{hd}", "ok": True}
        try:
            qkv = torch.randn(B, T, (hq + 2 * hkv) * hd, generator=g).to(dev, torch.bfloat16).requires_grad_()
            out = Fn.attention_qkv(qkv, hq, hkv, hd, True)
            seed = torch.randn(out.shape, generator=g).to(dev, torch.bfloat16)
            out.backward(seed)
            ref_in = qkv.detach().float().requires_grad_()
            q = ref_in[..., : hq * hd].unflatten(-1, (hq, hd)).transpose(1, 2)
            kk = ref_in[..., hq * hd: (hq + hkv) * hd].unflatten(-1, (hkv, hd)).transpose(1, 2)
            v = ref_in[..., (hq + hkv) * hd:].unflatten(-1, (hkv, hd)).transpose(1, 2)
            rep = hq // hkv
            s = q @ kk.repeat_interleave(rep, 1).transpose(-1, -2) / math.sqrt(hd)
            s = s.masked_fill(~torch.ones(T, T, dtype=torch.bool, device=dev).tril(), float("-inf"))
            ro = (torch.softmax(s, -1) @ v.repeat_interleave(rep, 1)).transpose(1, 2).reshape(B, T, hq * hd)
            ro.backward(seed.float())
            row["fwd"], row["bwd"] = _rel(out, ro), _rel(qkv.grad, ref_in.grad)
            row["ok"] = row["fwd"] < 2e-2 and row["bwd"] < 3e-2
        except Exception as e:                                    # noqa: BLE001
            row["ok"], row["error"] = False, f"{type(e).__name__}: {e}"
        row["status"] = _status(dev)
        row["ok"] = row["ok"] and not row["status"]
        rows.append(row)
    return rows


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(prog="forgeminds_b200.cli probe", description=__doc__.split("\n\n")[0])
    ap.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    ap.add_argument("--dtype", default=None, choices=("bf16", "fp32"))
    ap.add_argument("--json", action="store_true")
    a = ap.parse_args(argv)
    dev = torch.device(a.device)
    dt = {"bf16": torch.bfloat16, "fp32": torch.float32, None: torch.bfloat16 if dev.type == "cuda" else torch.float32}[a.dtype]
    from .. import kernels as K
    K.reset_stats()
    rows = run(dev, dt)
    if a.json:
        print(json.dumps({"rows": rows, "paths": K.stats()}, indent=1, default=str))
    else:
        for r in rows:
            tail = r.get("error") or f"fwd {r.get('fwd', float('nan')):.2e}" + (f"  bwd {r['bwd']:.2e}" if "bwd" in r else "")
            st = "" if r.get("status") in (None, 0) else f"  STATUS {r['status']}"
            print(f"{'ok  ' if r['ok'] else 'FAIL'} {r['case']:<34}{tail}{st}")
        print("paths taken:", K.stats())
    return 0 if all(r["ok"] for r in rows) else 1


if __name__ == "__main__":
    sys.exit(main())
