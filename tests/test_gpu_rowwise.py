"""LayerNorm, rotary positions, top-logit distillation and expert routing on the GPU against their definitions in 64 bits."""
import pytest
import torch

import rowwise_oracle as oracle
from rowwise_oracle import U32, within

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def K():
    import forgeminds_b200 as fm
    return fm.kernels


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, device="cuda", generator=gen(seed)) * scale).to(dtype)


@pytest.fixture(autouse=True)
def on_the_kernels():
    """Every test here runs on the kernels: a silent fall-back fails it."""
    K().reset_stats()
    yield
    st = K().stats()
    assert st["fast"] > 0 and st["fallback"] == 0, st


# ------------------------------------------------------------------------------ LayerNorm
LN_CASES = [(1, 1), (3, 7), (8, 64), (5, 1000), (300, 256), (300, 264), (77, 257), (129, 512), (64, 1024), (33, 1030), (40, 2048),
            (19, 4096), (9, 4099), (7, 8192), (5, 8200), (3, 16384), (3, 16392), (2, 16391), (2, 40000), (1, 70001)]


@pytest.mark.parametrize("rows,d", LN_CASES)
@pytest.mark.parametrize("dtype,wdtype", [("bf16", "bf16"), ("bf16", "fp32"), ("fp32", "fp32")])
def test_layer_norm(rows, d, dtype, wdtype):
    x = (randn(rows, d, seed=1) * 1.5 + 0.7).to(DT[dtype]).requires_grad_()
    w = (1 + 0.3 * randn(d, seed=2)).to(DT[wdtype]).requires_grad_()
    b = (0.2 * randn(d, seed=3)).to(DT[wdtype]).requires_grad_()
    dy = randn(rows, d, seed=4, dtype=DT[dtype])
    y = K().layer_norm(x, w, b, 1e-5)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert dw.dtype == w.dtype and dx.dtype == x.dtype
    want, off = oracle.layer_norm(x.detach(), w.detach(), b.detach(), 1e-5, dy)
    for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        assert within(got.detach(), want[name], off[name]) <= 0, name
    with torch.no_grad():
        assert torch.equal(K().layer_norm(x, w, b, 1e-5), y)


@pytest.mark.parametrize("rows,d", [(3, 7), (65, 1024), (17, 4096), (5, 1001), (2, 20000)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_add_layer_norm(rows, d, dtype):
    x, e = randn(rows, d, seed=5, dtype=DT[dtype]).requires_grad_(), randn(rows, d, seed=6, dtype=DT[dtype]).requires_grad_()
    w, b = (1 + 0.3 * randn(d, seed=7)).requires_grad_(), (0.2 * randn(d, seed=8)).requires_grad_()
    dy, ds = randn(rows, d, seed=9, dtype=DT[dtype]), randn(rows, d, seed=10, dtype=DT[dtype])
    total, y = K().add_layer_norm(x, e, w, b, 1e-5)
    assert torch.equal(total, (x.float() + e.float()).to(x.dtype))
    dx, de, dw, db = torch.autograd.grad((total, y), (x, e, w, b), (ds, dy), retain_graph=True)
    assert torch.equal(dx, de)
    want, off = oracle.layer_norm(total.detach(), w.detach(), b.detach(), 1e-5, dy, ds)
    for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        assert within(got.detach(), want[name], off[name]) <= 0, name
    # one of the two results alone
    (dx,) = torch.autograd.grad(y, x, dy, retain_graph=True)
    want, off = oracle.layer_norm(total.detach(), w.detach(), b.detach(), 1e-5, dy)
    assert within(dx, want["dx"], off["dx"]) <= 0
    (dx,) = torch.autograd.grad(total, x, ds)
    assert torch.equal(dx, ds)


@pytest.mark.parametrize("affine", ["none", "w", "b", "mixed"])
def test_layer_norm_parts_of_the_affine(affine):
    x, dy = randn(37, 320, seed=11, dtype=torch.bfloat16).requires_grad_(), randn(37, 320, seed=12, dtype=torch.bfloat16)
    w = None if affine in ("none", "b") else (1 + 0.1 * randn(320, seed=13)).to(torch.bfloat16).requires_grad_()
    b = None if affine in ("none", "w") else (0.1 * randn(320, seed=14)).requires_grad_()       # mixed: fp32 beside a bf16 weight
    y = K().layer_norm(x, w, b, 1e-5)
    leaves = [t for t in (x, w, b) if t is not None]
    got = dict(zip([n for n, t in (("dx", x), ("dw", w), ("db", b)) if t is not None], torch.autograd.grad(y, leaves, dy)))
    want, off = oracle.layer_norm(x.detach(), None if w is None else w.detach(), None if b is None else b.detach(), 1e-5, dy)
    assert within(y.detach(), want["y"], off["y"]) <= 0
    for name, g in got.items():
        assert within(g, want[name], off[name]) <= 0, name


def test_layer_norm_strides_and_broadcast_inputs():
    wide = randn(6, 50, 264, seed=15, dtype=torch.bfloat16)
    w, b = 1 + 0.1 * randn(256, seed=16), 0.1 * randn(256, seed=17)
    for x in (wide[..., :256], wide[..., 8:], wide[..., 3:259], wide[:, ::2, :256], wide[..., :256].transpose(0, 1)):
        x = x.detach().requires_grad_()
        y = K().layer_norm(x, w, b)
        dy = randn(*x.shape, seed=18, dtype=torch.bfloat16)
        (dx,) = torch.autograd.grad(y, x, dy)
        want, off = oracle.layer_norm(x.detach().reshape(-1, 256), w, b, 1e-5, dy.reshape(-1, 256))
        assert within(y.detach().reshape(-1, 256), want["y"], off["y"]) <= 0
        assert within(dx.reshape(-1, 256), want["dx"], off["dx"]) <= 0
    # one row for all, and a gradient that is one number everywhere
    row = randn(1, 256, seed=19, dtype=torch.float32).requires_grad_()
    y = K().layer_norm(row.expand(40, 256), w, b)
    (g,) = torch.autograd.grad(y.sum(), row)
    want, off = oracle.layer_norm(row.detach().expand(40, 256), w, b, 1e-5, torch.ones(40, 256, device="cuda"))
    assert within(g, want["dx"].sum(0, keepdim=True), off["dx"].sum(0, keepdim=True) + 40 * U32 * want["dx"].abs().sum(0, keepdim=True)) <= 0


def test_layer_norm_rows_without_spread_and_with_nan():
    x = torch.full((4, 512), 3.0, device="cuda")
    x[1] = 0.0
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    w, b = torch.full((512,), 2.0, device="cuda"), torch.full((512,), 0.25, device="cuda")
    y = K().layer_norm(x, w, b)
    assert torch.equal(y[:2], torch.full((2, 512), 0.25, device="cuda")) and bool(torch.isnan(y[2:]).all())


def test_layer_norm_large_offset_keeps_its_precision():
    """Values of spread 1 around 4096: a variance from sums of squares would lose them in fp32."""
    x = randn(16, 1024, seed=20) + 4096.0
    want, off = oracle.layer_norm(x, None, None, 1e-5)
    y = K().layer_norm(x)
    assert within(y, want["y"], off["y"]) <= 0
    assert float((y.double() - want["y"]).abs().max()) < 1e-3


def test_layer_norm_no_rows():
    x = torch.empty(0, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w, b = torch.ones(128, device="cuda", requires_grad=True), torch.zeros(128, device="cuda", requires_grad=True)
    y = K().layer_norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b))
    assert y.shape == (0, 128) and gx.shape == x.shape and not gw.any() and not gb.any()


def test_layer_norm_is_the_same_every_time():
    x, dy = randn(5000, 1024, seed=21, dtype=torch.bfloat16).requires_grad_(), randn(5000, 1024, seed=22, dtype=torch.bfloat16)
    w, b = torch.ones(1024, device="cuda", requires_grad=True), torch.zeros(1024, device="cuda", requires_grad=True)
    first = None
    for _ in range(3):
        got = torch.autograd.grad(K().layer_norm(x, w, b), (x, w, b), dy)
        first = first or got
        assert all(torch.equal(a, c) for a, c in zip(first, got))


# ------------------------------------------------------------------------------ rotary positions
ROTARY_SHAPES = [(1, 1, 1, 1, 2, 2), (2, 5, 3, 1, 10, 6), (2, 33, 4, 2, 64, 64), (1, 17, 7, 1, 80, 80), (3, 9, 8, 8, 128, 64),
                 (2, 40, 4, 4, 96, 32), (1, 7, 2, 1, 192, 48), (2, 11, 5, 5, 256, 256), (64, 1, 32, 8, 128, 128), (1, 300, 16, 4, 72, 24)]


@pytest.mark.parametrize("B,T,hq,hk,D,R", ROTARY_SHAPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("packed", [False, True])
def test_rotary_qk(B, T, hq, hk, D, R, interleaved, dtype, packed):
    cos, sin = K().rotary_tables(max(T, 50), R, device="cuda")
    if packed:
        qkv = randn(B, T, (hq + 2 * hk) * D, seed=30, dtype=DT[dtype])
        q, k = qkv[..., : hq * D].unflatten(-1, (hq, D)), qkv[..., hq * D: (hq + hk) * D].unflatten(-1, (hk, D))
    else:                                                   # heads first, as attention keeps them
        q, k = randn(B, hq, T, D, seed=31, dtype=DT[dtype]).transpose(1, 2), randn(B, hk, T, D, seed=32, dtype=DT[dtype]).transpose(1, 2)
    q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
    at = torch.randint(0, cos.shape[0], (B, T), device="cuda", generator=gen(33))
    for positions in (None, at, at[0].to(torch.int32)):
        a, b = K().rotary_qk(q, k, cos, sin, positions, interleaved)
        ga, gb = randn(*a.shape, seed=34, dtype=DT[dtype]), randn(*b.shape, seed=35, dtype=DT[dtype])
        dq, dk = torch.autograd.grad((a, b), (q, k), (ga, gb))
        for got, x, sign in ((a, q, 1), (b, k, 1), (dq, ga, -1), (dk, gb, -1)):
            want, off = oracle.rotary(x.detach(), cos, sin, positions, interleaved, sign)
            assert within(got.detach(), want, off) <= 0
        assert torch.equal(K().rotary(q.detach(), cos, sin, positions, interleaved), a)


def test_rotary_one_gradient_alone_and_tables_to_broadcast():
    q, k = randn(2, 6, 3, 32, seed=36).requires_grad_(), randn(2, 6, 1, 32, seed=37).requires_grad_()
    cos, sin = K().rotary_tables(6, 32, device="cuda")
    a, b = K().rotary_qk(q, k, cos, sin)
    assert torch.autograd.grad(a.sum(), (q, k), allow_unused=True, retain_graph=True)[1] is None
    (dk,) = torch.autograd.grad(b.sum(), k)
    want, off = oracle.rotary(torch.ones_like(k), cos, sin, None, False, -1.0)
    assert within(dk, want, off) <= 0
    a4, b4 = K().rotary_qk(q, k, cos[None, :, None], sin[None, :, None])
    assert torch.equal(a, a4) and torch.equal(b, b4)
    half = K().rotary(q.detach(), cos.to(torch.bfloat16), sin.to(torch.bfloat16))         # tables of another type are widened
    want, off = oracle.rotary(q.detach(), cos.to(torch.bfloat16), sin.to(torch.bfloat16), None, False)
    assert within(half, want, off) <= 0


@pytest.mark.parametrize("R", [8, 64])
def test_rotary_positions_outside_the_table(R):
    x = randn(2, 5, 3, 64, seed=38)
    cos, sin = K().rotary_tables(9, R, device="cuda")
    pos = torch.tensor([[-1, 0, 8, 9, 2 ** 40], [-2 ** 40, 3, 9, -7, 1]], device="cuda")
    for interleaved in (False, True):
        got = K().rotary(x, cos, sin, pos, interleaved)
        want, off = oracle.rotary(x, cos, sin, pos, interleaved)
        assert within(got, want, off) <= 0
        assert torch.equal(got[0, 0], x[0, 0]) and bool(torch.isnan(got[0, 3, :, :R]).all())
        assert torch.equal(got[0, 3, :, R:], x[0, 3, :, R:])


def test_rotary_far_positions_stay_exact():
    """An angle of a million turns' worth: a table in 32 bits would be off by more than the rounding of the result."""
    cos, sin = K().rotary_tables(1_000_001, 64, device="cuda")
    x = randn(1, 1, 4, 64, seed=39)
    pos = torch.tensor([1_000_000], device="cuda")
    got = K().rotary(x, cos, sin, pos)
    freq = 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64, device="cuda") / 64)
    c, s = (1_000_000 * freq).cos(), (1_000_000 * freq).sin()
    a, b = x.double().chunk(2, -1)
    want = torch.cat((a * c - b * s, a * s + b * c), -1)
    assert float((got.double() - want).abs().max()) <= 8 * U32 * float(x.abs().max()) * 2


def test_rotary_nothing_to_do():
    cos, sin = K().rotary_tables(4, 32, device="cuda")
    q = torch.empty(0, 4, 2, 32, device="cuda")
    k = torch.empty(2, 4, 0, 32, device="cuda")
    a, b = K().rotary_qk(randn(2, 4, 2, 32), k, cos, sin)
    assert b.shape == k.shape and a.shape == (2, 4, 2, 32) and K().rotary is not None
    K().layer_norm(randn(1, 8))                              # the empty call takes the PyTorch statement without counting
    assert K().rotary(q, cos, sin).shape == q.shape


# ------------------------------------------------------------------------------ distillation from top logits
def kl_inputs(rows, V, keep, seed, dtype, tdtype, spread=2.0):
    base = randn(rows, V, seed=seed)
    teacher = base * spread + randn(rows, V, seed=seed + 1)
    values, index = teacher.topk(keep, dim=-1)
    student = (base * spread + randn(rows, V, seed=seed + 2)).to(DT[dtype])
    return student, values.to(DT[tdtype]), index, teacher


def check_kl(student, values, index, tau, lse=None, reduction="mean", upstream=1.0):
    s = student.detach().requires_grad_()
    loss = K().kl_topk_logits(s, values, index, temperature=tau, reduction=reduction, teacher_lse=lse)
    up = torch.as_tensor(upstream, dtype=torch.float32, device="cuda")
    (grad,) = torch.autograd.grad(loss, s, up.expand(loss.shape) if loss.dim() else up.reshape(()), retain_graph=True)
    want, wgrad, off, goff = oracle.kl_topk(student, values, index, tau, lse, reduction, up.double())
    assert within(loss.detach(), want, off) <= 0
    assert within(grad, wgrad, goff) <= 0
    with torch.no_grad():
        assert torch.equal(K().kl_topk_logits(s, values, index, temperature=tau, reduction=reduction, teacher_lse=lse), loss)
    return s, loss, grad


@pytest.mark.parametrize("rows,V,keep", [(1, 1, 1), (3, 7, 3), (5, 100, 100), (64, 1000, 16), (17, 1001, 5), (33, 4096, 64), (9, 32000, 128),
                                         (7, 32003, 33), (3, 70000, 256), (2, 128259, 1000), (2, 300001, 8), (600, 512, 4)])
@pytest.mark.parametrize("dtype,tdtype", [("bf16", "bf16"), ("bf16", "fp32"), ("fp32", "fp32"), ("fp32", "bf16")])
def test_kl_topk(rows, V, keep, dtype, tdtype):
    student, values, index, teacher = kl_inputs(rows, V, keep, 40, dtype, tdtype)
    for tau in (1.0, 3.0):
        check_kl(student, values, index, tau)
    check_kl(student, values, index, 2.0, torch.logsumexp(teacher / 2.0, -1))


@pytest.mark.parametrize("reduction", ["sum", "none", "mean"])
def test_kl_topk_reductions_and_upstream_gradients(reduction):
    student, values, index, _ = kl_inputs(70, 3001, 12, 43, "bf16", "fp32")
    up = 1.0 if reduction != "none" else torch.where(torch.arange(70) % 3 == 0, 1.0, torch.linspace(-2, 2, 70)).cuda()
    check_kl(student, values, index, 1.5, None, reduction, up)
    check_kl(student, values, index, 1.5, None, reduction, 0.3)
    check_kl(student, values, index, 1.5, None, reduction, 0.0)
    # a second backward pass of the same graph, and another upstream gradient
    s, loss, first = check_kl(student, values, index, 1.5, None, reduction, 0.3)
    (again,) = torch.autograd.grad(loss.sum(), s, torch.tensor(0.3, device="cuda"), retain_graph=True)
    assert torch.equal(first, again)
    (other,) = torch.autograd.grad(loss.sum(), s)
    _, wgrad, _, goff = oracle.kl_topk(student, values, index, 1.5, None, reduction, 1.0)
    assert within(other, wgrad, goff) <= 0


def test_kl_topk_slots_that_do_not_count():
    student, values, index, _ = kl_inputs(9, 500, 6, 46, "fp32", "fp32")
    index, values = index.clone(), values.clone()
    index[0] = -1                                            # a row of padding
    values[1] = float("-inf")                                # a row whose mask leaves nothing
    index[2, 3:] = -1
    values[3, :2] = float("-inf")
    values[4, 1:] = torch.finfo(torch.float32).min           # a mask of the type's lowest value
    index[5, 0], index[5, 1] = 500, 2 ** 40                  # beyond the vocabulary
    index[6, 0] = -2 ** 40
    s, loss, grad = check_kl(student, values, index, 1.0)
    assert not grad[:2].any() and bool((grad[2:] != 0).any(-1).all())
    check_kl(student, values, index, 1.0, None, "none", 0.7)
    nothing = K().kl_topk_logits(student, values, torch.full_like(index, -1))
    assert float(nothing) == 0.0


def test_kl_topk_an_index_that_stands_twice():
    student, values, index, _ = kl_inputs(6, 300, 8, 49, "fp32", "fp32")
    index[:, 3] = index[:, 0]
    index[2, :] = 17
    check_kl(student, values, index, 1.0)
    check_kl(student, values, index, 1.0, torch.full((6,), 9.0, device="cuda"), "sum", -0.5)


def test_kl_topk_masked_student_logits():
    student, values, index, _ = kl_inputs(6, 300, 8, 52, "fp32", "fp32")
    keep = torch.zeros(6, 300, dtype=torch.bool, device="cuda").scatter_(1, index, True)
    off = ~keep & (torch.arange(300, device="cuda") % 2 == 0)
    check_kl(student.masked_fill(off, float("-inf")), values, index, 1.0)
    check_kl(student.masked_fill(off, torch.finfo(torch.float32).min), values, index, 1.0)
    check_kl(student * 1000, values, index, 1.0)             # one logit has everything
    s = student.clone()
    s[0] = float("-inf")
    s[1, 3] = float("nan")
    s[2, 3] = float("inf")
    s.requires_grad_()
    rows = K().kl_topk_logits(s, values, index, reduction="none")
    (grad,) = torch.autograd.grad(rows.sum(), s)
    assert bool(torch.isnan(rows[:3]).all()) and bool(torch.isfinite(rows[3:]).all())
    assert bool(torch.isnan(grad[:3]).all()) and bool(torch.isfinite(grad[3:]).all())


def test_kl_topk_strides_and_shapes():
    wide = randn(4, 6, 1030, seed=55, dtype=torch.bfloat16)
    values, index = randn(4, 6, 1000, seed=56).topk(7, dim=-1)
    for x in (wide[..., :1000], wide[..., 5:1005], wide[:, ::2, 8:1008], wide[..., :1000].transpose(0, 1)):
        rows = x.shape[:-1]
        v, i = (t.expand(*t.shape)[:, :: 2] if rows[1] == 3 else t for t in (values, index))
        if rows != v.shape[:-1]:
            v, i = v.transpose(0, 1), i.transpose(0, 1)
        x = x.detach().requires_grad_()
        out = K().kl_topk_logits(x, v, i.to(torch.int32), reduction="none")
        assert out.shape == rows
        (g,) = torch.autograd.grad(out.sum(), x)
        want, wgrad, off, goff = oracle.kl_topk(x.detach().reshape(-1, 1000), v.reshape(-1, 7), i.reshape(-1, 7), 1.0, None, "none")
        assert within(out.detach().reshape(-1), want, off) <= 0 and within(g.reshape(-1, 1000), wgrad, goff) <= 0
    assert float(K().kl_topk_logits(wide[:0, 0], values[:0, 0], index[:0, 0])) == 0.0


def test_kl_topk_agrees_with_differences():
    student, values, index, _ = kl_inputs(2, 40, 4, 58, "fp32", "fp32")
    s = student.requires_grad_()
    (g,) = torch.autograd.grad(K().kl_topk_logits(s, values, index, temperature=1.3), s)
    h = 2.0 ** -7
    for r, c in ((0, int(index[0, 0])), (0, 11), (1, int(index[1, 2])), (1, 39)):
        up, down = student.detach().clone(), student.detach().clone()
        up[r, c] += h
        down[r, c] -= h
        slope = (float(K().kl_topk_logits(up, values, index, temperature=1.3)) -
                 float(K().kl_topk_logits(down, values, index, temperature=1.3))) / (2 * h)
        # third derivatives of at most 1 times h^2 / 6, and two losses of about 5 rounded to 2^-24 of their parts
        assert abs(slope - float(g[r, c])) < h * h / 6 + 64 * U32 * 5 / h


@pytest.mark.parametrize("hdtype", ["bf16", "fp32"])
def test_kl_topk_distill_loss(hdtype):
    n, d, V, keep = 300, 64, 1000, 9
    h = randn(n, d, seed=60, dtype=DT[hdtype]).requires_grad_()
    w = (0.2 * randn(V, d, seed=61)).requires_grad_()
    values, index = (randn(n, V, seed=62) * 2).topk(keep, dim=-1)
    index = index.clone()
    index[::7] = -1
    loss = K().kl_topk_distill_loss(h, w, values, index, temperature=2.0, chunk=128)
    gh, gw = torch.autograd.grad(loss * 3.0, (h, w))
    # the definition on the logits as this path stores them: bf16 where the hidden states are bf16
    ws = w.detach().to(h.dtype)
    logits = h.detach().double() @ ws.double().t()
    want, g, off, _ = oracle.kl_topk(logits.float(), values, index, 2.0, upstream=3.0)
    step = 2.0 ** -8 if hdtype == "bf16" else 2e-3           # the fp32 product may run in tf32: ten bits of each factor
    dz = step * logits.abs().amax()                          # each logit is off by at most this
    assert abs(float(loss.detach()) - float(want)) <= 2 * float(dz) / 2.0 + float(off)
    # entries of the gradient move by at most 2 dz / tau of q + p, and are rounded to bf16 themselves
    mass = (g.abs() + 3.0 / (2.0 * int((index >= 0).any(-1).sum())) * 2) * (2 * dz / 2.0) + step * g.abs()
    assert bool(((gh.double() - g @ ws.double()).abs() <= mass @ ws.double().abs() * 1.1 + step * (g @ ws.double()).abs() + 1e-6).all())
    assert bool(((gw.double() - g.t() @ h.detach().double()).abs() <= mass.t() @ h.detach().double().abs() * 1.1 + 1e-5).all())


# ------------------------------------------------------------------------------ routing to experts
def check_route(logits, k, score="softmax", bias=None, groups=1, top_groups=1, best=2, renorm=True, scale=1.0, aux=(0.0, 0.0), daux=1.3):
    z = logits.detach().requires_grad_()
    w, idx, counts, a = K().route_experts(z, k, score=score, bias=bias, n_groups=groups, top_groups=top_groups, group_best=best,
                                          renormalise=renorm, scale=scale, aux_coef=aux[0], z_coef=aux[1])
    dw = randn(*w.shape, seed=70)
    outs, ups = ((w, a), (dw, torch.tensor(daux, device="cuda"))) if a is not None else ((w,), (dw,))
    (grad,) = torch.autograd.grad(outs, z, ups)
    want = oracle.route(logits.cpu(), k, score, None if bias is None else bias.cpu(), groups, top_groups, best, renorm, scale,
                        dw.cpu(), *aux, daux=daux if a is not None else 0.0)
    assert torch.equal(idx.cpu().long(), want["idx"])
    assert torch.equal(counts.cpu().long(), want["counts"]) and w.dtype == torch.float32 and idx.dtype == torch.int32
    span = float(logits.float().abs().max()) + 1.0
    E = logits.shape[1]
    rel = U32 * (40 + 8 * span)                              # exponentials of sums that are off by a unit of their size, sums 35 deep
    assert within(w.detach().cpu(), want["weights"], rel * want["weights"].abs()) <= 0
    if a is not None:
        assert abs(float(a.detach()) - float(want["aux"])) <= (rel + 2e-6) * float(want["aux"]) + 1e-12
    size = abs(scale) * dw.cpu().double().abs().amax(1, keepdim=True)
    s = torch.softmax(logits.cpu().double(), 1)
    if score == "sigmoid":
        s = torch.sigmoid(logits.cpu().double())
    low = (want["weights"].abs() / max(abs(scale), 1e-30)).new_zeros(s.shape).scatter_(1, want["idx"], want["weights"].abs().double() / max(abs(scale), 1e-30))
    per = 4 * rel * (low + s * (0.0 if renorm else 1.0)) * size * (1 + k)
    # the oracle's own arithmetic: where the exact value is 0 (sum of s ds of renormalised weights) it leaves a sum of at most
    # E terms s (d - sum d w) / total, each rounded to 2^-53, times s
    per = per + 2.0 ** -52 * E * s * size / s.gather(1, want["idx"]).sum(1, keepdim=True)
    if a is not None:
        n = logits.shape[0]
        lse = torch.logsumexp(logits.cpu().double(), 1, keepdim=True).abs()
        per = per + 8 * rel * abs(daux) * (aux[0] * E / n * (s / s.sum(1, keepdim=True) + s) + aux[1] * 2 / n * (lse + 1) * torch.softmax(logits.cpu().double(), 1))
    assert within(grad.cpu(), want["grad"], per) <= 0


@pytest.mark.parametrize("E,k", [(1, 1), (3, 2), (8, 2), (8, 8), (9, 3), (16, 4), (20, 5), (32, 1), (60, 6), (64, 8), (65, 7), (128, 8),
                                 (130, 16), (256, 8), (256, 32), (257, 4), (384, 12), (512, 16)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_route(E, k, score, dtype):
    logits = randn(75, E, seed=71, dtype=DT[dtype])
    for bias in (None, 0.05 * randn(E, seed=72)):
        check_route(logits, k, score, bias)
        check_route(logits, k, score, bias, renorm=False, scale=2.5, aux=(0.02, 0.003))


@pytest.mark.parametrize("groups,size,top_groups,k", [(2, 4, 1, 3), (4, 5, 2, 10), (8, 32, 4, 8), (8, 8, 8, 6), (32, 2, 5, 7), (3, 1, 2, 2),
                                                     (5, 13, 3, 9), (16, 32, 7, 12)])
@pytest.mark.parametrize("best", [1, 2])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_groups(groups, size, top_groups, k, best, score):
    E = groups * size
    for dtype in (torch.float32, torch.bfloat16):
        logits = randn(53, E, seed=73, dtype=dtype)
        for bias in (None, 0.05 * randn(E, seed=74)):
            check_route(logits, k, score, bias, groups, top_groups, best, scale=0.5)


@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 129, 5000])
@pytest.mark.parametrize("E,k,groups", [(8, 2, 1), (64, 6, 1), (256, 8, 8)])
def test_route_token_counts(tokens, E, k, groups):
    bias = 0.02 * randn(E, seed=75)
    check_route(randn(tokens, E, seed=76), k, "sigmoid", bias, groups, max(1, groups // 2), aux=(0.01, 0.001))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_equal_and_nearly_equal_scores(score, groups):
    """Ties go to the lower number; scores that differ by less than fp32 holds keep their exact order."""
    E, k = 64, 6
    bias = torch.zeros(E, device="cuda")
    same = torch.zeros(20, E, device="cuda")                 # a router that starts from zero
    check_route(same, k, score, bias, groups, max(1, groups // 2))
    check_route(same, k, score, None, groups, max(1, groups // 2))
    few = (randn(40, E, seed=77) * 2).round() / 2            # many equal logits
    check_route(few, k, score, bias, groups, max(1, groups // 2))
    check_route(few, k, score, 0.25 * (randn(E, seed=78)).round(), groups, max(1, groups // 2))
    base = randn(40, 1, seed=79)
    near = base + U32 * base.abs() * 2 * torch.randint(-4, 5, (40, E), device="cuda", generator=gen(80))
    check_route(near, k, score, bias, groups, max(1, groups // 2))
    check_route(near, k, score, 1e-7 * randn(E, seed=81), groups, max(1, groups // 2))


def test_route_far_and_masked_logits():
    E, k = 32, 4
    z = randn(6, E, seed=82)
    z[0, :20] = float("-inf")                                # some experts are closed
    z[1] = float("-inf")                                     # all of them
    z[2, 2:] = torch.finfo(torch.float32).min
    z[3] = -95.0 - torch.arange(E, device="cuda") * 0.25     # sigmoids that fp32 cannot hold
    z[4, 7] = 90.0
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            x = z.clone().requires_grad_()
            w, idx, counts, aux = K().route_experts(x, k, score=score, renormalise=renorm, aux_coef=0.01, z_coef=0.001)
            (g,) = torch.autograd.grad((w.sum(), aux), x, (torch.tensor(1.0, device="cuda"), torch.tensor(1.0, device="cuda")))
            assert bool(torch.isfinite(w).all()) and bool(torch.isfinite(g).all()) and bool(torch.isfinite(aux))
            assert idx.max() < E and idx.min() >= 0 and int(counts.sum()) == 6 * k
            assert not w[1].any() and idx[1].tolist() == list(range(k)) and not g[1].any()
            if renorm:
                assert torch.allclose(w[3].sum(), torch.ones((), device="cuda"))
                want = torch.softmax(torch.nn.functional.logsigmoid(z[3].double()) if score == "sigmoid" else z[3].double(), 0)[:k]
                assert torch.allclose(w[3].double(), want / want.sum(), rtol=1e-5)
    z[5, 3] = float("nan")
    w, idx, counts, _ = K().route_experts(z, k, bias=torch.zeros(E, device="cuda"))
    assert idx.max() < E and idx.min() >= 0 and int(counts.sum()) == 6 * k
    banned = torch.zeros(E, device="cuda")
    banned[5:] = float("-inf")                               # a bias that closes experts
    _, idx, _, _ = K().route_experts(randn(50, E, seed=83), k, score="sigmoid", bias=banned)
    assert int(idx.max()) < 5


def test_route_strides_and_no_tokens():
    wide = randn(30, 72, seed=84, dtype=torch.bfloat16)
    for z in (wide[:, :64], wide[:, 3:67], wide[::2, 8:72]):
        check_route(z, 5, "sigmoid", 0.01 * randn(64, seed=85))
    z = torch.empty(0, 16, device="cuda", requires_grad=True)
    w, idx, counts, aux = K().route_experts(z, 3, aux_coef=0.1)
    assert w.shape == (0, 3) and idx.shape == (0, 3) and not counts.any() and float(aux.detach()) == 0.0
    assert torch.autograd.grad(w.sum(), z)[0].shape == (0, 16)


def test_route_only_aux_has_a_gradient():
    z = randn(40, 24, seed=86).requires_grad_()
    _, _, _, aux = K().route_experts(z, 3, score="sigmoid", aux_coef=0.1, z_coef=0.01)
    (g,) = torch.autograd.grad(aux, z)
    want = oracle.route(z.detach().cpu(), 3, "sigmoid", None, 1, 1, 2, True, 1.0, torch.zeros(40, 3), 0.1, 0.01, 1.0)
    assert within(g.cpu(), want["grad"], 1e-5 * want["grad"].abs().amax()) <= 0
