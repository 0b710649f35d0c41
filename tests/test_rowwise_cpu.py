"""LayerNorm, rotary positions, top-logit distillation and expert routing on the CPU: the PyTorch statements against the
definitions in 64 bits, gradients against differences, and the calls that are refused."""
import math

import pytest
import torch
import torch.nn.functional as F

import forgeminds_b200 as fm
import rowwise_oracle as oracle
from rowwise_oracle import U32, within

K = fm.kernels


def _randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ------------------------------------------------------------------------------ LayerNorm
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("d", [1, 7, 64])
def test_layer_norm(dtype, d):
    x, w, b = _randn(5, d, seed=1, dtype=dtype), 1 + 0.2 * _randn(d, seed=2), 0.1 * _randn(d, seed=3)
    want, off = oracle.layer_norm(x, w, b, 1e-5)
    y = K.layer_norm(x, w, b)
    assert y.dtype == dtype and within(y, want["y"], off["y"]) <= 0
    total, y = K.add_layer_norm(x, x, w, b)
    assert torch.equal(total, x + x)
    want, off = oracle.layer_norm(total, w, b, 1e-5)
    assert within(y, want["y"], off["y"]) <= 0


def test_layer_norm_gradients_are_the_differences():
    x, w, b = (_randn(*s, seed=i, dtype=torch.float64).requires_grad_() for i, s in enumerate([(2, 3, 6), (6,), (6,)]))
    assert torch.autograd.gradcheck(K.layer_norm, (x, w, b))
    assert torch.autograd.gradcheck(lambda *a: K.add_layer_norm(a[0], a[0] * 2, *a[1:]), (x, w, b))
    assert torch.autograd.gradcheck(lambda t: K.layer_norm(t), (x,))
    want, _ = oracle.layer_norm(x.detach().reshape(-1, 6), w.detach(), b.detach(), 1e-5, torch.ones(6, 6))
    got = torch.autograd.grad(K.layer_norm(x, w, b).sum(), (x, w, b))
    assert torch.allclose(got[0].reshape(-1, 6), want["dx"]) and torch.allclose(got[1], want["dw"]) and torch.allclose(got[2], want["db"])


def test_layer_norm_refuses():
    x = _randn(4, 8)
    for call in (lambda: K.layer_norm(x, torch.ones(7)), lambda: K.layer_norm(x, torch.ones(8), torch.ones(2, 4)),
                 lambda: K.layer_norm(torch.ones(4, 8, dtype=torch.int64)), lambda: K.layer_norm(torch.ones(())),
                 lambda: K.layer_norm(torch.ones(3, 0)), lambda: K.add_layer_norm(x, x[:2]),
                 lambda: K.add_layer_norm(x, x.double()), lambda: K.layer_norm(x, torch.ones(8, device="meta"))):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------------------ rotary positions
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("R", [2, 6, 10])
def test_rotary(interleaved, R):
    q, k = _randn(2, 5, 3, 10, seed=4), _randn(2, 5, 1, 10, seed=5)
    cos, sin = K.rotary_tables(9, R)
    for pos in (None, torch.tensor([8, 0, 3, 3, 1]), torch.tensor([[8, 0, 3, 3, 1], [-1, 9, 10 ** 12, -5, 2]]), torch.tensor([[1, 2, 3, 4, 5]], dtype=torch.int32)):
        a, b = K.rotary_qk(q, k, cos, sin, pos, interleaved)
        for got, x in ((a, q), (b, k)):
            want, off = oracle.rotary(x, cos, sin, pos, interleaved)
            assert within(got, want, off) <= 0
        assert torch.equal(K.rotary(q, cos[None, :, None], sin[None, :, None], pos, interleaved).nan_to_num(9.0), a.nan_to_num(9.0))


def test_rotary_gradients_are_the_differences():
    q, k = _randn(2, 3, 2, 8, seed=6, dtype=torch.float64).requires_grad_(), _randn(2, 3, 1, 8, seed=7, dtype=torch.float64).requires_grad_()
    cos, sin = (t.double() for t in K.rotary_tables(7, 4))
    for interleaved in (False, True):
        assert torch.autograd.gradcheck(lambda a, b: K.rotary_qk(a, b, cos, sin, torch.tensor([6, 0, 2]), interleaved), (q, k))


def test_rotary_layouts_are_permutations_of_each_other():
    x = _randn(1, 6, 2, 8, seed=8)
    cos, sin = K.rotary_tables(6, 8)
    pairs = torch.tensor([0, 4, 1, 5, 2, 6, 3, 7])
    assert torch.equal(K.rotary(x, cos, sin)[..., pairs], K.rotary(x[..., pairs], cos, sin, interleaved=True))


def test_rotary_tables():
    n, d = 300, 16
    i = torch.arange(0, d, 2, dtype=torch.float64)
    freq, at = 10000.0 ** (-i / d), torch.arange(n, dtype=torch.float64)[:, None]

    def same(got, freq, gain=1.0):
        c, s = got
        assert c.dtype == torch.float32 and c.shape == (n, d // 2)
        assert within(c, gain * (at * freq).cos(), 1e-12) <= 0 and within(s, gain * (at * freq).sin(), 1e-12) <= 0

    same(K.rotary_tables(n, d), freq)
    same(K.rotary_tables(n, d, scaling="linear", factor=8.0), freq / 8)
    ntk = (10000.0 * 8.0 ** (d / (d - 2))) ** (-i / d)
    same(K.rotary_tables(n, d, scaling="ntk", factor=8.0), ntk)
    assert math.isclose(float(ntk[0]), 1.0) and math.isclose(float(ntk[-1]), float(freq[-1]) / 8)
    turns = 2048 * freq / (2 * math.pi)
    keep = ((turns - 1) / 31).clamp(0, 1)
    same(K.rotary_tables(n, d, scaling="yarn", factor=8.0, trained=2048), freq * keep + freq / 8 * (1 - keep), 0.1 * math.log(8) + 1)
    same(K.rotary_tables(n, d, scaling="yarn", factor=8.0, trained=2048, attention_factor=1.0), freq * keep + freq / 8 * (1 - keep))
    from forgeminds_b200.models.gpt import rope_tables
    c, s = rope_tables(n, d, 10000.0, "cpu", torch.float32)
    assert torch.allclose(c[0, :, 0], K.rotary_tables(n, d)[0], atol=3e-5)      # the model's own table takes its angles in fp32
    for bad in (dict(n=0, dim=4), dict(n=4, dim=3), dict(n=4, dim=0), dict(n=4, dim=4, theta=0.0), dict(n=4, dim=4, factor=0.5),
                dict(n=4, dim=4, scaling="cubic"), dict(n=4, dim=4, scaling="yarn"),
                dict(n=4, dim=4, scaling="yarn", trained=8, fast_turns=1.0)):
        with pytest.raises(ValueError):
            K.rotary_tables(**bad)


def test_rotary_refuses():
    q, k = _randn(2, 5, 3, 8), _randn(2, 5, 1, 8)
    cos, sin = K.rotary_tables(5, 8)
    wide = K.rotary_tables(5, 10)
    for call in (lambda: K.rotary(q[0], cos, sin), lambda: K.rotary_qk(q, k[:, :4], cos, sin), lambda: K.rotary_qk(q, k.double(), cos, sin),
                 lambda: K.rotary_qk(q, k[..., :6], cos, sin), lambda: K.rotary(q, *wide), lambda: K.rotary(q, cos, sin[:4]),
                 lambda: K.rotary(q, cos[:4], sin[:4]), lambda: K.rotary(q, cos, sin, torch.zeros(5)),
                 lambda: K.rotary(q, cos, sin, torch.zeros(4, dtype=torch.int64)), lambda: K.rotary(q, cos, sin, torch.zeros(5, 2, dtype=torch.int64)),
                 lambda: K.rotary(q.long(), cos, sin), lambda: K.rotary(q, cos[:0], sin[:0], torch.zeros(5, dtype=torch.int64)),
                 lambda: K.rotary(q, cos.requires_grad_(), sin)):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------------------ distillation from top logits
def _kl_inputs(rows, V, keep, seed):
    teacher = 2 * _randn(rows, V, seed=seed)
    values, index = teacher.topk(keep, dim=-1)
    return teacher + _randn(rows, V, seed=seed + 1), values, index, teacher


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("tau", [1.0, 2.5])
def test_kl_topk(reduction, tau):
    student, values, index, teacher = _kl_inputs(7, 40, 6, 10)
    index[2] = -1
    index[3, 4:] = -1
    index[4, 1] = 40
    values[5, 0] = float("-inf")
    index[6, 1] = index[6, 0]
    for lse in (None, torch.logsumexp(teacher / tau, -1)):
        s = student.clone().requires_grad_()
        loss = K.kl_topk_logits(s, values, index, temperature=tau, reduction=reduction, teacher_lse=lse)
        (g,) = torch.autograd.grad(loss.sum(), s)
        want, grad, off, goff = oracle.kl_topk(student, values, index, tau, lse, reduction)
        assert within(loss.detach(), want, off) <= 0 and within(g, grad, goff) <= 0 and not g[2].any()


def test_kl_topk_with_everything_kept_is_the_full_divergence():
    student, values, index, teacher = _kl_inputs(6, 20, 20, 12)
    want = K.kl_div_logits(student, teacher)
    assert torch.allclose(K.kl_topk_logits(student, values, index), want, atol=1e-6)
    assert torch.allclose(K.kl_topk_logits(student, values, index.int(), teacher_lse=teacher.logsumexp(-1)), want, atol=1e-6)


def test_kl_topk_gradients_are_the_differences():
    student, values, index, _ = _kl_inputs(3, 12, 4, 14)
    s = student.double().requires_grad_()
    index[1] = -1
    for reduction in ("mean", "none"):
        assert torch.autograd.gradcheck(lambda t: K.kl_topk_logits(t, values, index, temperature=1.5, reduction=reduction), (s,))


def test_kl_topk_distill_loss():
    h, w = _randn(10, 6, seed=16).requires_grad_(), _randn(30, 6, seed=17).requires_grad_()
    values, index = _randn(10, 30, seed=18).topk(5, dim=-1)
    index[4] = -1
    want = K.kl_topk_logits(h @ w.t(), values, index, temperature=2.0)
    for chunk in (3, 100):
        loss = K.kl_topk_distill_loss(h.view(2, 5, 6), w, values.view(2, 5, 5), index.view(2, 5, 5), temperature=2.0, chunk=chunk)
        assert torch.allclose(loss, want, atol=1e-6)
        for a, b in zip(torch.autograd.grad(loss, (h, w)), torch.autograd.grad(want, (h, w), retain_graph=True)):
            assert torch.allclose(a, b, atol=1e-6)
    none = K.kl_topk_distill_loss(h[:0], w, values[:0], index[:0])
    assert float(none.detach()) == 0.0 and torch.autograd.grad(none, h)[0].shape == h.shape


def test_kl_topk_refuses():
    student, values, index, teacher = _kl_inputs(4, 10, 3, 19)
    for call in (lambda: K.kl_topk_logits(student, values, index, reduction="batchmean"), lambda: K.kl_topk_logits(student, values, index, temperature=0.0),
                 lambda: K.kl_topk_logits(student, values, index, temperature=float("inf")), lambda: K.kl_topk_logits(student, values[:2], index),
                 lambda: K.kl_topk_logits(student, values[:2], index[:2]), lambda: K.kl_topk_logits(student, values, index.float()),
                 lambda: K.kl_topk_logits(student, values.long(), index), lambda: K.kl_topk_logits(student.long(), values, index),
                 lambda: K.kl_topk_logits(student, values[:, :0], index[:, :0]), lambda: K.kl_topk_logits(student[:, :0], values, index),
                 lambda: K.kl_topk_logits(student, values, index, teacher_lse=torch.zeros(3)),
                 lambda: K.kl_topk_distill_loss(student, torch.ones(5, 9), values, index),
                 lambda: K.kl_topk_distill_loss(student, torch.ones(5, 10), values, index, chunk=0)):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------------------ routing to experts
ROUTES = [dict(), dict(score="sigmoid"), dict(bias=True), dict(score="sigmoid", bias=True, n_groups=3, top_groups=2),
          dict(n_groups=3, top_groups=1, group_best=1), dict(score="sigmoid", renormalise=False, scale=2.0),
          dict(renormalise=False, aux_coef=0.1, z_coef=0.01), dict(score="sigmoid", bias=True, aux_coef=0.1, z_coef=0.01)]


@pytest.mark.parametrize("opts", ROUTES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
def test_route(opts, dtype):
    opts = dict(opts)
    E, k = 12, 4
    logits = _randn(9, E, seed=20, dtype=dtype).requires_grad_()
    bias = 0.1 * _randn(E, seed=21) if opts.pop("bias", False) else None
    w, idx, counts, aux = K.route_experts(logits, k, bias=bias, **opts)
    dw = _randn(9, k, seed=22).to(w.dtype)
    outs, ups = ([w], [dw]) if aux is None else ([w, aux], [dw, torch.ones_like(aux)])
    (grad,) = torch.autograd.grad(outs, logits, ups)
    want = oracle.route(logits.detach(), k, opts.get("score", "softmax"), bias, opts.get("n_groups", 1), opts.get("top_groups", 1),
                        opts.get("group_best", 2), opts.get("renormalise", True), opts.get("scale", 1.0), dw, opts.get("aux_coef", 0.0),
                        opts.get("z_coef", 0.0), 1.0)
    assert torch.equal(idx.long(), want["idx"]) and torch.equal(counts.long(), want["counts"]) and idx.dtype == torch.int32
    assert within(w.detach(), want["weights"], 64 * U32 * want["weights"]) <= 0
    assert aux is None or abs(float(aux.detach()) - float(want["aux"])) <= 64 * U32 * float(want["aux"])
    assert within(grad, want["grad"], 64 * U32 * (1 + want["grad"].abs())) <= 0


def test_route_gradients_are_the_differences():
    z = _randn(4, 8, seed=23, dtype=torch.float64).requires_grad_()
    for opts in (dict(), dict(score="sigmoid"), dict(renormalise=False), dict(score="sigmoid", renormalise=False)):
        assert torch.autograd.gradcheck(lambda t: K.route_experts(t, 3, **opts)[0], (z,))
        assert torch.autograd.gradcheck(lambda t: K.route_experts(t, 3, aux_coef=0.5, z_coef=0.1, **opts)[3], (z,))


def test_route_rows_with_nothing():
    z = _randn(3, 8, seed=24)
    z[1] = float("-inf")
    z.requires_grad_()
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            w, idx, counts, aux = K.route_experts(z, 3, score=score, renormalise=renorm, aux_coef=0.1, z_coef=0.1)
            (g,) = torch.autograd.grad(w.sum() + aux, z)
            assert not w[1].any() and idx[1].tolist() == [0, 1, 2] and bool(torch.isfinite(g).all()) and bool(torch.isfinite(aux))
    w, idx, counts, aux = K.route_experts(z[:0], 3, aux_coef=0.1)
    assert w.shape == (0, 3) and not counts.any() and float(aux.detach()) == 0.0


def test_route_refuses():
    z = _randn(4, 8)
    for opts in (dict(k=0), dict(k=9), dict(k=2, score="tanh"), dict(k=2, n_groups=3), dict(k=2, n_groups=0), dict(k=2, n_groups=4, top_groups=0),
                 dict(k=2, n_groups=4, top_groups=5), dict(k=5, n_groups=4, top_groups=2), dict(k=2, group_best=3), dict(k=2, bias=torch.zeros(7)),
                 dict(k=2, bias=torch.zeros(8, dtype=torch.int64)), dict(k=2, bias=torch.zeros(8, device="meta"))):
        with pytest.raises(ValueError):
            K.route_experts(z, **opts)
    for bad in (z[0], z.long(), z[:, :0]):
        with pytest.raises(ValueError):
            K.route_experts(bad, 1)


# ------------------------------------------------------------------------------ modules that take them
def test_layer_norm_module():
    mine, theirs = fm.nn.LayerNorm(24), torch.nn.LayerNorm(24)
    torch.nn.init.normal_(theirs.weight)
    torch.nn.init.normal_(theirs.bias)
    mine.load_state_dict(theirs.state_dict())
    theirs.load_state_dict(mine.state_dict())
    x, r = _randn(3, 5, 24, seed=30), _randn(3, 5, 24, seed=31)
    assert torch.allclose(mine(x), theirs(x), atol=1e-6)
    y, total = mine.forward_with_residual(x, r)
    assert torch.equal(total, x + r) and torch.allclose(y, theirs(x + r), atol=1e-6)
    assert mine.forward_with_residual(x)[1] is x
    assert [n for n, _ in fm.nn.LayerNorm(8, bias=False).named_parameters()] == ["weight"]
    assert not list(fm.nn.LayerNorm(8, elementwise_affine=False).parameters())
    assert "eps=1e-05" in repr(mine) and "no bias" in repr(fm.nn.LayerNorm(8, bias=False))
    for bad in (lambda: fm.nn.LayerNorm(0), lambda: mine(x[..., :8]), lambda: mine.forward_with_residual(x, r[:1])):
        with pytest.raises(ValueError):
            bad()


def test_patching_a_layer_norm_has_to_be_asked_for():
    model = torch.nn.Sequential(torch.nn.LayerNorm(16), torch.nn.Linear(16, 16), torch.nn.LayerNorm((4, 4)))
    K.enable(model)
    assert model._fm_fused == {"norm": 0, "mlp": 0} and not K.patch(model[0])
    x = _randn(3, 16, seed=32)
    before = model[0](x)
    K.enable(model, layer_norm=True)
    assert model._fm_fused == {"norm": 0, "mlp": 0, "layer_norm": 1} and "forward" in model[0].__dict__
    assert torch.allclose(model[0](x), before, atol=1e-6)
    K.revert(model)
    assert "forward" not in model[0].__dict__
    assert K.patch(model[0], kind="layer_norm") and K.patch(model[0], kind="layer_norm")
    for m in (model[1], model[2]):
        with pytest.raises(TypeError):
            K.patch(m, kind="layer_norm")


@pytest.mark.parametrize("opts", [dict(score="sigmoid"), dict(balance_bias=True), dict(n_groups=2, top_groups=1),
                                  dict(renormalise=False), dict(score="sigmoid", balance_bias=True, n_groups=2, top_groups=2, route_scale=2.5)])
def test_moe_takes_the_routing_options(opts):
    torch.manual_seed(5)
    moe = fm.MoE(16, 32, 8, 3, **opts)
    if moe.router.bias is not None:
        assert "router.bias" in moe.state_dict()
        moe.router.bias.copy_(0.1 * _randn(8, seed=33))
    else:
        assert "router.bias" not in moe.state_dict()
    x = _randn(4, 6, 16, seed=34).requires_grad_()
    y = moe(x)
    names = dict(opts)
    names["scale"] = names.pop("route_scale", 1.0)
    names.pop("balance_bias", None)
    flat = x.reshape(-1, 16)
    w, idx, counts, aux = K.route_experts(moe.router.gate(flat), 3, bias=moe.router.bias, aux_coef=1e-2, z_coef=1e-3, **names)
    want = torch.zeros_like(flat)
    for e in range(8):
        h = (F.silu(flat @ moe.experts.w1[e]) * (flat @ moe.experts.w3[e])) @ moe.experts.w2[e]
        want = want + h * (w * (idx == e)).sum(-1, keepdim=True)
    assert torch.allclose(y.reshape(-1, 16), want, atol=1e-6) and torch.allclose(moe.last_aux, aux)
    assert torch.equal(moe.router.last_counts, counts)
    for a, b in zip(torch.autograd.grad(y.sum() + moe.last_aux, (x, moe.router.gate.weight)),
                    torch.autograd.grad(want.sum() + aux, (x, moe.router.gate.weight))):
        assert torch.allclose(a, b, atol=1e-5)


def test_moe_balance():
    torch.manual_seed(6)
    moe = fm.MoE(16, 32, 4, 1, score="sigmoid", balance_bias=True, aux_coef=0.0, z_coef=0.0)
    with pytest.raises(RuntimeError):
        moe.router.rebalance(0.1)                            # no forward pass yet
    with torch.no_grad():
        moe.router.gate.weight[2] += 0.5                     # a favourite
    x = _randn(200, 16, seed=35).abs()
    moe(x)
    assert float(moe.last_aux) == 0.0 and moe.router.last_counts.argmax() == 2
    first = moe.router.last_counts.clone()
    for _ in range(40):
        moe.router.rebalance(0.02)
        moe(x)
    assert moe.router.last_counts.max() < first.max() and moe.router.bias[2] < 0
    with pytest.raises(RuntimeError):
        fm.MoE(16, 32, 4, 1).router.rebalance(0.1)
    for bad in (dict(score="tanh"), dict(n_groups=3), dict(n_groups=2, top_groups=3), dict(n_groups=4, top_groups=1, score="sigmoid")):
        with pytest.raises(ValueError):
            fm.MoE(16, 32, 4, 2, **bad)


def test_moe_defaults_route_as_before():
    torch.manual_seed(7)
    moe = fm.MoE(16, 32, 4, 2)
    assert moe.router.plain and set(moe.state_dict()) == {"router.gate.weight", "experts.w1", "experts.w3", "experts.w2"}
    x = _randn(9, 16, seed=36)
    w, idx, aux, z = moe.router(x)
    probs = moe.router.gate(x).softmax(-1)
    v, i = probs.topk(2, dim=-1)
    assert torch.equal(idx, i) and torch.allclose(w, v / v.sum(-1, keepdim=True))


def test_rotary_leaves_negative_positions_as_they_are():
    x = _randn(1, 3, 2, 8)
    x[0, 1, 0, 2] = float("inf")
    x.requires_grad_()
    cos, sin = K.rotary_tables(4, 6)
    for interleaved in (False, True):
        y = K.rotary(x, cos, sin, torch.tensor([2, -1, 0]), interleaved)
        assert torch.equal(y[:, 1], x[:, 1])
        (g,) = torch.autograd.grad(y[:, 1].sum(), x)
        assert torch.equal(g[:, 1], torch.ones_like(g[:, 1])) and not g[:, ::2].any()


def test_the_balance_bias_stays_in_fp32():
    moe = fm.MoE(16, 32, 8, 2, balance_bias=True)
    moe.router.bias += 0.501
    before = moe.router.bias.clone()
    moe.to(torch.bfloat16)
    assert moe.router.bias.dtype == torch.float32 and torch.equal(moe.router.bias, before)
    assert moe.router.gate.weight.dtype == torch.bfloat16 and "router.bias" in moe.state_dict()
    moe.double()
    assert moe.router.bias.dtype == torch.float32 and moe.router.gate.weight.dtype == torch.float64
    meta = fm.MoE(16, 32, 8, 2, balance_bias=True).to("meta").to_empty(device="cpu")
    assert meta.router.bias.shape == (8,) and meta.router.bias.dtype == torch.float32
    assert fm.MoE(16, 32, 8, 2).to(torch.bfloat16).router.bias is None
