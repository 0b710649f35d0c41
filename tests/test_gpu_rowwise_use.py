"""LayerNorm, rotary positions, expert routing and top-logit distillation as programs use them: a student's training step,
captured graphs, several streams, calls on one graph twice."""
import pytest
import torch
import torch.nn.functional as F

import forgeminds_b200 as fm
import rowwise_oracle as oracle

pytestmark = pytest.mark.gpu
K = fm.kernels


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, device="cuda", generator=gen(seed)) * scale).to(dtype)


# ------------------------------------------------------------------------------ a student against stored teacher logits
class Student(torch.nn.Module):
    """Pre-norm blocks with LayerNorm, interleaved rotary positions on half of each head and routed experts."""

    def __init__(self, vocab=211, dim=64, heads=4, kv=2, layers=2):
        super().__init__()
        self.hd, self.heads, self.kv = dim // heads, heads, kv
        self.emb = torch.nn.Embedding(vocab, dim)
        self.blocks = torch.nn.ModuleList()
        for _ in range(layers):
            self.blocks.append(torch.nn.ModuleDict(dict(
                n1=fm.nn.LayerNorm(dim), n2=fm.nn.LayerNorm(dim), qkv=torch.nn.Linear(dim, (heads + 2 * kv) * self.hd, bias=False),
                out=torch.nn.Linear(dim, dim, bias=False),
                moe=fm.MoE(dim, 2 * dim, 12, 3, score="sigmoid", balance_bias=True, n_groups=4, top_groups=2, route_scale=1.5))))
        self.norm, self.head = fm.nn.LayerNorm(dim, bias=False), torch.nn.Linear(dim, vocab, bias=False)

    def forward(self, tokens, positions, cos, sin):
        B, T = tokens.shape
        x, delta, aux = self.emb(tokens), None, 0.0
        for b in self.blocks:
            h, x = b["n1"].forward_with_residual(x, delta)
            qkv = b["qkv"](h).view(B, T, -1, self.hd)
            q, k = K.rotary_qk(qkv[:, :, : self.heads], qkv[:, :, self.heads: self.heads + self.kv], cos, sin, positions, True)
            v = qkv[:, :, self.heads + self.kv:]
            o = F.scaled_dot_product_attention(*(t.transpose(1, 2) for t in (q, k, v)), is_causal=True, enable_gqa=True)
            h, x = b["n2"].forward_with_residual(x, b["out"](o.transpose(1, 2).reshape(B, T, -1)))
            delta = b["moe"](h)
            aux = aux + b["moe"].last_aux
        return self.norm.forward_with_residual(x, delta)[0], aux


def _step(student, tokens, positions, cos, sin, values, index):
    h, aux = student(tokens, positions, cos, sin)
    loss = K.kl_topk_distill_loss(h, student.head.weight, values, index, temperature=2.0, chunk=50) + aux
    names = [n for n, p in student.named_parameters() if p.requires_grad]
    grads = torch.autograd.grad(loss, [p for p in student.parameters()])
    return loss.detach(), dict(zip(names, grads))


def test_a_training_step_agrees_with_its_pytorch_statements():
    """fp32: the same step through the kernels and through the PyTorch statements (in fp64, so that these say what is
    right). The router's choices agree because both are exact for scores that differ by far more than 2^-24."""
    torch.backends.cuda.matmul.allow_tf32, before = False, torch.backends.cuda.matmul.allow_tf32
    try:
        torch.manual_seed(3)
        student = Student().cuda()
        B, T = 3, 41
        tokens = torch.randint(0, 211, (B, T), device="cuda", generator=gen(1))
        positions = torch.stack([torch.arange(T), torch.arange(T) + 500, torch.arange(T) % 17]).cuda()
        cos, sin = K.rotary_tables(600, 8, scaling="yarn", factor=4.0, trained=128, device="cuda")
        values, index = (randn(B, T, 211, seed=2) * 2).topk(6, dim=-1)
        index = index.clone()
        index[2, 30:] = -1                                   # a padded sequence
        K.reset_stats()
        loss, grads = _step(student, tokens, positions, cos, sin, values, index)
        st = K.stats()
        # per step: 5 norms, 2 rotations, 2 choices and the chunks' loss call the dispatcher, all on the kernels
        assert st["fast"] >= 10 and st["fallback"] == 0, st
        counts = [b["moe"].router.last_counts.clone() for b in student.blocks]
        assert all(int(c.sum()) == B * T * 3 for c in counts)
        K.set_backend("fallback")
        want_loss, want = _step(student.double(), tokens, positions, cos.double(), sin.double(), values.double(), index)
        for b, c in zip(student.blocks, counts):
            assert torch.equal(b["moe"].router.last_counts, c)
        # a hundred operations deep, sums of up to 211 terms: relative errors of a few hundred units of 2^-24 in norm
        assert abs(float(loss) - float(want_loss)) <= 1000 * 2.0 ** -24 * float(want_loss)
        for name, g in grads.items():
            assert float((g - want[name]).norm()) <= 4000 * 2.0 ** -24 * float(want[name].norm()) + 1e-9, name
    finally:
        K.set_backend("auto")
        torch.backends.cuda.matmul.allow_tf32 = before


def test_moe_with_routing_options_on_the_grouped_products():
    torch.manual_seed(4)
    moe = fm.MoE(256, 512, 8, 2, grouped_mm=True, score="sigmoid", balance_bias=True, n_groups=4, top_groups=2, route_scale=2.0).cuda()
    moe.router.bias.copy_(0.05 * torch.randn(8))
    x = randn(3, 100, 256, seed=5, dtype=torch.bfloat16).requires_grad_()
    dy = randn(3, 100, 256, seed=6, dtype=torch.bfloat16)
    y = moe(x)
    grads = torch.autograd.grad(y, [x, moe.router.gate.weight, moe.experts.w1, moe.experts.w2], dy)
    # the same choice in fp32 on the bf16 gate logits that the layer routes by
    flat = x.detach().reshape(-1, 256)
    xf = flat.float().requires_grad_()
    gate = moe.router.gate.weight.detach().float().requires_grad_()
    w1, w3, w2 = (p.detach().to(torch.bfloat16).float().requires_grad_() for p in (moe.experts.w1, moe.experts.w3, moe.experts.w2))
    from forgeminds_b200.ops.functional import linear
    logits = xf @ gate.to(torch.bfloat16).float().t()
    seen = linear(flat, moe.router.gate.weight).detach().float()
    logits = logits + (seen - logits).detach()
    w, idx, counts, _ = K.route_experts(logits, 2, score="sigmoid", bias=moe.router.bias, n_groups=4, top_groups=2, scale=2.0)
    assert torch.equal(counts, moe.router.last_counts)
    out = torch.zeros_like(xf)
    for e in range(8):
        h = (F.silu(xf @ w1[e]) * (xf @ w3[e])) @ w2[e]
        out = out + h * (w * (idx == e)).sum(-1, keepdim=True)
    want = torch.autograd.grad(out, [xf, gate, w1, w2], dy.reshape(-1, 256).float())
    # activations, gradients and products are each rounded to bf16 (2^-8) some eight times on the way
    assert float((y.reshape(-1, 256).float() - out).detach().norm()) <= 8 * 2.0 ** -8 * float(out.detach().norm())
    for name, g, t in zip(("x", "gate", "w1", "w2"), grads, want):
        assert float((g.reshape(t.shape).float() - t).norm()) <= 12 * 2.0 ** -8 * float(t.norm()), name
    before = moe.router.bias.clone()
    moe.router.rebalance(0.01)
    load = counts.float()
    assert torch.allclose(moe.router.bias - before, 0.01 * torch.sign(load.mean() - load), atol=1e-7)


# ------------------------------------------------------------------------------ one call of each operator, with gradients
def _ln(seed):
    x, w, b = (t.requires_grad_() for t in (randn(70, 520, seed=seed, dtype=torch.bfloat16), 1 + randn(520, seed=seed + 1, scale=0.1), randn(520, seed=seed + 2)))
    dy = randn(70, 520, seed=seed + 3, dtype=torch.bfloat16)
    return [x, w, b, dy], lambda x, w, b, dy: _with_grads(K.layer_norm(x, w, b), [x, w, b], dy)


def _rotary(seed):
    q, k = (randn(3, 9, h, 64, seed=seed + h, dtype=torch.bfloat16).requires_grad_() for h in (4, 2))
    cos, sin = K.rotary_tables(64, 32, device="cuda")
    pos = torch.randint(0, 64, (3, 9), device="cuda", generator=gen(seed))
    gq, gk = torch.randn_like(q).detach(), torch.randn_like(k).detach()

    def run(q, k, pos, gq, gk):
        a, b = K.rotary_qk(q, k, cos, sin, pos)
        return [a.detach(), b.detach(), *torch.autograd.grad((a, b), (q, k), (gq, gk))]
    return [q, k, pos, gq, gk], run


def _kl(seed, V=4001, rows=40):
    s = randn(rows, V, seed=seed, dtype=torch.bfloat16).requires_grad_()
    v, i = randn(rows, V, seed=seed + 1).topk(11, dim=-1)
    up = torch.tensor(0.25 + seed % 3, device="cuda")
    return [s, v, i, up], lambda s, v, i, up: _with_grads(K.kl_topk_logits(s, v, i, temperature=1.5), [s], up)


def _kl_wide(seed):
    return _kl(seed, 90001, 20)


def _route(seed):
    z, bias, dw = randn(130, 64, seed=seed).requires_grad_(), randn(64, seed=seed + 1, scale=0.05), randn(130, 6, seed=seed + 2)

    def run(z, bias, dw):
        w, idx, counts, aux = K.route_experts(z, 6, score="sigmoid", bias=bias, n_groups=8, top_groups=3, aux_coef=0.1, z_coef=0.01)
        return [w.detach(), idx, counts, aux.detach(), *torch.autograd.grad((w, aux), (z,), (dw, torch.ones_like(aux)))]
    return [z, bias, dw], run


def _with_grads(out, leaves, up):
    return [out.detach(), *torch.autograd.grad(out, leaves, up)]


CALLS = [_ln, _rotary, _kl, _kl_wide, _route]


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b)) and len(a) == len(b)


@pytest.mark.parametrize("make", CALLS)
def test_captured_and_replayed_with_other_inputs(make):
    """Forward and backward in one graph: a replay on new contents of the inputs gives what an eager call gives."""
    first, run = make(100)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(*first)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*first)
    for seed in (100, 200, 300):
        other, _ = make(seed)
        with torch.no_grad():
            for a, b in zip(first, other):
                a.copy_(b)
        graph.replay()
        got = [t.clone() for t in out]
        assert _same(got, run(*other)), seed
        graph.replay()                                       # and again on the same ones
        assert _same(got, out)


@pytest.mark.parametrize("make", CALLS)
def test_two_captured_graphs_share_nothing(make):
    (a, run), (b, _) = make(400), make(500)
    run(*a)
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g, x in zip(graphs, (a, b)):
        with torch.cuda.graph(g):
            outs.append(run(*x))
    want = [run(*a), run(*b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):                                       # both at once
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert _same(outs[0], want[0]) and _same(outs[1], want[1])


@pytest.mark.parametrize("make", CALLS)
def test_on_other_streams_at_once(make):
    inputs = [make(600 + 10 * i) for i in range(4)]
    want = [run(*x) for x, run in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    for _ in range(3):
        got = []
        for s, (x, run) in zip(streams, inputs):
            with torch.cuda.stream(s):
                got.append(run(*x))
        torch.cuda.synchronize()
        assert all(_same(g, w) for g, w in zip(got, want))


def test_kl_backward_captured_alone_can_be_replayed_with_another_upstream_gradient():
    """The forward pass ran eagerly and left a gradient; a captured backward pass must not hand that tensor out."""
    (other, v, i, _), _ = _kl(700)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):                             # a leaf of its own: its gradient's place belongs to this stream
        s = other.detach().clone().requires_grad_()
        loss = K.kl_topk_logits(s, v, i, temperature=1.5)
        up = torch.tensor(0.5, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        (grad,) = torch.autograd.grad(loss, s, up, retain_graph=True)
    for value in (0.5, 2.0, 1.0, 0.5):
        up.fill_(value)
        torch.cuda.synchronize()
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        _, want, _, off = oracle.kl_topk(other.detach(), v, i, 1.5, upstream=value)
        assert oracle.within(grad, want, off) <= 0
        if value != 1.0:                                      # for 1 the forward pass's own gradient: another kernel's roundings
            (eager,) = torch.autograd.grad(K.kl_topk_logits(other, v, i, temperature=1.5), other, torch.tensor(value, device="cuda"))
            assert torch.equal(grad, eager)


@pytest.mark.parametrize("make", CALLS)
def test_a_second_derivative_is_refused(make):
    """Gradients of gradients would be wrong if they were taken for constants: asking for one raises."""
    inputs, _ = make(800)
    leaf = inputs[0]
    out = {_ln: lambda: K.layer_norm(*inputs[:3]), _rotary: lambda: K.rotary(leaf, *K.rotary_tables(64, 32, device="cuda")),
           _kl: lambda: K.kl_topk_logits(*inputs[:3]), _kl_wide: lambda: K.kl_topk_logits(*inputs[:3]),
           _route: lambda: K.route_experts(leaf, 6)[0]}[make]()
    (g,) = torch.autograd.grad(out.float().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        g.float().square().sum().backward()


def test_changing_an_input_before_the_backward_pass_is_noticed():
    for make in (_ln, _kl, _route):
        inputs, _ = make(900)
        leaf = inputs[0].detach().clone().requires_grad_()
        x = leaf * 1
        out = {_ln: lambda: K.layer_norm(x), _kl: lambda: K.kl_topk_logits(x, inputs[1], inputs[2]),
               _route: lambda: K.route_experts(x, 6)[0].square().sum()}[make]()
        x.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.float().sum().backward()


def test_without_gradients_nothing_is_kept():
    x = randn(256, 4096, seed=910, dtype=torch.bfloat16).requires_grad_()
    v, i = randn(256, 4096, seed=911).topk(4, dim=-1)
    with torch.no_grad():
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        loss = K.kl_topk_logits(x, v, i)
        assert not loss.requires_grad and torch.cuda.memory_allocated() - before <= 4096
        assert not K.layer_norm(x).requires_grad and not K.route_experts(x[:, :64], 2)[0].requires_grad
    with torch.inference_mode():
        y = K.layer_norm(randn(5, 64, seed=912))
        assert y.shape == (5, 64)


def test_other_types_take_the_pytorch_statements():
    K.reset_stats()
    x = randn(6, 32, seed=913, dtype=torch.float16).requires_grad_()
    y = K.layer_norm(x, torch.ones(32, device="cuda", dtype=torch.float16))
    assert y.dtype == torch.float16 and torch.autograd.grad(y.sum(), x)[0].dtype == torch.float16
    q = randn(2, 3, 4, 16, seed=914, dtype=torch.float64)
    cos, sin = K.rotary_tables(3, 16, device="cuda")
    assert K.rotary(q, cos, sin).dtype == torch.float64
    w, idx, counts, _ = K.route_experts(randn(4, 600, seed=915), 3)      # more experts than the kernel holds
    assert idx.shape == (4, 3) and int(counts.sum()) == 12
    v, i = randn(3, 5000, seed=916).topk(1100, dim=-1)                   # more kept logits
    assert bool(torch.isfinite(K.kl_topk_logits(randn(3, 5000, seed=917), v, i)))
    st = K.stats()
    assert st["fast"] == 0 and st["fallback"] == 2, st                   # limits are not counted as a missing kernel
