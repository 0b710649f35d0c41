"""Distillation from top logits with and without gradients, and derivatives that the row operators do not have."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import forgeminds_b200 as fm

pytestmark = pytest.mark.gpu
K = fm.kernels


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def test_an_evaluation_pass_keeps_chunk_rows_of_logits():
    """The head is a Parameter; without gradients the logits are ``chunk x V`` and no gradient is written."""
    n, V, d, chunk = 4096, 16000, 64, 256
    h, w = randn(n, d, dtype=torch.bfloat16), torch.nn.Parameter(randn(V, d, seed=1, dtype=torch.bfloat16))
    values, index = randn(n, 64, seed=2), torch.randint(0, V, (n, 64), device="cuda")
    with torch.no_grad():
        K.kl_topk_distill_loss(h, w, values, index, chunk=chunk)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        loss = K.kl_topk_distill_loss(h, w, values, index, chunk=chunk)
        peak = torch.cuda.max_memory_allocated() - before
    assert not loss.requires_grad
    # the chunk's logits, the teacher's mask of kept slots in its temporaries, and the rest of a megabyte or two
    assert peak <= 2 * chunk * V + 64 * n * 16 + 2 ** 22, peak
    with_grad = K.kl_topk_distill_loss(h, w, values, index, chunk=chunk)
    assert torch.equal(with_grad.detach(), loss)


def _forward_mode_calls(d):
    """A call for each differentiable input ``d`` stands in for: a dual number without ``requires_grad``."""
    x, w, b = randn(6, 64), 1 + 0.1 * randn(64, seed=3), randn(64, seed=4)
    q, k = randn(2, 6, 4, 32, seed=5), randn(2, 6, 2, 32, seed=6)
    cos, sin = K.rotary_tables(6, 32, device="cuda")
    v, i = randn(6, 64, seed=7).topk(5, dim=-1)
    z = randn(6, 16, seed=8)
    return {"layer_norm x": lambda: K.layer_norm(d(x), w, b), "layer_norm w": lambda: K.layer_norm(x, d(w), b),
            "layer_norm b": lambda: K.layer_norm(x, w, d(b)), "add_layer_norm x": lambda: K.add_layer_norm(d(x), x, w, b),
            "add_layer_norm delta": lambda: K.add_layer_norm(x, d(x)), "rotary": lambda: K.rotary(d(q), cos, sin),
            "rotary_qk q": lambda: K.rotary_qk(d(q), k, cos, sin), "rotary_qk k": lambda: K.rotary_qk(q, d(k), cos, sin),
            "kl": lambda: K.kl_topk_logits(d(x), v, i), "kl rows": lambda: K.kl_topk_logits(d(x), v, i, reduction="none"),
            "kl distill h": lambda: K.kl_topk_distill_loss(d(x), randn(40, 64, seed=9), v, i % 40),
            "kl distill bf16 h": lambda: K.kl_topk_distill_loss(d(x.bfloat16()), randn(40, 64, seed=9), v, i % 40),
            "kl distill bf16 w": lambda: K.kl_topk_distill_loss(x.bfloat16(), d(randn(40, 64, seed=9)), v, i % 40),
            "route": lambda: K.route_experts(d(z), 3), "route aux": lambda: K.route_experts(d(z), 3, aux_coef=0.1)}


NAMES = ["layer_norm x", "layer_norm w", "layer_norm b", "add_layer_norm x", "add_layer_norm delta", "rotary", "rotary_qk q",
         "rotary_qk k", "kl", "kl rows", "kl distill h", "kl distill bf16 h", "kl distill bf16 w", "route", "route aux"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_is_refused(name, grad_mode):
    """A tangent that a kernel does not carry is not dropped without a word, with reverse mode on or off."""
    with fwd.dual_level(), torch.set_grad_enabled(grad_mode):
        call = _forward_mode_calls(lambda t: fwd.make_dual(t, torch.ones_like(t)))[name]
        with pytest.raises((RuntimeError, NotImplementedError), match="(?i)forward|jvp"):
            call()


@pytest.mark.parametrize("which", [0, 1])
def test_tables_with_tangents_are_refused(which):
    q = randn(2, 6, 4, 32)
    with fwd.dual_level():
        tables = list(K.rotary_tables(6, 32, device="cuda"))
        tables[which] = fwd.make_dual(tables[which], torch.ones_like(tables[which]))
        with pytest.raises(ValueError, match="constants"):
            K.rotary(q, *tables)


def _negated(t):
    """``t``'s values as a view that is negated lazily."""
    view = torch.imag(torch.complex(torch.zeros_like(t), -t).conj())
    assert view.is_neg() and torch.equal(view, t)
    return view


def test_gradients_that_are_lazily_negated():
    x, q = randn(6, 64).requires_grad_(), randn(2, 6, 4, 32, seed=5).requires_grad_()
    tables = K.rotary_tables(6, 32, device="cuda")
    v, i = randn(6, 64, seed=7).topk(5, dim=-1)
    outs = [(K.layer_norm(x), x), (K.add_layer_norm(x, x.detach())[1], x), (K.rotary(q, *tables), q),
            (K.kl_topk_logits(x, v, i, reduction="none"), x), (K.route_experts(x, 4)[0], x)]
    for n, (y, leaf) in enumerate(outs):
        up = randn(*y.shape, seed=20 + n)
        (lazy,) = torch.autograd.grad(y, leaf, _negated(up), retain_graph=True)
        (want,) = torch.autograd.grad(y, leaf, up)
        assert torch.allclose(lazy, want, rtol=1e-5, atol=1e-6), n     # (of the loss another kernel's roundings)


def test_a_dtensor_takes_the_pytorch_statements(tmp_path):
    import torch.distributed as dist
    from torch.distributed.tensor import DTensor, Replicate, init_device_mesh
    if dist.is_initialized():
        pytest.skip("a process group is there already")
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/store", rank=0, world_size=1)
    try:
        mesh = init_device_mesh("cuda", (1,))

        def wrap(t):
            return DTensor.from_local(t, mesh, [Replicate()], run_check=False)
        x, w = randn(6, 64), 1 + 0.1 * randn(64, seed=3)
        K.reset_stats()
        y = K.layer_norm(wrap(x), wrap(w))
        z = K.rms_norm(wrap(x), wrap(w))
        assert K.stats()["fast"] == 0 and K.stats()["fallback"] == 2
        assert torch.allclose(y.to_local(), K.layer_norm(x, w), rtol=1e-5, atol=1e-5)
        assert torch.allclose(z.to_local(), K.rms_norm(x, w), rtol=1e-5, atol=1e-5)
        v, i = randn(6, 64, seed=7).topk(5, dim=-1)
        q, (cos, sin) = randn(2, 6, 4, 32, seed=5), K.rotary_tables(6, 32, device="cuda")
        for call in (lambda: K.kl_topk_logits(x, wrap(v), i), lambda: K.kl_topk_logits(x, v, wrap(i)), lambda: K.rotary(q, wrap(cos), sin),
                     lambda: K.route_experts(x, 4, bias=wrap(w)), lambda: K.kl_topk_distill_loss(x, randn(40, 64), wrap(v), i % 40)):
            with pytest.raises((TypeError, RuntimeError)):
                call()
    finally:
        dist.destroy_process_group()


def test_results_can_be_changed_in_place():
    """As those of ``torch.nn.functional.layer_norm``, which a patched module stands for."""
    x, w, up = randn(2, 3, 64).requires_grad_(), (1 + 0.1 * randn(64, seed=1)).requires_grad_(), randn(2, 3, 64, seed=2)
    v, i = randn(2, 3, 64, seed=3).topk(4, dim=-1)
    zero = torch.zeros_like(x)
    for n, call in enumerate((lambda: K.layer_norm(x, w), lambda: K.layer_norm(x[0], w), lambda: K.add_layer_norm(x, zero, w)[1],
                              lambda: K.kl_topk_logits(x, v, i, reduction="none"), lambda: K.kl_topk_logits(x[0], v[0], i[0], reduction="none"),
                              lambda: K.kl_topk_logits(x[0, 0], v[0, 0], i[0, 0], reduction="none"))):
        y = call()
        g = up.flatten()[: y.numel()].view(y.shape)
        (want,) = torch.autograd.grad(y * 2, x, g)
        (got,) = torch.autograd.grad(call().mul_(2), x, g)
        assert torch.equal(got, want), n


def _leaf_calls():
    x, q = randn(6, 64).requires_grad_(), randn(2, 6, 4, 32, seed=5).requires_grad_()
    v, i = randn(6, 64, seed=7).topk(5, dim=-1)
    tables = K.rotary_tables(6, 32, device="cuda")
    return [(lambda a: K.layer_norm(a), x), (lambda a: K.add_layer_norm(a, a)[1], x), (lambda a: K.rotary(a, *tables), q),
            (lambda a: K.kl_topk_logits(a, v, i, reduction="none"), x), (lambda a: K.route_experts(a, 4, aux_coef=0.1)[0], x)]


def test_checkpointed_and_offloaded_activations():
    from torch.utils.checkpoint import checkpoint
    for n, (f, leaf) in enumerate(_leaf_calls()):
        (want,) = torch.autograd.grad(f(leaf).square().sum(), leaf)
        (again,) = torch.autograd.grad(checkpoint(f, leaf, use_reentrant=False).square().sum(), leaf)
        with torch.autograd.graph.save_on_cpu():
            loss = f(leaf).square().sum()
        (moved,) = torch.autograd.grad(loss, leaf)
        assert torch.equal(again, want) and torch.equal(moved, want), n


def test_transforms_that_wrap_tensors_are_refused():
    for f, leaf in _leaf_calls():
        y = f(leaf)
        with pytest.raises((TypeError, RuntimeError), match="plain strided"):
            torch.autograd.grad(y, leaf, randn(3, *y.shape), is_grads_batched=True)
        for call in (lambda: torch.func.grad(lambda a: f(a).sum())(leaf.detach()), lambda: torch.func.vmap(f)(torch.stack([leaf.detach()] * 2)),
                     lambda: torch.func.jvp(f, (leaf.detach(),), (leaf.detach(),))):
            with pytest.raises(TypeError, match="plain strided"):
                call()
