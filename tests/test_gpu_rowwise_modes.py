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
