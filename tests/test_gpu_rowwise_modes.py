"""Distillation from top logits with and without gradients."""
import pytest
import torch

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
