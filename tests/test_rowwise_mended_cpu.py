"""The row operators' PyTorch statements, modules and host logic in the calls that are easy to get wrong."""
import pytest
import torch

import forgeminds_b200 as fm

K = fm.kernels


def _randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ------------------------------------------------------------------------------ top-logit KL
def _kl_exact(student, values, index, tau):
    z, t = student.double(), values.double()
    x = (z - z.amax(1, keepdim=True)) / tau
    logq = x - x.exp().sum(1, keepdim=True).log()
    tv = (t - t.amax(1, keepdim=True)) / tau
    logp = tv - tv.exp().sum(1, keepdim=True).log()
    p = logp.exp()
    row = torch.where(p > 0, p * (logp - logq.gather(1, index)), torch.zeros_like(p)).sum(1)
    return row, (logq.exp() - torch.zeros_like(z).scatter_add_(1, index, p)) / tau


@pytest.mark.parametrize("offset,tau", [(0.0, 1.0), (1e4, 3.0), (-1e5, 3.0), (0.0, 1e-6), (0.0, 1e-12), (0.0, 1e-20), (0.0, 1e20)])
def test_kl_topk_takes_differences_first(offset, tau):
    """fp32: logits far from 0, any temperature, and a row of nothing but the type's lowest value."""
    student, teacher = _randn(5, 200, seed=1) * 2 + offset, _randn(5, 200, seed=2) * 2 - offset
    values, index = teacher.topk(7, dim=-1)
    student[1] = torch.finfo(torch.float32).min
    student[2, 64:] = torch.finfo(torch.float32).min
    index[2] = torch.arange(7)
    values[3] = torch.finfo(torch.float32).min
    student.requires_grad_()
    rows = K.kl_topk_logits(student, values, index, temperature=tau, reduction="none")
    (grad,) = torch.autograd.grad(rows.sum(), student)
    want, wgrad = _kl_exact(student.detach(), values, index, tau)
    # exponents are spans over tau, each off by a few units of its own size; the loss is of the size of the spans
    assert torch.allclose(rows.detach().double(), want, rtol=100 * 2.0 ** -24, atol=200 * 2.0 ** -24)
    assert torch.allclose(grad.double() * tau, wgrad * tau, rtol=1e-4, atol=1e-6)
