"""Row operators at the ends of their ranges: masks of the type's lowest value over whole vectors, threads and blocks,
temperatures and offsets that scale every logit up, biases far from 0."""
import pytest
import torch

import forgeminds_b200 as fm
from rowwise_oracle import U32, within

pytestmark = pytest.mark.gpu
K = fm.kernels
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


# ------------------------------------------------------------------------------ top-logit KL
def kl_exact(student, values, index, tau):
    """Row losses and gradients of their sum in 64 bits, with bounds that do not know how large the logits are, only how far
    they lie from their row's largest one: fp32 arithmetic that takes this difference first is off by four units of the
    exponent (difference, 1 / tau with its logarithm, product), 2^x by 2^-22, sums of V values in chains of V / 512.
    A sum may be taken around a logit that is up to 8 in base 2 below the largest (6 in base e)."""
    V, keep = student.shape[1], index.shape[1]
    z, t = student.double(), values.double()
    high, first = z.amax(1, keepdim=True), t.amax(1, keepdim=True)
    x, tv = (z - high) / tau, (t - first) / tau
    total, mass = x.exp().sum(1, keepdim=True), tv.exp().sum(1, keepdim=True)
    q, p = x.exp() / total, tv.exp() / mass
    logp, logq = tv - mass.log(), x.gather(1, index) - total.log()
    row = torch.where(p > 0, p * (logp - logq), torch.zeros_like(p)).sum(1)
    want = torch.zeros_like(q).scatter_add_(1, index, p)
    span, tspan = x.abs().masked_fill(x == -float("inf"), 0.0), tv.abs()
    rtotal = 2.0 ** -20 + U32 * (V / 512 + 64) + 8 * U32 * (q * (span + 6)).sum(1, keepdim=True)
    rq = rtotal + 2.0 ** -22 + 8 * U32 * (span + 6)
    rp = 2.0 ** -22 + U32 * (16 + keep) + 8 * U32 * (tspan + (p * tspan).sum(1, keepdim=True))
    # (what 2^x gives below 2^-126 is 0)
    off_grad = ((rq + U32 * 8) * q + torch.zeros_like(q).scatter_add_(1, index, (rp + 8 * U32) * p) + 2.0 ** -125) / tau
    parts = rp * (logp - logq).abs() + 8 * U32 * (span.gather(1, index) + tspan + 6) + rtotal
    parts = parts + (keep + 40) * U32 * (logp.abs() + logq.abs() + total.log().abs())
    off_row = torch.where(p > 0, p * parts, torch.zeros_like(p)).sum(1)
    return row, (q - want) / tau, off_row, off_grad


def check_kl(student, values, index, tau, gradient_only=False):
    """Loss and both gradients: the one that the forward pass leaves (an upstream gradient of 1) and the backward kernel's."""
    row, grad, off_row, off_grad = kl_exact(student, values, index, tau)
    s = student.detach().requires_grad_()
    for up in (1.0, 0.5):
        rows = K.kl_topk_logits(s, values, index, temperature=tau, reduction="none")
        (g,) = torch.autograd.grad(rows, s, torch.full_like(rows, up))
        assert within(g, grad * up, off_grad * up) <= 0
        if not gradient_only:
            assert within(rows.detach(), row, off_row) <= 0


def kl_inputs(rows, V, keep, seed, dtype, lo=0, hi=None):
    """Teacher logits are those of [lo, hi) alone."""
    student = (randn(rows, V, seed=seed) * 2).to(DT[dtype])
    values, index = (randn(rows, V, seed=seed + 1) * 2)[:, lo:hi].topk(keep, dim=-1)
    return student, values.contiguous(), (index + lo).contiguous()


MASKED = [  # rows, V, kept, masked range: tails, heads, a middle, whole blocks of rows that a cluster shares, all but one
    (3, 1000, 16, 500, 700), (5, 1000, 16, 500, 1000), (5, 1000, 300, 500, 1000), (3, 1003, 8, 0, 640), (3, 40, 4, 8, 40),
    (2100, 520, 9, 256, 520), (2, 128259, 64, 0, 64000), (2, 128259, 64, 70001, 128259), (2, 128259, 500, 9, 128000),
    (40, 128259, 20, 40000, 128259), (2, 700001, 5, 8, 700001), (2, 900001, 5, 100, 800000)]


@pytest.mark.parametrize("rows,V,keep,lo,hi", MASKED)
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("mask", ["lowest", "inf"])
def test_kl_topk_ranges_of_masked_student_logits(rows, V, keep, lo, hi, dtype, mask):
    """Whole vectors, whole threads and whole blocks of nothing but masked logits."""
    open_lo, open_hi = (0, lo) if lo >= V - hi else (hi, V)
    student, values, index = kl_inputs(rows, V, min(keep, open_hi - open_lo), 10, dtype, open_lo, open_hi)
    student[:, lo:hi] = torch.finfo(DT[dtype]).min if mask == "lowest" else float("-inf")
    for tau in (1.0, 0.5, 2.0):
        check_kl(student, values, index, tau)


@pytest.mark.parametrize("V,keep", [(1000, 4), (1000, 300), (128259, 4)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_kl_topk_gradient_of_a_row_of_equal_lowest_logits(V, keep, dtype):
    student, values, index = kl_inputs(2, V, keep, 13, dtype)
    student[0] = torch.finfo(DT[dtype]).min
    check_kl(student, values, index, 1.0, gradient_only=True)


@pytest.mark.parametrize("V,keep", [(1001, 9), (1001, 300), (128259, 9)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("tau", [1e-3, 1e-6, 1e-9, 1e-12, 1e-20, 1e4, 1e20])
def test_kl_topk_gradient_at_any_temperature(V, keep, dtype, tau):
    student, values, index = kl_inputs(3, V, keep, 16, dtype)
    check_kl(student, values, index, tau, gradient_only=True)


@pytest.mark.parametrize("V,keep", [(1001, 9), (1001, 300), (128259, 9)])
@pytest.mark.parametrize("offset", [1e3, -1e4, 1e5])
@pytest.mark.parametrize("tau", [1.0, 3.0])
def test_kl_topk_gradient_of_logits_far_from_zero(V, keep, offset, tau):
    student, values, index = kl_inputs(3, V, keep, 19, "fp32")
    check_kl(student + offset, values, index, tau, gradient_only=True)


@pytest.mark.parametrize("V,keep", [(1001, 9), (1001, 300), (128259, 9)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("tau", [1e-3, 1e-6, 1e-9, 1e-12, 1e-20, 1e4, 1e20])
def test_kl_topk_loss_at_any_temperature(V, keep, dtype, tau):
    student, values, index = kl_inputs(3, V, keep, 22, dtype)
    check_kl(student, values, index, tau)


@pytest.mark.parametrize("V,keep", [(1001, 9), (1001, 300), (128259, 9)])
@pytest.mark.parametrize("offset,teacher_offset", [(1e3, 0), (-1e4, 1e4), (1e5, -1e5)])
@pytest.mark.parametrize("tau", [1.0, 3.0])
def test_kl_topk_loss_of_logits_far_from_zero(V, keep, offset, teacher_offset, tau):
    """Adding a number to all of a row's logits, or to all of the teacher's, changes nothing but their own roundings."""
    student, values, index = kl_inputs(3, V, keep, 25, "fp32")
    check_kl(student + offset, values + teacher_offset, index, tau)


@pytest.mark.parametrize("V,keep", [(1000, 4), (1000, 300), (128259, 4)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_kl_topk_of_rows_of_equal_lowest_logits(V, keep, dtype):
    student, values, index = kl_inputs(3, V, keep, 28, dtype)
    student[0] = torch.finfo(DT[dtype]).min
    values[1] = torch.finfo(torch.float32).min
    for tau in (1.0, 0.5, 2.0):
        check_kl(student, values, index, tau)


# ------------------------------------------------------------------------------ routing
def check_choice(logits, k, bias, **options):
    """The choice is the 64-bit statement's."""
    _, idx, counts, _ = K.route_experts(logits, k, bias=bias, **options)
    from forgeminds_b200.kernels import reference
    softmax = options.get("score", "softmax") == "softmax"
    _, want, want_counts, _ = reference.route_experts(logits, k, softmax, bias, options.get("n_groups", 1), options.get("top_groups", 1))
    assert torch.equal(idx, want) and torch.equal(counts, want_counts)


@pytest.mark.parametrize("E,k,groups", [(8, 2, 1), (64, 6, 8), (60, 6, 4), (256, 8, 8), (256, 8, 1), (512, 4, 1)])
@pytest.mark.parametrize("near", [3.5, 31.5, 63.5, 127.5, 255.5, 2e4, -63.5])
def test_route_with_biases_far_from_zero(E, k, groups, near):
    """One bias for all experts, a unit or more beyond ``near``, and biases spread over less than 1: whatever is added to
    them in 32 bits crosses a power of two. Scores reach 1."""
    logits = randn(300, E, seed=40) * 2
    at = torch.arange(300, device="cuda")
    logits[at, at * 7 % E] = 40.0                            # sigmoid 1, softmax 1
    logits[at[::3], at[::3] * 5 % E] = 14.0                  # sigmoid 1 - 8e-7
    base = torch.tensor(near, dtype=torch.float32, device="cuda")
    for units in (0, 1, 3, 2 ** 12):
        bias = (base.view(torch.int32) + units).view(torch.float32).repeat(E)
        for score in ("sigmoid", "softmax"):
            check_choice(logits, k, bias, score=score, n_groups=groups, top_groups=max(1, groups // 2))
            check_choice(logits.bfloat16(), k, bias, score=score, n_groups=groups, top_groups=max(1, groups // 2))
            spread = bias + randn(E, seed=41 + units) * 0.1
            check_choice(logits, k, spread, score=score, n_groups=groups, top_groups=max(1, groups // 2))


# ------------------------------------------------------------------------------ LayerNorm on clusters
@pytest.mark.parametrize("rows,d,dtype", [(700, 8200, "bf16"), (300, 16384, "bf16"), (301, 16384, "fp32"), (500, 4100, "fp32"), (3, 32768, "bf16")])
def test_layer_norm_wide_backward_is_the_same_every_time(rows, d, dtype):
    """Several rows for each cluster, whose blocks exchange their sums row by row."""
    x, dy, ds = (randn(rows, d, seed=50 + i, dtype=DT[dtype]) for i in range(3))
    w, b = 1 + 0.1 * randn(d, seed=53), randn(d, seed=54)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    total, y = K.add_layer_norm(x, torch.zeros_like(x), w, b)
    first = torch.autograd.grad((total, y), leaves, (ds, dy), retain_graph=True)
    for _ in range(20):
        again = torch.autograd.grad((total, y), leaves, (ds, dy), retain_graph=True)
        assert all(torch.equal(p, q) for p, q in zip(first, again))
