"""What the kernels' path of LayerNorm, rotary positions, expert routing and top-logit distillation refuses, the scratch it
uses, views of one row or one token with odd strides, and tensors of more than 2^31 values."""
import pytest
import torch

import forgeminds_b200 as fm
from forgeminds_b200 import ops
import test_gpu_rowwise as rowwise
from test_gpu_rowwise import check_route

pytestmark = pytest.mark.gpu
K = fm.kernels


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


# ------------------------------------------------------------------------------ refusals
def refused(calls):
    for n, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {n} was taken")


def test_layer_norm_refuses():
    x, one = randn(4, 8), torch.ones(8, device="cuda")
    refused([lambda: K.layer_norm(x, one[:7]), lambda: K.layer_norm(x, one, one.view(2, 4)), lambda: K.layer_norm(x.long()),
             lambda: K.layer_norm(x[0, 0]), lambda: K.layer_norm(x[:, :0]), lambda: K.add_layer_norm(x, x[:2]),
             lambda: K.add_layer_norm(x, x.double()), lambda: K.add_layer_norm(x, x.bfloat16()), lambda: K.layer_norm(x, one.cpu()),
             lambda: K.add_layer_norm(x, x.cpu()), lambda: K.add_layer_norm(x, x, one[:4])])


def test_rotary_refuses():
    q, k = randn(2, 5, 3, 8), randn(2, 5, 1, 8)
    cos, sin = K.rotary_tables(5, 8, device="cuda")
    wide = K.rotary_tables(5, 10, device="cuda")
    zeros = torch.zeros(5, dtype=torch.int64, device="cuda")
    refused([lambda: K.rotary(q[0], cos, sin), lambda: K.rotary_qk(q, k[:, :4], cos, sin), lambda: K.rotary_qk(q, k.bfloat16(), cos, sin),
             lambda: K.rotary_qk(q, k[..., :6], cos, sin), lambda: K.rotary_qk(q, k[0], cos, sin), lambda: K.rotary(q, *wide),
             lambda: K.rotary(q, cos, sin[:4]), lambda: K.rotary(q, cos[:4], sin[:4]), lambda: K.rotary(q, cos, sin, zeros.float()),
             lambda: K.rotary(q, cos, sin, zeros[:4]), lambda: K.rotary(q, cos, sin, zeros.view(5, 1).expand(5, 2)),
             lambda: K.rotary(q, cos, sin, zeros.cpu()), lambda: K.rotary(q, cos.cpu(), sin), lambda: K.rotary(q.long(), cos, sin),
             lambda: K.rotary(q, cos[:0], sin[:0], zeros), lambda: K.rotary(q, cos.long(), sin.long()),
             lambda: K.rotary(q, cos, sin.clone().requires_grad_())])


def test_kl_topk_refuses():
    student = randn(4, 10)
    values, index = randn(4, 10, seed=1).topk(3, dim=-1)
    refused([lambda: K.kl_topk_logits(student, values, index, reduction="batchmean"), lambda: K.kl_topk_logits(student, values, index, temperature=0.0),
             lambda: K.kl_topk_logits(student, values, index, temperature=float("inf")), lambda: K.kl_topk_logits(student, values, index, temperature=1e-30),
             lambda: K.kl_topk_logits(student, values, index, temperature=float("nan")), lambda: K.kl_topk_logits(student, values[:2], index),
             lambda: K.kl_topk_logits(student, values[:2], index[:2]), lambda: K.kl_topk_logits(student, values, index.float()),
             lambda: K.kl_topk_logits(student, values.long(), index), lambda: K.kl_topk_logits(student.long(), values, index),
             lambda: K.kl_topk_logits(student, values[:, :0], index[:, :0]), lambda: K.kl_topk_logits(student[:, :0], values, index),
             lambda: K.kl_topk_logits(student, values.cpu(), index), lambda: K.kl_topk_logits(student, values, index.cpu()),
             lambda: K.kl_topk_logits(student, values[0], index[0]), lambda: K.kl_topk_logits(student[0], values, index),
             lambda: K.kl_topk_logits(student, values, index, teacher_lse=student[:3, 0]),
             lambda: K.kl_topk_logits(student, values, index, teacher_lse=index[:, 0]),
             lambda: K.kl_topk_distill_loss(student, student[:, :9], values, index),
             lambda: K.kl_topk_distill_loss(student, student, values, index, chunk=0)])


def test_route_refuses():
    z, bias = randn(4, 8), randn(8)
    refused([lambda o=o: K.route_experts(z, **o) for o in (
        dict(k=0), dict(k=9), dict(k=2, score="tanh"), dict(k=2, n_groups=3), dict(k=2, n_groups=0), dict(k=2, n_groups=4, top_groups=0),
        dict(k=2, n_groups=4, top_groups=5), dict(k=5, n_groups=4, top_groups=2), dict(k=2, group_best=3), dict(k=2, bias=bias[:7]),
        dict(k=2, bias=bias.long()), dict(k=2, bias=bias.cpu()), dict(k=2, bias=bias.view(2, 4)))])
    refused([lambda b=b: K.route_experts(b, 1) for b in (z[0], z.long(), z[:, :0])])


# ------------------------------------------------------------------------------ scratch
@pytest.mark.parametrize("rows", [1, 9, 2048, 5000])
def test_kl_topk_scratch_holds_what_the_kernels_leave_there(rows):
    """The count kernel leaves one number per block behind the first four; together they are the rows that count."""
    student = randn(rows, 40)
    values, index = randn(rows, 40, seed=1).topk(2, dim=-1)
    index[::3] = -1
    counted = rows - (rows + 2) // 3
    ws = ops.require().kl_topk_fwd(student, values, index, None, 1.0, True, True, None, True, False)[4]
    blocks = min((rows + 31) // 32, 256)                       # 32 rows for each, as long as there are blocks
    assert ws.numel() >= 4 + blocks and int(ws[0]) == counted and int(ws[4: 4 + blocks].sum()) == counted


def test_kl_topk_leaves_its_neighbours_alone():
    """Small tensors stand around the scratch in the allocator's blocks: they keep their values."""
    student = randn(4096, 16, dtype=torch.bfloat16)
    values, index = randn(4096, 16, seed=1).topk(2, dim=-1)
    around = [torch.full((128,), 7, dtype=torch.int32, device="cuda") for _ in range(256)]
    for keep in (0, 1):
        for n in range(keep, 256, 2):
            around[n] = None                                   # holes of 512 bytes between those that stay
        K.kl_topk_logits(student, values, index)
        torch.cuda.synchronize()
        assert all(bool((t == 7).all()) for t in around if t is not None)
        around = [torch.full((128,), 7, dtype=torch.int32, device="cuda") for _ in range(256)]


# ------------------------------------------------------------------------------ one row, one token: strides that mean nothing
def odd(t, *dims):
    """The same values, with odd strides where there is only one of them."""
    strides = [s + 3 if d in dims else s for d, s in enumerate(t.stride())]
    return t.as_strided(t.shape, strides)


def test_strides_of_single_rows_do_not_matter():
    for dtype in (torch.bfloat16, torch.float32):
        x = randn(1, 1024, dtype=dtype)
        values, index = randn(1, 1024, seed=1).topk(8, dim=-1)
        for call in (K.layer_norm, lambda t: K.add_layer_norm(t, t)[1], lambda t: K.kl_topk_logits(t, values, index),
                     lambda t: K.route_experts(t[:, :256], 8)[0]):
            leaf, want = odd(x, 0).requires_grad_(), x.clone().requires_grad_()
            a, b = call(leaf), call(want)
            assert torch.equal(a, b)
            assert torch.equal(torch.autograd.grad(a.float().sum(), leaf)[0], torch.autograd.grad(b.float().sum(), want)[0])
        cos, sin = K.rotary_tables(9, 64, device="cuda")
        at = torch.tensor([8], device="cuda")
        q = randn(1, 1, 4, 64, seed=2, dtype=dtype)
        assert torch.equal(K.rotary(odd(q, 0, 1), cos, sin, at), K.rotary(q, cos, sin, at))
        one = randn(3, 5, 1, 64, seed=3, dtype=dtype)
        assert torch.equal(K.rotary(odd(one, 2), cos, sin), K.rotary(one, cos, sin))


# ------------------------------------------------------------------------------ more than 2^31 values
def long_rows(rows, width):
    t = torch.empty(rows, width, dtype=torch.bfloat16, device="cuda")
    t[:64] = randn(64, width, seed=1)
    t[64:-64] = 0.5
    t[-64:] = randn(64, width, seed=2)
    return t


def test_layer_norm_beyond_31_bits():
    x = long_rows(524400, 4096)
    w = randn(4096, seed=3)
    out = K.layer_norm(x, w)
    assert x.numel() > 2 ** 31 and torch.equal(out[-64:], K.layer_norm(x[-64:], w)) and torch.equal(out[:64], K.layer_norm(x[:64], w))
    dy = out
    del out
    x.requires_grad_()
    y = K.layer_norm(x, w)
    (dx,) = torch.autograd.grad(y, x, dy)
    tail = x.detach()[-64:].clone().requires_grad_()
    (want,) = torch.autograd.grad(K.layer_norm(tail, w), tail, dy[-64:])
    assert torch.equal(dx[-64:], want)


def test_rotary_beyond_31_bits():
    T = 262400
    q = long_rows(T, 64 * 128).view(1, T, 64, 128)
    cos, sin = K.rotary_tables(T, 128, device="cuda")
    out = K.rotary(q, cos, sin)
    at = torch.arange(T - 64, T, device="cuda")
    assert q.numel() > 2 ** 31 and torch.equal(out[:, -64:], K.rotary(q[:, -64:], cos, sin, at))


def test_kl_topk_beyond_31_bits():
    rows, V = 16800, 128259
    x = long_rows(rows, V).requires_grad_()
    values, index = torch.full((rows, 4), 1.0, device="cuda"), torch.arange(4, device="cuda").expand(rows, 4).contiguous()
    values[-64:], index[-64:] = x.detach()[-64:].float().topk(4, dim=-1)
    loss = K.kl_topk_logits(x, values, index, reduction="none")
    (g,) = torch.autograd.grad(loss.sum(), x)
    tail = x.detach()[-64:].clone().requires_grad_()
    part = K.kl_topk_logits(tail, values[-64:], index[-64:], reduction="none")
    (want,) = torch.autograd.grad(part.sum(), tail)
    # another number of blocks per row: sums of 128259 exponentials in another order, one rounding to bf16 of the gradient
    assert x.numel() > 2 ** 31 and torch.allclose(loss[-64:], part, rtol=1e-4, atol=1e-4)
    assert bool(((g[-64:].float() - want.float()).abs() <= 2 ** -7 * want.float().abs() + 1e-9).all())


def test_route_beyond_31_bits():
    z = long_rows(8400000, 256)
    w, idx, counts, _ = K.route_experts(z, 2, score="sigmoid")
    w2, idx2, _, _ = K.route_experts(z[-64:], 2, score="sigmoid")
    assert z.numel() > 2 ** 31 and torch.equal(w[-64:], w2) and torch.equal(idx[-64:], idx2) and int(counts.sum()) == 2 * z.shape[0]
    z.requires_grad_()
    (g,) = torch.autograd.grad(K.route_experts(z, 2, score="sigmoid")[0][:, 0].sum(), z)
    tail = z.detach()[-64:].clone().requires_grad_()
    (want,) = torch.autograd.grad(K.route_experts(tail, 2, score="sigmoid")[0][:, 0].sum(), tail)
    assert torch.equal(g[-64:], want)


# ------------------------------------------------------------------------------ orders that the fast choice leaves open
@pytest.mark.parametrize("E,k,groups", [(64, 8, 1), (100, 20, 1), (128, 8, 4), (256, 8, 1), (256, 16, 8), (512, 12, 1), (384, 9, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_route_when_neighbouring_experts_win(E, k, groups, dtype):
    """All choices lie side by side: one lane has more of them than it keeps in its list."""
    slope = torch.linspace(2, -2, E, device="cuda")
    z = torch.stack([slope.roll(s) + 1e-3 * randn(E, seed=s) for s in range(0, E, 7)]).to(dtype)
    bias = 0.01 * randn(E, seed=5)
    for score in ("softmax", "sigmoid"):
        for b in (None, bias):
            check_route(z, k, score, b, groups, max(1, groups // 2))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_route_signed_zeros_and_equal_logits(dtype):
    z = randn(50, 64, seed=6).round().to(dtype)
    z[:, ::3] = 0.0
    z[:, 1::3] = -0.0
    z[10:20, 5:] = float("-inf")
    z[20:30] = -z[20:30].abs()
    for score in ("softmax", "sigmoid"):
        for groups in (1, 8):
            check_route(z[:10], 6, score, None, groups, max(1, groups // 2))
            check_route(z[20:], 6, score, torch.zeros(64, device="cuda"), groups, max(1, groups // 2), best=1)
        w, idx, _, _ = K.route_experts(z[10:20], 5, score=score)
        assert torch.equal(idx.long(), z[10:20].double().sort(dim=1, descending=True, stable=True)[1][:, :5])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_route_many_tokens_that_are_decided_again(dtype):
    """More steps per warp than it takes before it goes back to the undecided tokens; every order is the logits'."""
    z = (randn(1200000, 64, seed=7) * 4).round().div(8).to(dtype)
    z[5::997, 3] = float("inf")
    z[7::501] = 0.25
    want = z.sort(dim=1, descending=True, stable=True)[1][:, :6]
    zeros = torch.zeros(64, device="cuda")
    for opts in (dict(), dict(score="sigmoid"), dict(score="sigmoid", bias=zeros)):
        w, idx, counts, _ = K.route_experts(z, 6, **opts)
        keep = torch.ones(len(z), dtype=torch.bool, device="cuda") if not opts else torch.isfinite(z).all(1)
        assert torch.equal(idx.long()[keep], want[keep])
        assert torch.equal(counts.long(), torch.bincount(idx.flatten().long(), minlength=64))


# ------------------------------------------------------------------------------ forms chosen by size
@pytest.mark.parametrize("D,R", [(64, 4), (64, 62), (96, 34), (128, 50), (256, 98), (8, 2), (80, 72)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_rotary_of_a_part_that_ends_inside_a_vector(D, R, interleaved, dtype):
    rowwise.test_rotary_qk(2, 37, 6, 3, D, R, interleaved, dtype, True)
    rowwise.test_rotary_qk(1, 700, 5, 1, D, R, interleaved, dtype, False)
    x = randn(1, 4, 3, D, seed=8, dtype=rowwise.DT[dtype])
    x[0, 1, 1] = float("inf")
    at = torch.tensor([0, -1, 99, -7], device="cuda")
    cos, sin = K.rotary_tables(9, R, device="cuda")
    y = K.rotary(x, cos, sin, at, interleaved)
    assert torch.equal(y[:, 1::2], x[:, 1::2])                 # negative positions: as they are, infinities too
    assert bool(torch.isnan(y[0, 2, :, :R]).all()) and torch.equal(y[..., R:], x[..., R:])


@pytest.mark.parametrize("rows,V,keep", [(2000, 1000, 100), (6000, 2056, 33), (1800, 12162, 128), (1800, 12167, 129), (2100, 31, 4)])
@pytest.mark.parametrize("dtype,tdtype", [("bf16", "bf16"), ("fp32", "fp32")])
def test_kl_topk_many_short_rows(rows, V, keep, dtype, tdtype):
    student, values, index, teacher = rowwise.kl_inputs(rows, V, keep, 41, dtype, tdtype)
    index[5::9, 1] = index[5::9, 0]                            # an index that stands twice
    index[7::11] = -1                                          # rows that do not count
    index[::13, keep - 1] = V                                  # and slots
    rowwise.check_kl(student, values, index, 2.0)
    rowwise.check_kl(student, values, index, 1.0, torch.logsumexp(teacher, -1), reduction="sum")


@pytest.mark.parametrize("rows,V,keep,dtype", [(3, 200003, 20, "fp32"), (2, 393000, 256, "fp32"), (2, 800001, 7, "bf16"), (2, 900001, 7, "fp32")])
def test_kl_topk_wider_than_eight_blocks_of_64_kb(rows, V, keep, dtype):
    student, values, index, _ = rowwise.kl_inputs(rows, V, keep, 42, dtype, "fp32")
    rowwise.check_kl(student, values, index, 1.5)


@pytest.mark.parametrize("d", [8256, 16384, 16388, 20001, 32768])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_layer_norm_wide_rows(d, dtype):
    rowwise.test_layer_norm(300, d, dtype, "fp32")
    rowwise.test_add_layer_norm(41, d, dtype)


@pytest.mark.parametrize("E,k", [(312, 14), (64, 8), (8, 3)])
def test_route_softmax_scores_that_a_bias_brings_together(E, k):
    """Pairs whose biased scores differ by a few units of 32 bits, on either side, and pairs that are equal by their inputs."""
    z = randn(400, E, seed=9)
    z[:, 1] = z[:, 0] - 0.5
    s = torch.softmax(z.double(), dim=1)
    for row in range(0, 400, 57):                              # the bias that makes experts 0 and 1 of this row nearly equal
        for off in (0.0, 3e-9, -3e-9, 1e-7):
            bias = 0.001 * randn(E, seed=10)
            bias[0] = 0.5
            bias[1] = (0.5 + s[row, 0] - s[row, 1] + off).float()
            check_route(z[row: row + 1], k, "softmax", bias)
    bias = torch.zeros(E, device="cuda")
    check_route(z, k, "softmax", bias)
    check_route(z, k, "softmax", 0.02 * randn(E, seed=11))


@pytest.mark.parametrize("rows,keep", [(1, 33), (37, 64), (9000, 40), (300, 500)])
def test_kl_topk_rows_whose_first_slots_do_not_count(rows, keep):
    student, values, index, _ = rowwise.kl_inputs(rows, 600, keep, 43, "fp32", "fp32")
    index[::2, : keep - 1] = -1                                # the last slot alone
    index[1::7] = 600
    values[3::5, :32] = float("-inf")
    rowwise.check_kl(student, values, index, 1.0)


def test_wide_layer_norm_in_a_captured_graph():
    """Kernels on clusters, launched and measured for the first time while a graph is captured."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = randn(70, 24008, seed=44, dtype=torch.bfloat16).requires_grad_()
        w, dy = randn(24008, seed=45).requires_grad_(), randn(70, 24008, seed=46, dtype=torch.bfloat16)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = K.layer_norm(x, w)
            dx, dw = torch.autograd.grad(y, (x, w), dy)
        for seed in (47, 48):
            with torch.no_grad():
                x.copy_(randn(70, 24008, seed=seed))
            graph.replay()
            other, weight = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
            want = K.layer_norm(other, weight)
            gx, gw = torch.autograd.grad(want, (other, weight), dy)
            assert torch.equal(y, want) and torch.equal(dx, gx) and torch.equal(dw, gw)
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_groups_that_differ_only_in_the_order_of_their_biases(score):
    """The same two logits with the same two biases, exchanged: equal groups, of which the lower ones are kept."""
    steps = (2 * randn(40, seed=12)).round() * 1e-3
    for size, groups in ((2, 16), (7, 16), (13, 4), (32, 8)):
        z = (randn(300, size * groups, seed=13)).round() / 2
        bias = steps[torch.randint(0, 40, (size * groups,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(14))]
        z[::2] = z[::2, :size].repeat(1, groups)               # the same logits in every group
        z[::4, :size] = z[::4, :size].flip(1)                  # and in another order
        for dtype in (torch.float32, torch.bfloat16):
            for b in (None, bias):
                check_route(z.to(dtype), 2, score, b, groups, groups // 2)
    leaf = randn(64, 16, seed=16).requires_grad_()
    (g,) = torch.autograd.grad(K.route_experts(leaf, 1, scale=1.5)[0], leaf, randn(64, 1, seed=17))
    assert not g.any()                                         # one renormalised choice has the weight 1, whatever its score
