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


# ------------------------------------------------------------------------------ sums that the blocks of a cluster exchange
def _unordered(slots, rows=8, ctas=2, warps=2):
    """Accesses of an exchange slot that the memory model leaves unordered, in the order of events of LayerNorm's backward
    kernel on clusters: per row the __syncthreads of the row's sums, the wait for the last row's exchange, reads of its slot,
    warp 0's writes to the peers' slots, its fence, the arrival. Warp 0's fence and arrival are ordered before a wait; the
    other warps' relaxed arrivals order nothing."""
    before = {}                                              # event -> events that happen before it, directly

    def event(name, *after):
        before.setdefault(name, set()).update(after)
        return name

    last = {}
    for i in range(rows + 1):
        more, had = i < rows, i > 0
        for c in range(ctas):
            if more:                                         # what stands before a __syncthreads is before what follows in any warp
                event(("sync", c, i), *[last[c, w] for w in range(warps) if (c, w) in last])
                for w in range(warps):
                    last[c, w] = ("sync", c, i)
        for c in range(ctas):
            for w in range(warps):
                def then(name, *after):
                    last[c, w] = event(name, *after, *([last[c, w]] if (c, w) in last else []))
                if had:
                    then(("wait", c, w, i - 1), *[("fence", o, i - 1) for o in range(ctas)])
                    then(("read", c, w, i - 1))
                if more and w == 0:
                    for o in range(ctas):
                        then(("write", c, o, i))
                    then(("fence", c, i))
    reach = {}

    def past(e):                                             # everything that happens before e
        if e not in reach:
            reach[e] = set()
            for b in before.get(e, ()):
                reach[e] |= {b} | past(b)
        return reach[e]

    bad = set()
    for i in range(rows):
        for c in range(ctas):
            for o in range(ctas):
                for w in range(warps):
                    read, write = ("read", o, w, i), ("write", c, o, i)
                    if write not in past(read):
                        bad.add((write, read))
                    if i + slots < rows and read not in past(("write", c, o, i + slots)):
                        bad.add((read, ("write", c, o, i + slots)))
    return bad


def test_the_exchange_of_wide_layer_norm_rows_is_ordered():
    import re
    from pathlib import Path
    source = (Path(fm.__file__).parent / "csrc" / "layernorm.cu").read_text()
    found = re.search(r"s_peers\[(\w+)\]\[8\];", source).group(1)
    slots = int(found) if found.isdigit() else int(re.search(rf"{found} = (\d+);", source).group(1))
    assert not _unordered(slots)
    assert _unordered(1) and _unordered(2) and not _unordered(4)


# ------------------------------------------------------------------------------ modules
class _ChannelsFirst(torch.nn.LayerNorm):
    def forward(self, x):
        return super().forward(x.movedim(1, -1)).movedim(-1, 1)


class _Renamed(torch.nn.LayerNorm):
    """No forward of its own."""


def test_layer_norms_with_a_forward_of_their_own_are_left_alone():
    own, plain, renamed, by_hand = _ChannelsFirst(6), torch.nn.LayerNorm(6), _Renamed(6), torch.nn.LayerNorm(6)
    by_hand.forward = lambda x: 2 * torch.nn.LayerNorm.forward(by_hand, x)
    model = torch.nn.ModuleList([own, plain, renamed, by_hand])
    x = _randn(2, 6, 6, 6, seed=5)
    want = [m(x) for m in model]
    K.enable(model, layer_norm=True)
    assert model._fm_fused["layer_norm"] == 2
    for m, y in zip(model, want):
        assert torch.allclose(m(x), y, atol=1e-5)
    for m in (own, by_hand):
        with pytest.raises(TypeError, match="layer_norm"):
            K.patch(m, kind="layer_norm")
        assert not getattr(m, "_fm_norm", False)
    K.revert(model)
    assert torch.equal(plain(x), want[1])


def _rebalance_rank(rank, path):
    import torch.distributed as dist
    torch.set_num_threads(1)
    dist.init_process_group("gloo", init_method=f"file://{path}", rank=rank, world_size=2)
    try:
        torch.manual_seed(8)
        moe = fm.MoE(16, 32, 4, 1, score="sigmoid", balance_bias=True)
        with torch.no_grad():
            moe(_randn(50 + 30 * rank, 16, seed=60 + rank).abs())
        router, own = moe.router, moe.router.last_counts.float()
        with pytest.raises(ValueError, match="several ranks"):
            router.rebalance(0.1)
        assert not router.bias.any()
        router.rebalance(0.1, dist.group.WORLD)
        total = own.clone()
        dist.all_reduce(total)
        assert torch.allclose(router.bias, 0.1 * torch.sign(total.mean() - total))
        router.bias.zero_()
        router.rebalance(0.1, "self")
        assert torch.allclose(router.bias, 0.1 * torch.sign(own.mean() - own))
    finally:
        dist.destroy_process_group()


def test_rebalance_of_several_ranks_needs_a_group(tmp_path):
    torch.multiprocessing.spawn(_rebalance_rank, args=(str(tmp_path / "store"),), nprocs=2)


# ------------------------------------------------------------------------------ tensors that are not the memory they seem to be
def _no_memory():
    """A wrapper subclass like DTensor, whose pointer is null; a lazily negated view; a sparse tensor."""
    class Wrapper(torch.Tensor):
        @staticmethod
        def __new__(cls, inner):
            return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            raise NotImplementedError(str(func))
    return [Wrapper(torch.ones(3, 8)), torch.imag(torch.ones(3, 8, dtype=torch.complex64).conj()), torch.eye(3, 8).to_sparse()]


def test_the_kernels_refuse_tensors_that_are_not_plain_memory():
    """The extension's own functions, before they look at anything else (so this needs no GPU)."""
    ext = pytest.importorskip("forgeminds_b200._C")
    x, v = torch.ones(3, 8), torch.ones(8)
    q, i = torch.ones(1, 3, 2, 4), torch.zeros(3, 8, dtype=torch.int64)
    for bad in _no_memory():
        calls = [lambda: ext.layer_norm(bad, v, v, 1e-5), lambda: ext.layer_norm(x, bad, v, 1e-5), lambda: ext.layer_norm(x, v, bad, 1e-5),
                 lambda: ext.add_layer_norm(x, bad, None, None, 1e-5), lambda: ext.rotary_one(bad, x, x, None, False),
                 lambda: ext.rotary_qk(q, bad, x, x, None, False), lambda: ext.rotary_one(q, bad, x, None, False),
                 lambda: ext.rotary_one(q, x, bad, None, False), lambda: ext.rotary_one(q, x, x, bad, False),
                 lambda: ext.kl_topk(bad, x, i, None, 1.0, 0), lambda: ext.kl_topk(x, bad, i, None, 1.0, 0),
                 lambda: ext.kl_topk(x, x, bad, None, 1.0, 0), lambda: ext.kl_topk(x, x, i, bad, 1.0, 0),
                 lambda: ext.kl_topk_fwd(x, bad, i, None, 1.0, True, True, None, True, False),
                 lambda: ext.route(bad, None, 2, True, 1, 1, 2, True, 1.0, 0.0, 0.0),
                 lambda: ext.route(x, bad, 2, True, 1, 1, 2, True, 1.0, 0.0, 0.0)]
        for call in calls:
            with pytest.raises(TypeError, match="plain strided"):
                call()
    with pytest.raises(TypeError, match="plain strided"):
        torch.func.vmap(lambda t: ext.layer_norm(t, v, v, 1e-5))(torch.ones(2, 3, 8))


def test_wrappers_are_seen_before_a_kernel_is_chosen():
    from forgeminds_b200.kernels import _state

    class Plain(torch.Tensor):
        pass
    wrapper = _no_memory()[0]
    assert _state._wrapper(wrapper) and not _state._wrapper(torch.ones(2)) and not _state._wrapper(torch.nn.Parameter(torch.ones(2)))
    assert not _state._wrapper(torch.ones(2).as_subclass(Plain))
