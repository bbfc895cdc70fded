"""Attention over packed sequences on the GPU: calls at the edges of what it takes."""
import pytest
import torch

from cppmega_b200.ops import functional as F_

pytestmark = pytest.mark.gpu


def _randn(*shape, dtype=torch.bfloat16, std=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 7919 * sum(shape))
    return torch.empty(shape, device="cuda").normal_(0.0, std, generator=g).to(dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_batched_upstream_gradients(dtype):
    """A batch of upstream gradients, which the definition takes, against the kernels one at a time.  Both are off by roundings that are independent from
    element to element: the result's on either side, ds (p) of the kernels.  Together less than twice half a step of the norm; four times that is allowed."""
    cu = _i32([0, 60, 90])
    leaves = [_randn(90, n, 64, dtype=dtype, seed=s).requires_grad_() for s, n in ((0, 4), (1, 2), (2, 2))]
    go = _randn(3, 90, 4, 64, dtype=dtype, seed=3)
    F_.reset_counters()
    o = F_.packed_attention(*leaves, cu, 0.125)
    got = torch.autograd.grad(o, leaves, go, is_grads_batched=True, retain_graph=True)
    assert F_.fallback_counts() == {"packed_attention_bwd(batched gradients)": 1}
    for i in range(3):
        for a, b in zip(got, torch.autograd.grad(o, leaves, go[i], retain_graph=True)):
            a, b = a[i].double(), b.double()
            assert (a - b).norm() <= 8 * torch.finfo(dtype).eps / 2 * b.norm()


NOTHING = [(0, 0, 2, 2), (0, 7, 2, 2), (7, 0, 4, 2), (7, 7, 0, 2)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,Tk,H,G", NOTHING)
def test_calls_of_nothing_wait_for_nothing(T, Tk, H, G, dtype):
    """No rows of queries, of keys, or no heads: zeros, and gradients of zeros, also in a captured graph, whose ends change in place."""
    leaves = [_randn(n, h, 64, dtype=dtype, seed=s).requires_grad_() for s, n, h in ((0, T, H), (1, Tk, G), (2, Tk, G))]
    cu, cu_k = _i32([0, T // 2, T]), _i32([0, Tk, Tk])

    def once():
        o = F_.packed_attention(*leaves, cu, -0.125, cu_k)
        return [o.detach(), *torch.autograd.grad(o, leaves, torch.ones_like(o))]

    F_.reset_counters()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = once()
    torch.cuda.current_stream().wait_stream(side)
    assert F_.launch_counts() == {"packed_attention": 1} and not F_.fallback_counts()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = once()
    g.replay()
    from cppmega_b200.ops import cuda as cu_
    cu_.check_errors()
    for outs in (eager, captured):
        assert outs[0].shape == (T, H, 64) and outs[0].dtype == dtype
        assert all(a.shape == b.shape and (a == 0).all() for a, b in zip(outs[1:], leaves)) and (outs[0] == 0).all()
    for ends, ends_k in (([0, T // 2, T + 1], [0, 0, Tk]), ([0, 0, T], [1, 1, 1]), ([0, -1, 0], [0, 0, 0]), ([0, 0, 0], [0, 5, 4])):
        cu.copy_(_i32(ends))
        cu_k.copy_(_i32(ends_k))
        g.replay()
        with pytest.raises(cu_.KernelError, match="bad argument"):
            cu_.check_errors()


def test_calls_of_nothing_can_be_differentiated_again():
    leaves = [_randn(n, 2, 64, seed=s).requires_grad_() for s, n in ((0, 5), (1, 0), (2, 0))]
    o = F_.packed_attention(*leaves, _i32([0, 5]), 0.1, _i32([0, 0]))
    (g,) = torch.autograd.grad(o.sum() + leaves[0].square().sum(), leaves[0], create_graph=True)
    assert torch.equal(torch.autograd.grad(g.sum(), leaves[0])[0], torch.full_like(leaves[0], 2))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("wanted,kernels", [([0], 1), ([1], 1), ([2], 1), ([1, 2], 1), ([0, 1], 2), ([0, 2], 2), ([0, 1, 2], 2)])
def test_gradients_that_nobody_asks_for_are_not_computed(wanted, kernels, dtype):
    """One large kernel for dq, one for dk and dv; the gradients that are asked for have the same bits."""
    cu = _i32([0, 60, 190])
    leaves = [_randn(190, n, 64, dtype=dtype, seed=s) for s, n in ((0, 4), (1, 2), (2, 2))]
    go = _randn(190, 4, 64, dtype=dtype, seed=3)
    every = [t.clone().requires_grad_() for t in leaves]
    want = torch.autograd.grad(F_.packed_attention(*every, cu, 0.125), every, go)
    some = [t.clone().requires_grad_(i in wanted) for i, t in enumerate(leaves)]
    F_.reset_counters()
    got = torch.autograd.grad(F_.packed_attention(*some, cu, 0.125), [some[i] for i in wanted], go)
    assert all(torch.equal(a, want[i]) for a, i in zip(got, wanted))
    assert F_.launch_counts()["packed_attention_bwd"] == kernels + (1 if dtype == torch.bfloat16 else 2)
