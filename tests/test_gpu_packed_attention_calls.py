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
