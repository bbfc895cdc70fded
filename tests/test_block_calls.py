"""The operators around a dense block, on the CPU: calls that reach them in less usual ways."""
import pytest
import torch
from torch.autograd import forward_ad

from cppmega_b200.ops import functional as F_
from cppmega_b200.ops import reference as ref
from cppmega_b200.ops.cuda import block


def _r(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + sum(shape))).to(dtype)


def _block_calls():
    """name -> (wrapper around the kernel, its tensors)"""
    bf = torch.bfloat16
    return {
        "rmsnorm_gated": (lambda x, w, z: block.rmsnorm_gated(x, w, z, 1e-5, 16, True), [_r(4, 16), _r(16), _r(4, 16, seed=1)]),
        "residual_rmsnorm": (lambda y, x, w, p, g: block.residual_rmsnorm(y, x, w, p, g, 1.0, 1e-5),
                             [_r(4, 16), _r(4, 16, seed=1), _r(16), _r(16, seed=2), _r(16, seed=3)]),
        "gated_mlp": (lambda x, w1, w2: block.gated_mlp(x, w1, w2, "silu"), [_r(4, 16, dtype=bf), _r(48, 16, dtype=bf), _r(16, 24, dtype=bf)]),
    }


@pytest.mark.parametrize("name,i", [(n, i) for n, (_, a) in _block_calls().items() for i in range(len(a))])
def test_kernels_leave_tangents_and_transforms_to_the_definitions(name, i):
    """A kernel reads memory: it would drop a forward-mode tangent, and under a function transform there is no memory to read."""
    call, args = _block_calls()[name]
    with forward_ad.dual_level():
        dual = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
        assert call(*dual) is None
    seen = []

    def inside(t):
        seen.append(call(*[t if j == i else a for j, a in enumerate(args)]))
        return t.sum()

    torch.func.grad(inside)(args[i])
    torch.func.vmap(inside)(args[i].expand(3, *args[i].shape))
    assert seen == [None, None]


@pytest.mark.parametrize("before", [True, False])
@pytest.mark.parametrize("gate", [True, False])
def test_gated_norm_takes_a_batch_of_upstream_gradients(monkeypatch, before, gate):
    """``is_grads_batched`` hands the backward gradients that have no memory a kernel could read."""
    x, w, z = (t.requires_grad_() for t in (_r(5, 24), _r(24), _r(5, 24, seed=1)))

    def forward(x, weight, z, eps, group, gate_first, keep):
        return ref.rmsnorm_gated(x, weight, z, eps, group, not gate_first), x, z, torch.empty(0)

    monkeypatch.setattr(block, "_gated_forward", forward)
    ins = [x, w, z] if gate else [x, w]
    many = _r(3, 5, 24, seed=2)
    got = torch.autograd.grad(block.rmsnorm_gated(x, w, z if gate else None, 1e-5, 8, before), ins, many, is_grads_batched=True)
    y = ref.rmsnorm_gated(x, w, z if gate else None, 1e-5, 8, before)
    for i, dy in enumerate(many):
        want = torch.autograd.grad(y, ins, dy, retain_graph=True)
        assert all(torch.allclose(g[i], t, rtol=1e-5, atol=1e-6) for g, t in zip(got, want))
