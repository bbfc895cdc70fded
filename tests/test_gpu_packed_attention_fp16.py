"""fp16 gradients of the attention over packed sequences where the range of the type is short: documents and heads with gradients of very
different sizes side by side, long rows, and values far below and far above one.

Tolerances from the exact values, with u = 2^-11, half a step, and e the error of a weight's exponent, twice the error of a score (its fp32 sum over
D products, D 2^-23 of their magnitudes in any order, and roundings of scale and maximum).  A weight p is off by p (u + e) in the result, and in the
gradient of the values by that and what the range loses; delta and dP by the result's error and fp32 sums over the value columns; ds by its rounding
u, by the errors of p and of dP - delta, and by what the range loses; a gradient by its operands' errors, its fp32 sum and its own rounding.
Lost is half of fp16's smallest step, 2^-25, under the powers that the operands are scaled by: 2^-39 of a weight, and 2^-37 |do| max |v| of a ds (Euclidean
norms: the row's own |do| in dq, the largest of the sequence and key head in dk).
"""
import math

import pytest
import torch

from cppmega_b200.ops import functional as F_

pytestmark = pytest.mark.gpu

U = 2.0 ** -11


def _randn(*shape, std=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 7919 * sum(shape))
    return torch.empty(shape, device="cuda").normal_(0.0, std, generator=g).half()


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _gradients(q, k, v, go, ends, scale, ends_k=None):
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    o = F_.packed_attention(*leaves, _i32(ends), scale, None if ends_k is None else _i32(ends_k))
    return [o.detach(), *torch.autograd.grad(o, leaves, go)]


def _check(got, want, bound, name):
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), (name, int(bad.sum()), float(((got.double() - want).abs() / bound)[bad].max()))


def _compare(q, k, v, go, scale, grads):
    """One sequence, one key head."""
    L, Lk, D, V = q.shape[0], k.shape[0], q.shape[2], v.shape[2]
    tiny = 2.0 ** -25
    kh, vh = k[:, 0].double(), v[:, 0].double()
    hidden = torch.ones(L, Lk, dtype=torch.bool, device="cuda").triu(Lk - L + 1)
    far = float(go.double().norm(dim=2).amax() * vh.norm(dim=1).amax())
    dk, dv, bk, bv = (torch.zeros_like(t) for t in (kh, vh, kh, vh))
    n = L * q.shape[1]
    for h in range(q.shape[1]):
        qh, g = q[:, h].double(), go[:, h].double()
        p = torch.softmax((qh @ kh.T * scale).masked_fill(hidden, -math.inf), 1)
        mags = (qh.abs() @ kh.abs().T * scale).masked_fill(hidden, 0.0)
        e = 2 * (((D + 8) * 2.0 ** -23) * mags).amax(1, keepdim=True) + 2.0 ** -19 + Lk * 2.0 ** -23
        out = p @ vh
        eo = 2 * (p * (U + e) + 2.0 ** -17 * p.amax(1, keepdim=True) * (p > 0)) @ vh.abs() + U * out.abs() * 2.0 ** -10 + 2.0 ** -25
        dp = g @ vh.T
        delta = (g * out).sum(1, keepdim=True)
        e_x = (V + 8) * 2.0 ** -23 * (g.abs() @ vh.abs().T) + (g.abs() * eo).sum(1, keepdim=True) + (V + 8) * 2.0 ** -23 * (g * out).abs().sum(1, keepdim=True)
        ds = p * (dp - delta)
        exact = p * e * (dp - delta).abs() + p * e_x
        lost_q = 2.0 ** -37 * g.norm(dim=1, keepdim=True) * vh.norm(dim=1).amax()
        dq = ds @ kh * scale
        eq = (U * ds.abs() + (1 + U) * exact + lost_q * (p > 0) + Lk * 2.0 ** -24 * ds.abs()) * scale
        _check(grads[0][:, h], dq, (eq @ kh.abs()) * (1 + U) + U * dq.abs() + tiny, "dq")
        ek = (U * ds.abs() + (1 + U) * exact + 2.0 ** -37 * far * (p > 0) + n * 2.0 ** -24 * ds.abs()) * scale
        dk += ds.T @ qh * scale
        bk += ek.T @ qh.abs()
        dv += p.T @ g
        bv += (p * (U + e) + 2.0 ** -39 * (p > 0) + n * 2.0 ** -24 * p).T @ g.abs()
    _check(grads[1][:, 0], dk, bk * (1 + U) + U * dk.abs() + tiny, "dk")
    _check(grads[2][:, 0], dv, bv * (1 + U) + U * dv.abs() + tiny, "dv")


@pytest.mark.parametrize("ratio", [1e3, 1e5])
@pytest.mark.parametrize("D,V", [(128, 128), (128, 64), (64, 64)])
def test_documents_and_heads_with_gradients_of_different_sizes(D, V, ratio):
    """Powers of two alone tell a document (and a key head) beside others with larger gradients and values from the same one by itself: the same bits."""
    ends, H, G = [0, 500, 800, 1300], 4, 2                    # 512 keys at most: no row is shared out among blocks
    q, k, v = _randn(1300, H, D), _randn(1300, G, D, seed=1), _randn(1300, G, V, seed=2)
    go = _randn(1300, H, V, std=0.1, seed=3)
    go[500:800] = (go[500:800].float() * ratio).clamp(-6e4, 6e4).half()
    go[800:, :2] *= 300
    v[800:, 0] *= 100
    whole = _gradients(q, k, v, go, ends, D ** -0.5)
    for a, b in zip(ends, ends[1:]):
        for g in range(G):
            h = slice(2 * g, 2 * g + 2)
            one = _gradients(q[a:b, h], k[a:b, g:g + 1], v[a:b, g:g + 1], go[a:b, h], [0, b - a], D ** -0.5)
            for x, y, heads in zip(whole, one, (h, h, slice(g, g + 1), slice(g, g + 1))):
                assert torch.equal(x[a:b, heads], y)


@pytest.mark.parametrize("v_std", [2e-3, 1.0, 3e3])
@pytest.mark.parametrize("go_std", [1e-3, 30.0])
def test_long_rows_and_values_of_any_size(v_std, go_std):
    """Weights of some 2^-12, whose ds would be below the range with values far below one, or above it far above."""
    if v_std * go_std > 1e4:
        go_std = 0.3
    q, k, v = _randn(2400, 2, 64), _randn(2400, 1, 64, seed=1), _randn(2400, 1, 64, std=v_std, seed=2)
    go = _randn(2400, 2, 64, std=go_std, seed=3)
    _compare(q, k, v, go, 0.125, _gradients(q, k, v, go, [0, 2400], 0.125)[1:])


def test_values_that_add_up_to_the_largest_products():
    """do v' of 128 columns of one sign and 2e4 each, the other sign at every other key."""
    q, k = _randn(200, 1, 128, std=0.3), _randn(200, 1, 128, std=0.3, seed=1)
    v = (2e4 * (1 - 2 * (torch.arange(200, device="cuda") % 2)))[:, None, None].expand(200, 1, 128).half()
    go = torch.full((200, 1, 128), 1e-3, device="cuda").half()
    grads = _gradients(q, k, v, go, [0, 200], 0.1)[1:]
    assert all(g.isfinite().all() for g in grads)
    _compare(q, k, v, go, 0.1, grads)


@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_rows_that_are_not_finite_set_no_scale(value):
    """An upstream row or a value row that is not finite reaches the gradients of its own sequence and key head alone."""
    q, k, v = _randn(300, 2, 64), _randn(300, 2, 64, seed=1), _randn(300, 2, 64, seed=2)
    go = _randn(300, 2, 64, seed=3)
    base = _gradients(q, k, v, go, [0, 130, 300], 0.125)
    v2, go2 = v.clone(), go.clone()
    go2[7, 0, 5] = value
    v2[200, 1, 9] = value
    got = _gradients(q, k, v2, go2, [0, 130, 300], 0.125)
    for a, b in zip(base, got):
        assert torch.equal(a[:130, 1], b[:130, 1]) and torch.equal(a[130:, 0], b[130:, 0])
    assert got[1][7, 0].isnan().any() and torch.equal(got[1][8:130, 0], base[1][8:130, 0])


def test_no_sequences_and_empty_ones():
    for ends, ends_k in (([0], [0]), ([0, 0, 0], [0, 0, 0]), ([0, 0, 40, 40], [0, 30, 30, 40]), ([0, 40, 40], [0, 0, 40])):
        q, k, v, go = (_randn(40, 2, 64, seed=s) for s in range(4))
        grads = _gradients(q, k, v, go, ends, 0.125, ends_k)
        assert all((g == 0).all() for g in grads)
    from cppmega_b200.ops import cuda as cu_
    cu_.check_errors()


def test_keys_far_below_one_without_values():
    """Weights that one key (its values zero) pushes 10 to 17 below it, the same for all the others, so that their roundings add up: 2^-11 of each, and
    2^-25 under the 2^7 that the largest counts at the least."""
    n, D = 300, 64
    q, k = torch.zeros(n, 1, D, device="cuda").half(), torch.zeros(n, 1, D, device="cuda").half()
    q[:, 0, 0] = torch.linspace(10, 17, n, device="cuda")
    k[0, 0, 0] = 1
    v = torch.full((n, 1, D), 8.0, device="cuda").half()
    v[0] = 0
    o = F_.packed_attention(q, k, v, _i32([0, n]), 1.0)[:, 0].double()
    s = (q[:, 0].double() @ k[:, 0].double().T).masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -math.inf)
    p = torch.softmax(s, 1)
    e = 2 * ((D + 8) * 2.0 ** -23) * s.masked_fill(s == -math.inf, 0).abs().amax(1, keepdim=True) + 2.0 ** -19 + n * 2.0 ** -23
    want = p @ v[:, 0].double()
    bound = (p * (U + e) + 2.0 ** -32 * (p > 0)) @ v[:, 0].double() + want * (U + e + U) + 2.0 ** -25
    _check(o, want, bound * (1 + U), "o")


def test_captured_for_other_lengths_and_sizes():
    """Forward and backward in a graph: the ends and the upstream gradients change in place, and with them the scales of each sequence."""
    cu = _i32([0, 100, 200, 256])
    q, k, v = (_randn(256, n, 64, seed=s).requires_grad_() for s, n in ((0, 4), (1, 2), (2, 2)))
    go = _randn(256, 4, 64, seed=3)

    def once():
        o = F_.packed_attention(q, k, v, cu, 0.125)
        return [o.detach(), *torch.autograd.grad(o, [q, k, v], go)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = once()
    for ends, std in (([0, 100, 200, 256], 1.0), ([0, 1, 1, 250], 1e3), ([0, 256, 256, 256], 1e-3), ([0, 0, 0, 0], 1.0), ([0, 130, 131, 200], 1e-2)):
        cu.copy_(_i32(ends))
        go.copy_(_randn(256, 4, 64, std=std, seed=ends[1]))
        g.replay()
        got = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, once()))
