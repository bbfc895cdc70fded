"""Attention over packed sequences on the GPU, with its gradients, against 64 bits.

Tolerances from the exact values, with u half a step of the type (2^-8 in bf16, 2^-11 in fp16) and e the error of a weight's exponent, twice the
error of a score (its fp32 sum over D products, D 2^-23 of their magnitudes in any order, and roundings of scale and maximum): a weight p is off
by p (u + e); o, whose sum of weights has the largest of every 64 keys as rounded, by p |v - o| (u + e) for those and p |v| (u + e) for the others,
at most (|p||v| + |o|) (u + e), and its own rounding; delta and dP by fp32 sums over the value columns of do, v and o as rounded; ds by
its rounding u and by the errors of p and of dP - delta; a gradient by its operands' errors, its fp32 sum and its own rounding.  In fp16 what is
below the range is lost: 2^-25 of a weight of up to 2^8, and of ds scaled so that |do| is at most 2^-4.
"""
import math

import pytest
import torch

from cppmega_b200.ops import functional as F_

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _randn(*shape, dtype=torch.bfloat16, std=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 7919 * sum(shape))
    return torch.empty(shape, device="cuda").normal_(0.0, std, generator=g).to(dtype)


def _ends(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _check(got, want, bound, name):
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), (name, int(bad.sum()), float(((got.double() - want).abs() / bound)[bad].max()), bad.nonzero()[0].tolist())


def _compare(q, k, v, ends, ends_k, scale, o, go=None, grads=None):
    """Every sequence and head by itself, with the bounds above."""
    dt = q.dtype
    u, D, V = HALF_STEP[dt], q.shape[2], v.shape[2]
    group = q.shape[1] // k.shape[1]
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    fp16 = dt == torch.float16
    dk, dv = (torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (k, v))
    bk, bv = dk.clone(), dv.clone()
    top = go[:ends[-1]].double().abs().max() if go is not None and ends[-1] else None
    for a, b, c, d in zip(ends, ends[1:], ends_k, ends_k[1:]):
        if a == b or c == d:
            assert (o[a:b] == 0).all() and (grads is None or (grads[0][a:b] == 0).all())
            continue
        L, Lk = b - a, d - c
        hidden = torch.ones(L, Lk, dtype=torch.bool, device="cuda").triu(Lk - L + 1)
        for h in range(q.shape[1]):
            qh, kh, vh = q[a:b, h].double(), k[c:d, h // group].double(), v[c:d, h // group].double()
            s = (qh @ kh.T * scale).masked_fill(hidden, -math.inf)
            p = torch.softmax(s, 1).nan_to_num(0.0)
            mags = (qh.abs() @ kh.abs().T * abs(scale)).masked_fill(hidden, 0.0)
            e = 2 * (((D + 8) * 2.0 ** -23) * mags).amax(1, keepdim=True) + 2.0 ** -19 + Lk * 2.0 ** -23
            lost = 2.0 ** -17 * p.amax(1, keepdim=True) * (p > 0) if fp16 else 0.0
            ep = p * (u + e) + lost
            out, eo = p @ vh, ep @ vh.abs()
            _check(o[a:b, h], out, (eo + ep.sum(1, keepdim=True) * out.abs()) * (1 + u) + u * out.abs() + tiny, "o")
            if go is None:
                continue
            g = go[a:b, h].double()
            dp = g @ vh.T
            e_dp = (V + 8) * 2.0 ** -23 * (g.abs() @ vh.abs().T)
            oh = o[a:b, h].double()
            delta = (g * out).sum(1, keepdim=True)
            e_delta = (g.abs() * (oh - out).abs()).sum(1, keepdim=True) + (V + 8) * 2.0 ** -23 * (g * oh).abs().sum(1, keepdim=True)
            x = dp - delta
            ds = p * x
            exact = p * e * x.abs() + p * (e_dp + e_delta)                  # p in fp32 here
            lost_q = 2.0 ** -21 * g.abs().amax(1, keepdim=True) * (p > 0) if fp16 else 0.0
            lost_k = 2.0 ** -20 * top * (p > 0) if fp16 else 0.0
            eq = (u * ds.abs() + (1 + u) * exact + lost_q + Lk * 2.0 ** -24 * ds.abs()) * abs(scale)
            dq = ds @ kh * scale
            _check(grads[0][a:b, h], dq, (eq @ kh.abs()) * (1 + u) + u * dq.abs() + tiny, "dq")
            n = L * group
            ek = (u * ds.abs() + (1 + u) * exact + lost_k + n * 2.0 ** -24 * ds.abs()) * abs(scale)
            dk[c:d, h // group] += ds.T @ qh * scale
            bk[c:d, h // group] += ek.T @ qh.abs()
            dv[c:d, h // group] += p.T @ g
            bv[c:d, h // group] += (ep + n * 2.0 ** -24 * p).T @ g.abs()
    if go is not None:
        _check(grads[1], dk, bk * (1 + u) + u * dk.abs() + tiny, "dk")
        _check(grads[2], dv, bv * (1 + u) + u * dv.abs() + tiny, "dv")
    assert (o[ends[-1]:] == 0).all()
    if grads is not None:
        assert (grads[0][ends[-1]:] == 0).all() and all((g[ends_k[-1]:] == 0).all() for g in grads[1:])


def _run(lens, H, G, D, V, dtype, lens_k=None, tail=0, train=True, scale=None, std=1.0, tail_value=math.nan):
    ends, ends_k = _ends(lens), _ends(lens if lens_k is None else lens_k)
    T, Tk = ends[-1] + tail, ends_k[-1] + tail
    q, k, v = _randn(T, H, D, dtype=dtype, std=std), _randn(Tk, G, D, dtype=dtype, seed=1), _randn(Tk, G, V, dtype=dtype, seed=2)
    go = _randn(T, H, V, dtype=dtype, std=0.1, seed=3)
    for t, n in ((q, ends[-1]), (k, ends_k[-1]), (v, ends_k[-1]), (go, ends[-1])):
        t[n:] = tail_value
    scale = D ** -0.5 if scale is None else scale
    cu, cu_k = _i32(ends), None if lens_k is None else _i32(ends_k)
    F_.reset_counters()
    if not train:
        o = F_.packed_attention(q, k, v, cu, scale, cu_k)
        _compare(q, k, v, ends, ends_k, scale, o)
    else:
        leaves = [t.requires_grad_() for t in (q, k, v)]
        o = F_.packed_attention(*leaves, cu, scale, cu_k)
        grads = torch.autograd.grad(o, leaves, go)
        with torch.no_grad():
            assert torch.equal(F_.packed_attention(q, k, v, cu, scale, cu_k), o)
            _compare(q.detach(), k.detach(), v.detach(), ends, ends_k, scale, o.detach(), go, grads)
    assert not F_.fallback_counts()
    from cppmega_b200.ops import cuda as cu_
    cu_.check_errors()


DTYPES = [torch.bfloat16, torch.float16]
WIDTHS = [(128, 128), (128, 64), (64, 64), (64, 128), (96, 80), (8, 16)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,V", WIDTHS)
@pytest.mark.parametrize("lens", [[1], [128], [127, 129], [5, 0, 300, 64, 1, 0], [256, 255, 257], [700, 33]])
def test_one_head(lens, D, V, dtype):
    _run(lens, 1, 1, D, V, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,V", [(128, 128), (64, 64)])
def test_rows_that_settle_on_few_keys(D, V, dtype):
    """o = sum p (1 + d) v / sum p (1 + d'), |d| <= u + e, where d' is d for the largest weight of every 64 keys and without u for the others, is off by at most
    the sum of p |v - o| (u + e) over those and of p (|v| u + |v - o| e) over the others, each over 1 - u - e, and its rounding: nearly nothing but the rounding
    where one weight is nearly all of a row, although that weight is no power of two while the maximum lags."""
    L, u = 400, HALF_STEP[dtype]
    q, k, v = _randn(L, 1, D, dtype=dtype, std=1.5), _randn(L, 1, D, dtype=dtype, seed=1), _randn(L, 1, V, dtype=dtype, seed=2)
    k[70::100] *= 4
    o = F_.packed_attention(q, k, v, _i32([0, L]), D ** -0.5)[:, 0].double()
    qh, kh, vh = q[:, 0].double(), k[:, 0].double(), v[:, 0].double()
    hidden = torch.ones(L, L, dtype=torch.bool, device="cuda").triu(1)
    p = torch.softmax((qh @ kh.T * D ** -0.5).masked_fill(hidden, -math.inf), 1)
    assert (p.amax(1) > 0.99).sum() > 10
    mags = (qh.abs() @ kh.abs().T * D ** -0.5).masked_fill(hidden, 0.0)
    e = 2 * (((D + 8) * 2.0 ** -23) * mags).amax(1, keepdim=True) + 2.0 ** -19 + L * 2.0 ** -23
    out = p @ vh
    parts = torch.nn.functional.pad(p, (0, -L % 64)).view(L, -1, 64)
    largest = (parts == parts.amax(2, keepdim=True)).view(L, -1)[:, :L]
    away = (vh[None] - out[:, None]).abs()
    spread = (p[:, :, None] * torch.where(largest[:, :, None], away, torch.maximum(away, vh.abs()[None]))).sum(1)
    lost = 2.0 ** -17 * p.amax(1, keepdim=True) * vh.abs().sum(0, keepdim=True) if dtype == torch.float16 else 0.0
    _check(o, out, spread * (u + e) / (1 - u - e) + lost + u * out.abs() * (1 + u) + 2.0 ** -24 * L * (p @ vh.abs()), "o")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,G", [(8, 8), (8, 2), (14, 2), (12, 4), (16, 1), (96, 1), (130, 1), (33, 3), (128, 1)])
@pytest.mark.parametrize("D,V", [(128, 128), (128, 64)])
def test_grouped_heads(H, G, D, V, dtype):
    _run([67, 1, 150, 18], H, G, D, V, dtype, tail=3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,V", [(128, 128), (64, 64)])
@pytest.mark.parametrize("lens,lens_k", [([100, 1, 40], [300, 129, 40]), ([5, 200, 3], [0, 70, 1000]), ([0, 130, 1], [60, 1, 513]), ([128], [4000])])
def test_keys_with_their_own_ends(lens, lens_k, D, V, dtype):
    """Keys from before, fewer keys than queries (queries that see nothing), no keys, no queries."""
    _run(lens, 6, 2, D, V, dtype, lens_k=lens_k, tail=2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,V", [(128, 128), (96, 48), (64, 64)])
@pytest.mark.parametrize("lens,lens_k,H,G", [
    ([64], [5000], 8, 2), ([1], [3001], 4, 1), ([3, 33, 1, 70], [4000, 33, 0, 640], 4, 2), ([200], [1100], 3, 1), ([2, 0, 300], [1, 50, 2500], 1, 1),
    ([900], [900], 2, 1),
])
def test_few_rows_on_many_keys(lens, lens_k, H, G, D, V, dtype):
    """Keys shared out among blocks: shares that end inside a tile's mask, that some rows do not reach, sequences too short to be shared."""
    _run(lens, H, G, D, V, dtype, lens_k=lens_k, tail=2, train=lens[0] != 64)


def test_few_rows_on_many_keys_captured():
    """The same graph for lengths that are shared out and for lengths that are not."""
    q, k, v = (_randn(n, h, 64, seed=s) for s, n, h in ((0, 40, 4), (1, 3000, 2), (2, 3000, 2)))
    cu, cu_k = _i32([0, 20, 40]), _i32([0, 1500, 3000])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        F_.packed_attention(q, k, v, cu, 0.125, cu_k)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = F_.packed_attention(q, k, v, cu, 0.125, cu_k)
    for ends, ends_k in (([0, 20, 40], [0, 1500, 3000]), ([0, 1, 40], [0, 2990, 3000]), ([0, 40, 40], [0, 100, 100]), ([0, 0, 7], [0, 2000, 2700])):
        cu.copy_(_i32(ends))
        cu_k.copy_(_i32(ends_k))
        g.replay()
        _compare(q, k, v, ends, ends_k, 0.125, o.clone())


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_sequences(dtype):
    _run([2500, 1300], 4, 2, 128, 128, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_sequences(dtype):
    _run([(7 * i) % 41 for i in range(700)] + [600], 2, 1, 64, 64, dtype, tail=100)


@pytest.mark.parametrize("tail_value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D,V", [(128, 128), (128, 64), (64, 64)])
def test_rows_behind_the_last_sequence_do_not_matter(D, V, tail_value):
    _run([70, 200], 6, 2, D, V, torch.bfloat16, tail=500, tail_value=tail_value)


@pytest.mark.parametrize("D,V", [(128, 128), (128, 64), (64, 64)])
def test_a_sequence_of_nan_leaves_the_others_alone(D, V):
    """The sequences before and behind one that is not finite, in tiles that reach into it, are as without it, bit for bit."""
    ends, cu = [0, 77, 77 + 133, 400], _i32([0, 77, 210, 400])
    make = lambda n, s: _randn(400, n, D if s < 2 else V, seed=s)  # noqa: E731
    q, k, v, go = make(6, 0), make(2, 1), make(2, 2), make(6, 3)
    results = []
    for value in (None, math.nan, math.inf):
        args = [t.clone() for t in (q, k, v, go)]
        if value is not None:
            for t in args:
                t[77:210] = value
        leaves = [t.requires_grad_() for t in args[:3]]
        o = F_.packed_attention(*leaves, cu, 0.1)
        results.append([o.detach(), *torch.autograd.grad(o, leaves, args[3])])
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.equal(a[:77], b[:77]) and torch.equal(a[210:], b[210:])
    assert ends[-1] == 400


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale,std", [(-0.2, 1.0), (0.0, 1.0), (1.0, 3.0), (1e-4, 1.0)])
def test_scales(scale, std, dtype):
    _run([200, 50], 4, 2, 64, 64, dtype, scale=scale, std=std)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_inputs_are_read_where_they_are(dtype):
    """Heads of one projection, a layout with the heads outside, and a broadcast upstream gradient."""
    cu = _i32([0, 100, 130])
    qkv = _randn(130, 12, 64, dtype=dtype).requires_grad_()
    outer = _randn(2, 130, 72, dtype=dtype, seed=1)[..., :64].transpose(0, 1)
    o = F_.packed_attention(qkv[:, :8], qkv[:, 8:10], outer, cu, 0.125)
    (g,) = torch.autograd.grad(o.sum(), qkv)
    q, k = qkv.detach()[:, :8].contiguous().requires_grad_(), qkv.detach()[:, 8:10].contiguous().requires_grad_()
    o2 = F_.packed_attention(q, k, outer.contiguous(), cu, 0.125)
    gq, gk = torch.autograd.grad(o2, [q, k], torch.ones_like(o2))
    assert torch.equal(o, o2) and torch.equal(g[:, :8], gq) and torch.equal(g[:, 8:10], gk) and (g[:, 10:] == 0).all()


def test_broadcast_and_misaligned_inputs():
    """One key head given for four by expand, and rows off the 16-byte grid: copied, with the gradients of the originals."""
    cu = _i32([0, 60, 90])
    q = _randn(90, 4, 65).requires_grad_()
    k1, v1 = _randn(90, 1, 64, seed=1).requires_grad_(), _randn(90, 1, 64, seed=2).requires_grad_()
    go = _randn(90, 4, 64, seed=3)
    got = torch.autograd.grad(F_.packed_attention(q[..., 1:], k1.expand(90, 4, 64), v1.expand(90, 4, 64), cu, 0.1), [q, k1, v1], go)
    want = torch.autograd.grad(F_.packed_attention(q[..., 1:].contiguous(), k1, v1, cu, 0.1), [q, k1, v1], go)
    assert torch.equal(got[0], want[0])
    for a, b in zip(got[1:], want[1:]):                       # four gradients rounded and added in bf16: 2^-8 of each and of each sum
        assert ((a.double() - b.double()).abs() <= 8 * 2.0 ** -8 * b.double().abs().max()).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_are_those_of_differences(dtype):
    """The loss over a small step along a direction, in 64 bits on the CPU, against the gradients' product with it."""
    ends = [0, 9, 30]
    cu = _i32(ends)
    leaves = [_randn(30, n, 16, dtype=dtype, seed=s).requires_grad_() for s, n in ((0, 4), (1, 2), (2, 2))]
    go = _randn(30, 4, 16, dtype=dtype, seed=3)
    grads = torch.autograd.grad(F_.packed_attention(*leaves, cu, 0.25), leaves, go)

    def loss(q, k, v):
        total = 0.0
        for a, b in zip(ends, ends[1:]):
            for h in range(4):
                s = q[a:b, h] @ k[a:b, h // 2].T * 0.25
                s = s.masked_fill(torch.ones(b - a, b - a, dtype=torch.bool).triu(1), -math.inf)
                total = total + (torch.softmax(s, 1) @ v[a:b, h // 2] * go[a:b, h].double().cpu()).sum()
        return float(total)

    base = [t.detach().double().cpu() for t in leaves]
    for i in range(3):
        way = torch.randn(base[i].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(i))
        step = 1e-5
        up, down = ([t + s * way if j == i else t for j, t in enumerate(base)] for s in (step, -step))
        slope = (loss(*up) - loss(*down)) / (2 * step)
        terms = (grads[i].double().cpu() * way).abs().sum()
        assert abs(float((grads[i].double().cpu() * way).sum()) - slope) <= 4 * HALF_STEP[dtype] * float(terms)


@pytest.mark.parametrize("power", [-14, 0, 12])
def test_fp16_gradients_of_any_size(power):
    """Upstream gradients far below and far above one: relative errors stay those of values near one."""
    cu = _i32([0, 150, 190])
    leaves = [_randn(190, n, 64, dtype=torch.float16, seed=s).requires_grad_() for s, n in ((0, 4), (1, 2), (2, 2))]
    go = _randn(190, 4, 64, dtype=torch.float16, seed=3) * 2.0 ** -4
    base = torch.autograd.grad(F_.packed_attention(*leaves, cu, 0.125), leaves, go)
    got = torch.autograd.grad(F_.packed_attention(*leaves, cu, 0.125), leaves, go * 2.0 ** power)
    for a, b in zip(got, base):
        a, b = a.double(), b.double() * 2.0 ** power
        assert (a - b).norm() <= (2.0 ** -9 if power >= 0 else 2.0 ** -4) * b.norm()


def test_same_bits_every_time_and_on_another_stream():
    cu = _i32([0, 900, 901, 1500])
    leaves = [_randn(1500, n, 128, seed=s).requires_grad_() for s, n in ((0, 8), (1, 2), (2, 2))]
    go = _randn(1500, 8, 128, seed=3)

    def once():
        o = F_.packed_attention(*leaves, cu, 0.1)
        return [o.detach(), *torch.autograd.grad(o, leaves, go)]

    want = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(10):
            assert all(torch.equal(a, b) for a, b in zip(once(), want))
    torch.cuda.current_stream().wait_stream(side)


def test_captured_for_other_lengths():
    """Forward and backward in a graph; the ends change in place, and with them the sequences, the empty ones and the rows behind the last."""
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
    for ends in ([0, 100, 200, 256], [0, 1, 1, 250], [0, 256, 256, 256], [0, 0, 0, 0], [0, 130, 131, 200]):
        cu.copy_(_i32(ends))
        g.replay()
        got = [t.clone() for t in outs]
        _compare(q.detach(), k.detach(), v.detach(), ends, ends, 0.125, got[0], go, got[1:])


@pytest.mark.parametrize("form", ["apart", "wider", "offset"])
def test_saved_tensors_given_back_in_another_form(form):
    cu = _i32([0, 60, 90])
    leaves = [_randn(90, n, 64, seed=s).requires_grad_() for s, n in ((0, 4), (1, 2), (2, 2))]
    go = _randn(90, 4, 64, seed=3)
    want = torch.autograd.grad(F_.packed_attention(*leaves, cu, 0.1), leaves, go)

    def pack(t):
        if form == "apart":
            return t.new_empty(*t.shape, 2)[..., 0].copy_(t.detach())
        if form == "wider":
            return t.detach().float() if t.dtype == torch.bfloat16 else t.detach()
        return t.new_empty(t.numel() + 1)[1:].view(t.shape).copy_(t.detach())

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        o = F_.packed_attention(*leaves, cu, 0.1)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(o, leaves, go), want))


def test_second_derivatives_raise():
    cu = _i32([0, 20])
    leaves = [_randn(20, 2, 64, seed=s).requires_grad_() for s in range(3)]
    (g,) = torch.autograd.grad(F_.packed_attention(*leaves, cu, 0.1).float().square().sum(), leaves[0], create_graph=True)
    with pytest.raises(RuntimeError, match="first derivatives"):
        torch.autograd.grad(g.float().sum(), leaves[1])


@pytest.mark.parametrize("ends", [[0, 50, 40, 90], [0, 50, 91], [1, 50, 90], [0, -5, 90], [-3, 50], [0, 2 ** 31 - 1]])
def test_ends_that_do_not_hold_are_reported(ends):
    from cppmega_b200.ops import cuda as cu_
    leaves = [_randn(90, 2, 64, seed=s).requires_grad_() for s in range(3)]
    o = F_.packed_attention(*leaves, _i32(ends), 0.1)
    with pytest.raises(cu_.KernelError, match="bad argument"):
        cu_.check_errors()
    torch.autograd.grad(o, leaves, torch.ones_like(o))
    with pytest.raises(cu_.KernelError, match="bad argument"):
        cu_.check_errors()
    cu_.check_errors()


def test_forms_without_a_kernel_run_the_definition():
    cu = _i32([0, 20, 33])
    F_.reset_counters()
    for dtype, width in ((torch.float32, 64), (torch.bfloat16, 136), (torch.bfloat16, 12)):
        leaves = [_randn(33, n, width, dtype=dtype, seed=n).requires_grad_() for n in (4, 2, 2)]
        o = F_.packed_attention(*leaves, cu, 0.1)
        assert all(g.isfinite().all() for g in torch.autograd.grad(o.sum(), leaves))
    assert F_.fallback_counts() == {"packed_attention(shape/dtype)": 3} and not F_.launch_counts()


def test_a_prompt_continued_from_a_cache_and_then_generated():
    """Prompts attended whole; or their beginnings written to a quantised or plain cache, read back, and the rest attended as a continuation;
    or token by token over the pages: the same results within the roundings of the type."""
    lens, H, G, D, page = [50, 7, 130], 8, 2, 64, 16
    ends = _ends(lens)
    q, k, v = _randn(187, H, D), _randn(187, G, D, seed=1), _randn(187, G, D, seed=2)
    want = F_.packed_attention(q, k, v, _i32(ends), 0.125).float()
    counts = [-(-n // page) for n in lens]
    order = torch.randperm(sum(counts)).tolist()
    table = _i32([[order.pop() for _ in range(c)] + [-1] * (max(counts) - c) for c in counts])
    rows = table.tolist()
    slots = torch.tensor([rows[s][p // page] * page + p % page for s, n in enumerate(lens) for p in range(n)], device="cuda")
    kc, vc = (torch.zeros(sum(counts), page, G, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    F_.cache_write(k, v, kc, vc, slots)
    kr, vr = F_.cache_read(kc, vc, table, _i32(ends), 187)
    assert torch.equal(kr, k) and torch.equal(vr, v)
    new = [20, 7, 1]
    pick = torch.cat([torch.arange(e - n, e) for e, n in zip(ends[1:], new)]).cuda()
    rest = F_.packed_attention(q[pick], kr, vr, _i32(_ends(new)), 0.125, _i32(ends)).float()
    size = v.float().abs().max()
    assert ((rest - want[pick]).abs() <= 4 * 2.0 ** -8 * size).all()
    for n in (1, 5, 7):
        at = torch.tensor([ends[0] + n - 1, ends[1] + n - 1, ends[2] + n - 1], device="cuda")
        one = F_.paged_attention(q[at], kc, vc, table, _i32([n, n, n]), 0.125).float()
        assert ((one - want[at]).abs() <= 4 * 2.0 ** -8 * size).all()


def test_calls_of_nothing():
    for T, n in ((3, 0), (200, 0), (0, 0)):
        leaves = [_randn(T, 2, 64, seed=s).requires_grad_() for s in range(3)]
        o = F_.packed_attention(*leaves, _i32([0] * (n + 1)), 1.0)
        assert o.shape == (T, 2, 64) and (o == 0).all()
        assert all((g == 0).all() for g in torch.autograd.grad(o, leaves, torch.ones_like(o)))
    q, none = _randn(3, 2, 64).requires_grad_(), _randn(0, 2, 64)
    o = F_.packed_attention(q, none, none, _i32([0, 3]), 1.0, _i32([0, 0]))
    assert (o == 0).all()
    from cppmega_b200.ops import cuda as cu_
    cu_.check_errors()


def test_tensors_behind_32_bits():
    """More than 2^31 elements of q, o and their gradients: the last sequences against the same ones by themselves, bit for bit."""
    T, H, D = 131200, 128, 128
    assert T * H * D > 2 ** 31
    ends = [*range(0, T - 200, 1000), T - 150, T - 20, T]
    q, go = torch.empty(T, H, D, dtype=torch.bfloat16, device="cuda"), torch.empty(T, H, D, dtype=torch.bfloat16, device="cuda")
    for t, seed in ((q, 1), (go, 2)):
        t.normal_(generator=torch.Generator(device="cuda").manual_seed(seed))
    k, v = _randn(T, 4, D, seed=3), _randn(T, 4, D, seed=4)
    at = ends[-4]
    few = [e - at for e in ends[-4:]]
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = F_.packed_attention(*leaves, _i32(ends), 0.09)
    got = [o.detach()[at:], *[g[at:] for g in torch.autograd.grad(o, leaves, go)]]
    del o
    leaves = [t.detach()[at:].requires_grad_() for t in leaves]
    o = F_.packed_attention(*leaves, _i32(few), 0.09)
    assert all(torch.equal(a, b) for a, b in zip(got, [o.detach(), *torch.autograd.grad(o, leaves, go[at:])]))


def test_two_calls_at_once():
    """Forward and backward on two streams at the same time, each with its own data, leave each other alone."""
    cu = _i32([0, 700, 1500])
    data = [[_randn(1500, n, 64, dtype=torch.float16, seed=10 * i + s).requires_grad_() for s, n in ((0, 8), (1, 4), (2, 4))] for i in range(2)]
    go = [_randn(1500, 8, 64, dtype=torch.float16, std=10.0 ** (-2 * i), seed=77) for i in range(2)]

    def once(i):
        o = F_.packed_attention(*data[i], cu, 0.125)
        return [o.detach(), *torch.autograd.grad(o, data[i], go[i])]

    want = [once(0), once(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, once(i)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i, x in got for a, b in zip(x, want[i]))
