"""The paged key-value cache and the packed and paged attention on the CPU: definitions and refusals."""
import math

import pytest
import torch

from cppmega_b200.ops import functional as F_
from cppmega_b200.ops import reference as ref

E4M3 = torch.float8_e4m3fn


def _randn(*shape, dtype=torch.float32, std=1.0, seed=0):
    g = torch.Generator().manual_seed(seed + 7919 * sum(shape))
    return torch.empty(shape).normal_(0.0, std, generator=g).to(dtype)


def _cache(pages, page, heads, dim, vdim, store, fill=0.0):
    if store == E4M3:
        kc, vc = (torch.zeros(pages, page, heads, n, dtype=torch.uint8).view(E4M3) for n in (dim, vdim))
        return kc, vc, *(torch.full((pages, page, heads), 127, dtype=torch.uint8) for _ in range(2))
    return torch.full((pages, page, heads, dim), fill, dtype=store), torch.full((pages, page, heads, vdim), fill, dtype=store), None, None


# ---- quantised rows ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantised_rows_are_within_half_a_step(dtype):
    """E4M3 has 4 bits: 2^-4 of the value, and half of 2^-9 of the power of two among the subnormals."""
    x = _randn(64, 3, 40, dtype=dtype) * torch.logspace(-3, 3, 64, dtype=torch.float64)[:, None, None].to(dtype)
    payload, byte = ref.cache_row_quantize(x)
    power = ref.cache_power(byte).double()[..., None]
    err = (payload.double() * power - x.double()).abs()
    assert (err <= torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * power)).all()
    amax = x.double().abs().amax(-1)
    assert (amax <= 448 * power[..., 0]).all() and (amax > 224 * power[..., 0]).all()


@pytest.mark.parametrize("amax,byte", [(448.0, 127), (449.0, 128), (1.75, 119), (1.7500001, 120), (2.0 ** -149, 1), (0.0, 127),
                                       (3.0e38, 247), (math.inf, 127), (math.nan, 127)])
def test_exponent_byte(amax, byte):
    x = torch.tensor([[0.0, -amax, 0.0]])
    payload, got = ref.cache_row_quantize(x)
    assert int(got) == byte
    if math.isfinite(amax):
        assert payload.float().isfinite().all()
    else:
        assert payload.float()[0, 1].isnan() and (payload.float()[0, [0, 2]] == 0).all()


def test_a_value_that_is_not_finite_leaves_its_row_usable():
    x = torch.tensor([[1.0, math.inf, -3.5, math.nan]])
    payload, byte = ref.cache_row_quantize(x)
    y = payload.float() * ref.cache_power(byte)
    assert y[0, 0] == 1 and y[0, 2] == -3.5 and y[0, [1, 3]].isnan().all()


# ---- write and read ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("store", [torch.float32, torch.bfloat16, E4M3])
def test_write_then_read_back(store):
    lens, page = [5, 0, 9, 1], 4
    table = torch.tensor([[6, 2, 99], [99, 99, 99], [0, 5, 3], [4, 99, 99]], dtype=torch.int32)
    ends = torch.tensor([0, 5, 5, 14, 15], dtype=torch.int32)
    dtype = torch.bfloat16 if store == E4M3 else store
    k, v = _randn(17, 2, 8, dtype=dtype), _randn(17, 2, 16, dtype=dtype, seed=1)
    slots = torch.full((17,), -1)
    for s, n in enumerate(lens):
        for p in range(n):
            slots[int(ends[s]) + p] = int(table[s, p // page]) * page + p % page
    kc, vc, ks, vs = _cache(7, page, 2, 8, 16, store)
    F_.cache_write(k, v, kc, vc, slots, ks, vs)
    rk, rv = F_.cache_read(kc, vc, table, ends, 16, ks, vs)
    for got, x in ((rk, k), (rv, v)):
        want = x[:15]
        if store == E4M3:
            payload, byte = ref.cache_row_quantize(want)
            want = (payload.float() * ref.cache_power(byte)[..., None]).to(dtype)
        assert got.dtype == dtype and torch.equal(got[:15], want) and (got[15:] == 0).all()
    only, none = F_.cache_read(kc, None, table, ends, 16, ks, None)
    assert none is None and torch.equal(only, rk)


def test_of_equal_slots_the_last_row_stays():
    kc, vc, _, _ = _cache(2, 3, 1, 4, 4, torch.float32, fill=7.0)
    k = torch.arange(5.0)[:, None, None].expand(5, 1, 4)
    F_.cache_write(k, -k, kc, vc, torch.tensor([4, 0, 4, -1, 0], dtype=torch.int32))
    flat = kc.view(6, 4)[:, 0].tolist()
    assert flat == [4, 7, 7, 7, 2, 7] and vc.view(6, 4)[:, 0].tolist() == [-4, 7, 7, 7, -2, 7]


def test_a_cache_takes_values_without_gradients():
    kc, _, _, _ = _cache(1, 2, 1, 4, 4, torch.float32)
    k = torch.ones(1, 1, 4, requires_grad=True)
    F_.cache_write(k, None, kc, None, torch.tensor([1]))
    assert not kc.requires_grad and (kc[0, 1] == 1).all()


# ---- attention ---------------------------------------------------------------------------------------------------------

def test_paged_attention_is_the_last_row_of_the_packed_one():
    lens, page, H, G, D, V = [7, 1, 12], 5, 6, 2, 8, 12
    ends = torch.tensor([0, 7, 8, 20], dtype=torch.int32)
    q, k, v = _randn(20, H, D), _randn(20, G, D, seed=1), _randn(20, G, V, seed=2)
    table = torch.tensor([[3, 0, -5], [1, 77, 77], [6, 2, 4]], dtype=torch.int32)
    kc, vc, _, _ = _cache(7, page, G, D, V, torch.float32, fill=math.nan)
    slots = torch.tensor([int(table[s, p // page]) * page + p % page for s, n in enumerate(lens) for p in range(n)])
    F_.cache_write(k, v, kc, vc, slots)
    full = F_.packed_attention(q, k, v, ends, 0.3)
    got = F_.paged_attention(q[[6, 7, 19]], kc, vc, table, torch.tensor(lens, dtype=torch.int32), 0.3)
    assert torch.allclose(got, full[[6, 7, 19]], rtol=1e-5, atol=1e-6)
    none = F_.paged_attention(q[:1], kc, vc, torch.full((1, 2), -1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 0.3)
    assert (none == 0).all()


def test_packed_attention_against_one_sequence_at_a_time():
    ends = torch.tensor([0, 3, 3, 8], dtype=torch.int32)
    q, k, v = (_randn(10, n, 8, seed=i).requires_grad_() for i, n in enumerate((4, 2, 2)))
    o = F_.packed_attention(q, k, v, ends, 0.5)
    assert (o[8:] == 0).all()
    for a, b in ((0, 3), (3, 8)):
        want = torch.nn.functional.scaled_dot_product_attention(
            *(t[a:b].repeat_interleave(4 // t.shape[1], 1).transpose(0, 1) for t in (q, k, v)), is_causal=True, scale=0.5).transpose(0, 1)
        assert torch.allclose(o[a:b], want, rtol=1e-5, atol=1e-6)
    grads = torch.autograd.grad(o.square().sum(), [q, k, v])
    assert all((g[8:] == 0).all() and g[:8].abs().max() > 0 for g in grads)


def test_packed_attention_with_keys_before_and_without_any():
    """Four sequences: keys from before, fewer keys than queries (the first queries see nothing), no keys at all, no queries."""
    cq, ck = torch.tensor([0, 2, 5, 7, 7], dtype=torch.int32), torch.tensor([0, 6, 8, 8, 10], dtype=torch.int32)
    q, k, v = _randn(7, 2, 4), _randn(10, 1, 4, seed=1), _randn(10, 1, 4, seed=2)
    o = F_.packed_attention(q, k, v, cq, 1.0, ck)
    whole = F_.packed_attention(torch.cat([_randn(4, 2, 4, seed=9), q[:2]]), k[:6], v[:6], torch.tensor([0, 6], dtype=torch.int32), 1.0)
    assert torch.allclose(o[:2], whole[4:], rtol=1e-5, atol=1e-6)
    assert (o[2] == 0).all() and torch.allclose(o[3], v[6].expand(2, 4)) and o[4].abs().max() > 0 and (o[5:] == 0).all()


# ---- refusals ----------------------------------------------------------------------------------------------------------

def _i32(*values):
    return torch.tensor(values, dtype=torch.int32)


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(4, 3, 8)), dict(q=torch.zeros(4, 2, 16)), dict(q=torch.zeros(4, 16)), dict(v=torch.zeros(3, 2, 8)),
    dict(k=torch.zeros(4, 0, 8), v=torch.zeros(4, 0, 8)), dict(k=torch.zeros(5, 2, 8), v=torch.zeros(5, 2, 8)),
    dict(k=torch.zeros(4, 2, 8, dtype=torch.float64)), dict(cu=torch.tensor([0, 4])), dict(cu=_i32(0, 5)), dict(cu=_i32(1, 4)), dict(cu=_i32(0, 3, 2)),
    dict(cu=torch.zeros(0, dtype=torch.int32)), dict(cu=_i32(0, 4)[None]), dict(cu_k=_i32(0, 1, 4)), dict(cu_k=_i32(0, 9)),
])
def test_packed_attention_refuses(change):
    args = dict(q=torch.zeros(4, 2, 8), k=torch.zeros(4, 2, 8), v=torch.zeros(4, 2, 8), cu=_i32(0, 4), cu_k=None)
    F_.packed_attention(args["q"], args["k"], args["v"], args["cu"], 1.0, args["cu_k"])
    args.update(change)
    with pytest.raises(ValueError):
        F_.packed_attention(args["q"], args["k"], args["v"], args["cu"], 1.0, args["cu_k"])


@pytest.mark.parametrize("change", [
    dict(k=torch.zeros(3, 2, 16)), dict(k=torch.zeros(3, 1, 8)), dict(k=torch.zeros(3, 2, 8, dtype=torch.float16)), dict(v=None),
    dict(slots=torch.tensor([0, 1])), dict(slots=torch.tensor([0.0, 1, 2])), dict(slots=torch.tensor([0, 1, 8])), dict(ks=torch.zeros(2, 4, 2, dtype=torch.uint8)),
    dict(kc=torch.zeros(2, 4, 2, 8, dtype=torch.uint8).view(E4M3)), dict(vc=torch.zeros(2, 5, 2, 8)), dict(kc=torch.zeros(8, 2, 8)),
    dict(kc=torch.zeros(2, 4, 2, 8, requires_grad=True)), dict(kc=torch.zeros(1, 4, 2, 8).expand(2, 4, 2, 8)), dict(slots=torch.tensor(3)),
])
def test_cache_write_refuses(change):
    args = dict(k=torch.ones(3, 2, 8), v=torch.ones(3, 2, 8), kc=torch.zeros(2, 4, 2, 8), vc=torch.zeros(2, 4, 2, 8), slots=torch.tensor([0, 5, 7]),
                ks=None, vs=None)
    F_.cache_write(args["k"], args["v"], args["kc"], args["vc"], args["slots"])
    args.update(change)
    with pytest.raises((ValueError, RuntimeError)):
        F_.cache_write(args["k"], args["v"], args["kc"], args["vc"], args["slots"], args["ks"], args["vs"])


@pytest.mark.parametrize("change", [
    dict(ends=torch.tensor([0, 3])), dict(ends=_i32(0, 3, 4)), dict(ends=_i32(0, 9)), dict(ends=_i32(1, 3)), dict(total=2), dict(total=-1),
    dict(table=torch.tensor([[1]])), dict(table=_i32(1)), dict(table=_i32(2)[None]), dict(table=_i32(-1)[None]), dict(dtype=torch.float64),
])
def test_cache_read_refuses(change):
    args = dict(kc=torch.zeros(2, 4, 2, 8), vc=torch.zeros(2, 4, 2, 8), table=_i32(1)[None], ends=_i32(0, 3), total=3, dtype=None)
    F_.cache_read(args["kc"], args["vc"], args["table"], args["ends"], args["total"])
    args.update(change)
    with pytest.raises(ValueError):
        F_.cache_read(args["kc"], args["vc"], args["table"], args["ends"], args["total"], dtype=args["dtype"])


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(1, 3, 8)), dict(q=torch.zeros(1, 4, 16)), dict(q=torch.zeros(4, 8)), dict(lens=_i32(3, 3)), dict(lens=torch.tensor([3])),
    dict(lens=_i32(5)), dict(lens=_i32(-1)), dict(table=_i32(2)[None]), dict(table=_i32(-1)[None]), dict(table=_i32(1, 1)[:, None]), dict(vc=None),
    dict(kc=torch.zeros(2, 0, 2, 8), vc=torch.zeros(2, 0, 2, 8)), dict(vc=torch.zeros(2, 4, 2, 8, dtype=torch.float64)),
])
def test_paged_attention_refuses(change):
    args = dict(q=torch.zeros(1, 4, 8), kc=torch.zeros(2, 4, 2, 8), vc=torch.zeros(2, 4, 2, 8), table=_i32(1)[None], lens=_i32(3))
    F_.paged_attention(args["q"], args["kc"], args["vc"], args["table"], args["lens"], 1.0)
    args.update(change)
    with pytest.raises(ValueError):
        F_.paged_attention(args["q"], args["kc"], args["vc"], args["table"], args["lens"], 1.0)


def test_calls_of_nothing():
    """No sequences, no tokens, no columns, no rows to read."""
    for T, Tk in ((3, 3), (0, 0)):
        o = F_.packed_attention(torch.ones(T, 2, 8), torch.ones(Tk, 2, 8), torch.ones(Tk, 2, 8), _i32(0), 1.0)
        assert o.shape == (T, 2, 8) and (o == 0).all()
        leaves = [torch.ones(n, 2, 8, requires_grad=True) for n in (T, Tk, Tk)]
        assert all((g == 0).all() for g in torch.autograd.grad(F_.packed_attention(*leaves, _i32(0), 1.0).sum(), leaves))
    assert (F_.packed_attention(torch.ones(3, 2, 8), torch.ones(0, 2, 8), torch.ones(0, 2, 8), _i32(0, 3), 1.0, _i32(0, 0)) == 0).all()
    kc, vc = torch.ones(2, 4, 2, 8), torch.ones(2, 4, 2, 8)
    F_.cache_write(torch.zeros(0, 2, 8), torch.zeros(0, 2, 8), kc, vc, torch.zeros(0, dtype=torch.int64))
    assert (kc == 1).all() and (vc == 1).all()
    none = torch.zeros(0, 3, dtype=torch.int32)
    assert F_.cache_read(kc, vc, none, _i32(0), 0)[0].shape == (0, 2, 8) and (F_.cache_read(kc, vc, none, _i32(0), 5)[1] == 0).all()
    assert F_.paged_attention(torch.ones(0, 4, 8), kc, vc, none, _i32(), 1.0).shape == (0, 4, 8)
    assert (F_.paged_attention(torch.ones(2, 4, 8), kc, vc, none.new_zeros(2, 0), _i32(0, 0), 1.0) == 0).all()


def test_a_cache_that_was_saved_for_a_gradient_and_written():
    kc, vc, q = torch.ones(2, 4, 2, 8), torch.ones(2, 4, 2, 8), torch.ones(1, 4, 8, requires_grad=True)
    before = kc._version, vc._version
    F_.cache_write(torch.zeros(1, 2, 8), torch.zeros(1, 2, 8), kc, vc, torch.tensor([5]))
    assert kc._version > before[0] and vc._version > before[1]
