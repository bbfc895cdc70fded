"""The paged key-value cache and its attention on the GPU: inputs and calls at the edges of what they take."""
import math

import pytest
import torch

from cppmega_b200.ops import functional as F_
from cppmega_b200.ops import reference as ref

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _randn(*shape, dtype=torch.bfloat16, std=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 7919 * sum(shape))
    return torch.empty(shape, device="cuda").normal_(0.0, std, generator=g).to(dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _caches(pages, page, heads, widths, store):
    """(keys, values, their exponent bytes or None) of zeros."""
    if store != E4M3:
        return [torch.zeros(pages, page, heads, n, dtype=store, device="cuda") for n in widths] + [None, None]
    return ([torch.zeros(pages, page, heads, n, dtype=torch.uint8, device="cuda").view(E4M3) for n in widths]
            + [torch.full((pages, page, heads), 127, dtype=torch.uint8, device="cuda") for _ in widths])


@pytest.mark.parametrize("v_std", [1.0, 0.05])
@pytest.mark.parametrize("gap", [9.0, 14.0])
@pytest.mark.parametrize("D,V,heads,group", [(128, 128, 2, 4), (128, 64, 1, 32), (64, 64, 2, 3), (128, 128, 1, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_keys_without_values_set_no_reference(dtype, D, V, heads, group, gap, v_std):
    """Keys far above the rest whose values are zero, in an E4M3 cache.  A weight times its value's power is rounded to fp16 (2^-11) against the
    largest of them over rows that are not zero, below which 2^-25 of a payload of up to 448 is lost for each key."""
    n, page = 3000, 16
    kc, vc, ks, vs = _caches(200, page, heads, (D, V), E4M3)
    k, v = _randn(n, heads, D, dtype=dtype), _randn(n, heads, V, dtype=dtype, std=v_std, seed=1)
    q = _randn(1, heads * group, D, dtype=dtype, seed=2)
    k[..., 0] = 0
    q[..., 0] = 8
    above = torch.tensor([0, 5, 1000, 1016, 2999], device="cuda")
    k[above] = 0
    k[above, :, 0] = gap * D ** 0.5 / 8
    v[above] = 0
    v[1, 0] = -0.0
    table = torch.randperm(200, device="cuda").int()[None]
    pos = torch.arange(n, device="cuda")
    F_.cache_write(k, v, kc, vc, table[0].long()[pos // page] * page + pos % page, ks, vs)
    got = F_.paged_attention(q, kc, vc, table, _i32([n]), D ** -0.5, ks, vs)[0].double()
    kd, vd = (t.double() for t in F_.cache_read(kc, vc, table, _i32([0, n]), n, ks, vs, dtype=torch.float32))
    half = HALF_STEP[dtype]
    for h in range(heads * group):
        kh, vh, qh = kd[:, h // group], vd[:, h // group], q[0, h].double()
        s = kh @ qh * D ** -0.5
        p = torch.softmax(s, 0)
        e = 2 * ((D + 4) * 2.0 ** -23 * (kh.abs() @ qh.abs() * D ** -0.5).amax() + 2.0 ** -22 * s.abs().amax()) + 2.0 ** -20 + 4 * n * 2.0 ** -24
        want, size = p @ vh, p @ vh.abs()
        largest = (p * vh.abs().amax(1)).amax() * 2               # a row's largest payload is above 224
        bound = (half + 2.0 ** -11) * want.abs() + (1 + half) * (size * (2.0 ** -11 + e) + n * 2.0 ** -25 * largest) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        assert ((got[h] - want).abs() <= bound).all(), float(((got[h] - want).abs() / bound).max())


def test_a_cache_of_keys_without_values_gives_zeros():
    kc, vc, ks, vs = _caches(4, 16, 1, (64, 64), E4M3)
    F_.cache_write(_randn(50, 1, 64), torch.zeros(50, 1, 64, dtype=torch.bfloat16, device="cuda"), kc, vc, torch.arange(50, device="cuda"), ks, vs)
    assert (F_.paged_attention(_randn(1, 4, 64), kc, vc, _i32([[0, 1, 2, 3]]), _i32([50]), 0.125, ks, vs) == 0).all()


def _reported():
    from cppmega_b200.ops import cuda as cu
    with pytest.raises(cu.KernelError, match="bad argument"):
        cu.check_errors()
    cu.check_errors()


@pytest.mark.parametrize("bad", [-1, 40, 2 ** 31 - 1, -2 ** 31])
@pytest.mark.parametrize("page", [16, 64, 24, 7, 1])
@pytest.mark.parametrize("store", [torch.bfloat16, E4M3])
def test_keys_of_pages_outside_the_cache_have_no_weight(store, page, bad):
    """The attention over the other keys, as if those of the page were not there: pages of whole steps, of parts of steps, first, last, and all of
    them."""
    heads, H, D, pages = 2, 8, 64, 40
    caches = _caches(pages, page, heads, (D, D), store)
    n = pages * page
    k, v = _randn(n, heads, D, std=0.3), _randn(n, heads, D, seed=1) + 2
    F_.cache_write(k, v, caches[0], caches[1], torch.arange(n, device="cuda"), *caches[2:])
    if store == E4M3:
        k, v = (t.bfloat16() for t in F_.cache_read(*caches[:2], torch.arange(pages, device="cuda").int()[None], _i32([0, n]), n, *caches[2:]))
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(page)).tolist()
    table = [[*order[:5], bad, *order[5:9]], [bad, *order[10:19]], [*order[20:28], bad, bad], [bad] * 10, order[:10]]
    lens = [10 * page, 10 * page - page // 2, 9 * page + 1, 10 * page, 10 * page]
    q = _randn(5, H, D, seed=2)
    got = F_.paged_attention(q, *caches[:2], _i32(table), _i32(lens), 1.0, *caches[2:])
    _reported()
    kd, vd, half = k.double().view(pages, page, heads, D), v.double().view(pages, page, heads, D), 2.0 ** -8
    for b, (row, length) in enumerate(zip(table, lens)):
        pos = torch.arange(length, device="cuda")
        pos = pos[torch.tensor([row[p // page] != bad for p in pos.tolist()], device="cuda")]
        at = torch.tensor(row, device="cuda")[pos // page], pos % page
        for h in range(H):
            kh, vh, qh = kd[at[0], at[1], h // 4], vd[at[0], at[1], h // 4], q[b, h].double()
            if len(pos) == 0:
                assert (got[b] == 0).all()
                continue
            s = kh @ qh
            p = torch.softmax(s, 0)
            e = 2 * ((D + 4) * 2.0 ** -23 * (kh.abs() @ qh.abs()).amax() + 2.0 ** -22 * s.abs().amax()) + 2.0 ** -20 + 4 * length * 2.0 ** -24
            want, size = p @ vh, p @ vh.abs()
            bound = 2 * half * want.abs() + (1 + half) * size * (half + e) + length * 2.0 ** -15 * float(store == E4M3) * (p * vh.abs().amax(1)).amax()
            assert ((got[b, h].double() - want).abs() <= bound).all(), float(((got[b, h].double() - want).abs() / bound).max())


@pytest.mark.parametrize("swap", [False, True])
def test_tokens_moved_inside_a_cache(swap):
    """Every token one place further, keys to keys or to values, in one call over many blocks."""
    kc, vc = _randn(1000, 16, 4, 64), _randn(1000, 16, 4, 64, seed=1)
    was = [t.clone().view(16000, 4, 64) for t in (kc, vc)]
    k, v = (t.view(16000, 4, 64)[:15999] for t in ((vc, kc) if swap else (kc, vc)))
    F_.cache_write(k, v, kc, vc, torch.arange(1, 16000, device="cuda"))
    for got, rows, old in zip((kc, vc), reversed(was) if swap else was, was):
        assert torch.equal(got.view(16000, 4, 64)[1:], rows[:15999]) and torch.equal(got.view(16000, 4, 64)[0], old[0])


@pytest.mark.parametrize("lens", [[0, 1], [-1, 0], [2 ** 31 - 1, 0]])
def test_lengths_over_a_table_of_no_columns_are_reported(lens):
    kc, vc = _randn(5, 16, 2, 64), _randn(5, 16, 2, 64, seed=1)
    got = F_.paged_attention(_randn(2, 4, 64), kc, vc, torch.zeros(2, 0, dtype=torch.int32, device="cuda"), _i32(lens), 0.1)
    _reported()
    assert (got == 0).all()


@pytest.mark.parametrize("store", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("heads", [2, 0])
@pytest.mark.parametrize("ends", [[0, 1], [1, 0], [0, -1], [-1, 0]])
def test_ends_of_a_read_of_no_rows_are_reported(ends, heads, store):
    kc, vc, ks, vs = _caches(5, 16, heads, (64, 64), store)
    k, v = F_.cache_read(kc, vc, _i32([[1, 4, 3]]), _i32(ends), 0, ks, vs)
    _reported()
    assert k.shape == v.shape == (0, heads, 64)
    k, _ = F_.cache_read(kc, vc, _i32([[1, 4, 3]]), _i32([0, 0]), 0, ks, vs)
    from cppmega_b200.ops import cuda as cu
    cu.check_errors()


@pytest.mark.parametrize("store", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("pages,heads", [(5, 0), (0, 2)])
def test_pages_and_slots_of_a_cache_of_nothing_are_reported(pages, heads, store):
    kc, vc, ks, vs = _caches(pages, 16, heads, (64, 64), store)
    k, v = F_.cache_read(kc, vc, _i32([[1, 5, 3]]), _i32([0, 40]), 40, ks, vs)
    _reported()
    assert k.shape == v.shape == (40, heads, 64) and (k == 0).all() and (v == 0).all()
    F_.cache_write(_randn(2, heads, 64), _randn(2, heads, 64), kc, vc, torch.tensor([3, 80], device="cuda"), ks, vs)
    _reported()
    slots = [3, -1] if pages else [-1, -1]
    F_.cache_write(_randn(2, heads, 64), _randn(2, heads, 64), kc, vc, torch.tensor(slots, device="cuda"), ks, vs)
    F_.cache_write(_randn(0, heads, 64), _randn(0, heads, 64), kc, vc, torch.zeros(0, dtype=torch.int32, device="cuda"), ks, vs)
    from cppmega_b200.ops import cuda as cu
    cu.check_errors()


@pytest.mark.parametrize("store", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("page", [16, 7])
def test_attention_over_a_cache_of_no_pages(page, store):
    kc, vc, ks, vs = _caches(0, page, 2, (64, 64), store)
    table = torch.zeros(2, 30, dtype=torch.int32, device="cuda")
    assert (F_.paged_attention(_randn(2, 4, 64), kc, vc, table, _i32([0, 0]), 0.1, ks, vs) == 0).all()
    from cppmega_b200.ops import cuda as cu
    cu.check_errors()
    assert (F_.paged_attention(_randn(2, 4, 64), kc, vc, table, _i32([0, 200]), 0.1, ks, vs) == 0).all()
    _reported()


@pytest.mark.parametrize("store", [torch.float16, E4M3])
@pytest.mark.parametrize("group", [1, 12])
def test_keys_far_below_one_with_few_values(store, group):
    """Weights that one key pushes 10 to 17 below it, the same for all the others, so that their roundings add up: 2^-11 of each, and 2^-25 under the 2^7 that
    the largest (over E4M3 times its values' power, which is 2^-20 for that key) counts at the least."""
    n, D, page, dtype = 300, 64, 16, torch.float16
    kc, vc, ks, vs = _caches(20, page, 1, (D, D), store)
    q, k = torch.zeros(64, group, D, device="cuda").half(), torch.zeros(n, 1, D, device="cuda").half()
    q[:, :, 0] = torch.linspace(10, 17, 64 * group, device="cuda").view(64, group)
    k[40, 0, 0] = 1
    v = torch.full((n, 1, D), 7.0, device="cuda").half()
    v[40] = 7 * 2.0 ** -20 if store == E4M3 else 0
    F_.cache_write(k, v, kc, vc, torch.arange(n, device="cuda"), ks, vs)
    table = torch.arange(20, device="cuda").int()[None].expand(64, -1)
    got = F_.paged_attention(q, kc, vc, table, _i32([n] * 64), 1.0, ks, vs).double()
    s = q.double() @ k[:, 0].double().T
    p = torch.softmax(s, -1)
    e = 2 * ((D + 4) * 2.0 ** -23 + 2.0 ** -22) * 17 + 2.0 ** -20 + 4 * n * 2.0 ** -24
    rows = v[:, 0].double()
    want = p @ rows
    lost = 2.0 ** -32 * (rows if store != E4M3 else (p[..., None] * rows).amax(-2, keepdim=True).expand(-1, -1, n, -1)).sum(-2)
    u = 2.0 ** -11
    bound = (p * (u + e)) @ rows + lost + want * (u + e + u) + 2.0 ** -25
    assert ((got - want).abs() <= bound * (1 + u)).all(), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("store", [torch.bfloat16, E4M3])
def test_equal_slots_among_slots_of_one_hash_place(store):
    """Blocks of 128 tokens whose slots fall to three places of the hash table, 20 different ones to each and some often: chains of 40 and more, in which
    equal slots and others follow one another.  Of equal slots the last row stays."""
    slots = torch.arange(1 << 17, dtype=torch.int64)
    place = (slots * 2654435769 % (1 << 32)) >> 21             # as the kernel has it
    some = torch.cat([slots[place == p][:20] for p in (0, 777, 2047)])
    assert len(some) == 60
    T = 80000
    g = torch.Generator().manual_seed(1)
    drawn = some[torch.randint(0, 60, (T,), generator=g)]
    drawn[::7] = -1
    drawn[::13] = torch.randint(0, 1 << 17, (len(drawn[::13]),), generator=g)
    drawn = drawn.cuda()
    k = _randn(T, 1, 16)
    (kc, _, ks, _), (wk, _, wks, _) = _caches(1 << 13, 16, 1, (16, 8), store), _caches(1 << 13, 16, 1, (16, 8), store)
    F_.cache_write(k, None, kc, None, drawn, ks)
    ref.cache_write(k, None, wk, None, drawn, wks)
    assert torch.equal(kc.view(torch.uint8 if store == E4M3 else torch.int16), wk.view(torch.uint8 if store == E4M3 else torch.int16))
    assert ks is None or torch.equal(ks, wks)
