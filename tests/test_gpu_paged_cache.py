"""The paged key-value cache on the GPU: rows written and read back, and the attention of one token over them.

Tolerances of the attention, in terms of the exact weights p: a weight is rounded once (2^-8 in bf16, 2^-11 in fp16) and carries twice the error of
a score: its fp32 sum over D products (D 2^-23 of their magnitudes, however they are added) and two roundings of scale and power; the exponential is
good to 2^-21 (its argument's rounding at up to 2^8 included apart, as 2^-24 of the score); the sums of weights and of weighted values add n
2^-24.  The result is rounded once.  In an E4M3 cache weights below 2^-24 of the reference are lost: 2^-25 each of the largest contribution times 2^8.
"""
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


def _blank(pages, page, heads, width, store):
    """A cache of NaN (its rows that nobody writes stay so) and exponent bytes of 255."""
    if store == E4M3:
        return (torch.full((pages, page, heads, width), 0x7f, dtype=torch.uint8, device="cuda").view(E4M3),
                torch.full((pages, page, heads), 255, dtype=torch.uint8, device="cuda"))
    return torch.full((pages, page, heads, width), math.nan, dtype=store, device="cuda"), None


def _bits(t):
    return t if t is None else t.contiguous().view(torch.uint8 if t.element_size() == 1 else torch.int16)


def _tables(lens, page, seed=0):
    """Pages in a random order, garbage behind a sequence's last one; (table, pages)."""
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + 2
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).tolist()
    table = [[order.pop() for _ in range(c)] for c in counts]
    width = max(max(counts), 1) + 1
    return _i32([row + [2 ** 31 - 1 - i for i in range(width - len(row))] for row in table]), pages


def _slots(table, lens, page):
    rows = table.tolist()
    return torch.tensor([rows[s][p // page] * page + p % page for s, n in enumerate(lens) for p in range(n)], dtype=torch.int64, device="cuda")


def _same(got, want):
    """Equal bits, but a NaN may be any NaN."""
    if got.dtype == E4M3:
        a, b = got.float(), want.float()
        return bool(((a == b) | (a.isnan() & b.isnan())).all())
    a, b = _bits(got), _bits(want)
    nan = got.isnan() & want.isnan() if got.is_floating_point() else torch.zeros_like(a, dtype=torch.bool)
    return bool(((a == b) | nan).all())


# ---- write and read ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("D,V", [(128, 128), (128, 64), (8, 256), (40, 80), (200, 16)])
@pytest.mark.parametrize("store,dtype", [(E4M3, torch.bfloat16), (E4M3, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)])
def test_write_and_read(store, dtype, D, V, wide):
    lens, page, heads = [37, 0, 1, 130, 64], 12, 3
    table, pages = _tables(lens, page)
    T = sum(lens)
    slots = torch.cat([_slots(table, lens, page), torch.tensor([-1, -7], device="cuda")])
    scales = torch.logspace(-6, 4, T + 2, device="cuda")[:, None, None]
    k, v = ((_randn(T + 2, heads, n, dtype=torch.float32, seed=n) * scales).to(dtype) for n in (D, V))
    k[5, 1] = 0
    (kc, ks), (vc, vs) = _blank(pages, page, heads, D, store), _blank(pages, page, heads, V, store)
    wk, wv, wks, wvs = (None if t is None else t.clone() for t in (kc, vc, ks, vs))
    F_.reset_counters()
    F_.cache_write(k, v, kc, vc, slots if wide else slots.int(), ks, vs)
    assert F_.launch_counts() == {"cache_write": 1} and not F_.fallback_counts()
    ref.cache_write(k, v, wk, wv, slots, wks, wvs)
    assert _same(kc, wk) and _same(vc, wv)
    if ks is not None:
        assert torch.equal(ks, wks) and torch.equal(vs, wvs)
    ends = _i32([0] + torch.tensor(lens).cumsum(0).tolist())
    got = F_.cache_read(kc, vc, table, ends, T + 5, ks, vs, dtype=dtype)
    want = ref.cache_read(kc, vc, table, ends, T + 5, ks, vs, dtype)
    assert F_.launch_counts() == {"cache_write": 1, "cache_read": 1}
    assert all(_same(a, b) and a.dtype == dtype for a, b in zip(got, want)) and (got[0][T:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_write_of_rows_at_the_edges(dtype):
    """Largest magnitudes next to 448 * 2^e, subnormals, infinities and NaN: the same bytes as the definition's."""
    top = torch.finfo(dtype).max
    amax = torch.tensor([448, 450, 224, 225, 1.75, 1.7578125, 3.5, 2.0 ** -14, 2.0 ** -20, torch.finfo(dtype).smallest_normal / 64, top, 0.0,
                         math.inf, math.nan], device="cuda")
    x = torch.linspace(-1, 1, 64, device="cuda") * torch.where(amax.isfinite(), amax, torch.ones_like(amax))[:, None]
    x[~amax.isfinite(), 5] = amax[~amax.isfinite()]
    x = x.to(dtype)[:, None]
    (kc, ks), (wk, wks) = _blank(2, 8, 1, 64, E4M3), _blank(2, 8, 1, 64, E4M3)
    slots = torch.arange(len(amax), device="cuda")
    F_.cache_write(x, None, kc, None, slots, ks)
    ref.cache_write(x, None, wk, None, slots, wks)
    assert _same(kc, wk) and torch.equal(ks, wks)


def test_of_equal_slots_the_last_row_stays():
    """Equal slots inside a block, across blocks, and slots that share a place in the block's bit table."""
    T, pages, page = 5000, 640, 16
    g = torch.Generator(device="cuda").manual_seed(3)
    slots = torch.randint(-3, 700, (T,), generator=g, device="cuda")
    slots = torch.where(slots > 600, slots - 600 + 8192, slots)          # the same low bits as others
    k = torch.arange(T, device="cuda").float()[:, None, None].expand(T, 2, 8).to(torch.bfloat16) + _randn(T, 2, 8)
    for store in (torch.bfloat16, E4M3):
        (kc, ks), (wk, wks) = _blank(pages, page, 2, 8, store), _blank(pages, page, 2, 8, store)
        F_.cache_write(k, None, kc, None, slots, ks)
        ref.cache_write(k, None, wk, None, slots, wks)
        assert _same(kc, wk) and (ks is None or torch.equal(ks, wks))


def test_strided_rows_and_caches():
    """Rows that are columns of a projection, keys and values interleaved in one cache, heads of a wider cache."""
    T, page = 33, 16
    qkv = _randn(T, 10, 64)
    k, v = qkv[:, 4:7], qkv[:, 7:10]
    both = torch.zeros(4, 2, page, 6, 64, dtype=torch.bfloat16, device="cuda")
    kc, vc = both[:, 0, :, 1:4], both[:, 1, :, 2:5]
    slots = torch.randperm(4 * page, device="cuda")[:T]
    F_.cache_write(k, v, kc, vc, slots)
    want = torch.zeros_like(both)
    ref.cache_write(k, v, want[:, 0, :, 1:4], want[:, 1, :, 2:5], slots)
    assert torch.equal(both, want)
    table, ends = _i32([[2, 0, 3]]), _i32([0, 40])
    got = F_.cache_read(kc, vc, table, ends, 40)
    assert all(torch.equal(a, b) for a, b in zip(got, ref.cache_read(kc, vc, table, ends, 40)))
    odd = _randn(T, 3, 65)[..., 1:]                                       # rows off the 16-byte grid are copied
    F_.cache_write(odd, None, kc, None, slots)
    assert torch.equal(kc.reshape(-1, 3, 64)[slots], odd)


# ---- attention ---------------------------------------------------------------------------------------------------------

def _exact(q, kc, vc, table, lens, scale, ks, vs):
    """(result, weighted magnitudes, score error, smallest-weight error) in 64 bits, one sequence at a time."""
    B, H, D = q.shape
    page, G, V = kc.shape[1], kc.shape[2], vc.shape[3]
    outs = [torch.zeros(B, H, V, dtype=torch.float64, device="cuda") for _ in range(4)]
    for b, n in enumerate(lens):
        if n == 0:
            continue
        pages = table[b, :-(-n // page)].long()
        k, v = (c.view(torch.uint8)[pages].view(E4M3).double() if s is not None else c[pages].double() for c, s in ((kc, ks), (vc, vs)))
        if ks is not None:
            k, v = k * ref.cache_power(ks[pages]).double()[..., None], v * ref.cache_power(vs[pages]).double()[..., None]
        k, v = (t.reshape(-1, G, t.shape[-1])[:n].repeat_interleave(H // G, 1).transpose(0, 1) for t in (k, v))
        qb = q[b].double()[:, None]
        s = (qb @ k.transpose(1, 2)) * scale
        mags = (qb.abs() @ k.abs().transpose(1, 2)) * abs(scale)
        p = torch.softmax(s, -1)
        outs[0][b] = (p @ v)[:, 0]
        outs[1][b] = (p @ v.abs())[:, 0]
        outs[2][b] = ((D + 4) * 2.0 ** -23 * mags).amax(-1) + 2.0 ** -22 * s.abs().amax(-1)
        largest = v.abs().amax(-1, keepdim=True).transpose(1, 2) * 2       # 448 * 2^e of each row is at most twice its largest magnitude
        if vs is not None:
            largest = (448 * ref.cache_power(vs[pages]).double().reshape(-1, G)[:n].repeat_interleave(H // G, 1).T)[:, None]
        outs[3][b] = n * 2.0 ** -17 * (p * largest).amax(-1)
    return outs


def _check(q, kc, vc, table, lens, scale, ks=None, vs=None, got=None):
    if got is None:
        F_.reset_counters()
        got = F_.paged_attention(q, kc, vc, table, _i32(lens), scale, ks, vs)
        assert F_.launch_counts() == {"paged_attention": 1} and not F_.fallback_counts()
    want, size, e_score, lost = _exact(q, kc, vc, table, lens, scale, ks, vs)
    half = HALF_STEP[q.dtype]
    weight = 2.0 ** -11 if ks is not None else half
    n = max(max(lens), 1)
    # over a 16-bit cache the sum is that of the rounded weights: sum p (1 + d) v / sum p (1 + d) is off by sum p d (v - o), |d| <= weight
    own = half * want.abs() if ks is not None else (half + weight) * want.abs()
    bound = own + (1 + half) * (size * (weight + 2 * e_score + 2.0 ** -20 + 4 * n * 2.0 ** -24) + (lost if ks is not None else 0))
    bound = bound + torch.finfo(q.dtype).smallest_normal
    assert got.dtype == q.dtype and ((got.double() - want).abs() <= bound).all(), ((got.double() - want).abs() / bound).max()
    return got


def _filled(lens, page, heads, D, V, store, dtype, seed=0):
    """A cache filled by the writer; NaN wherever no token lies."""
    table, pages = _tables(lens, page, seed)
    T = sum(lens)
    (kc, ks), (vc, vs) = _blank(pages, page, heads, D, store), _blank(pages, page, heads, V, store)
    big = 1 + 3 * (torch.rand(T, 1, 1, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)) < 0.05)
    k, v = _randn(T, heads, D, dtype=dtype, seed=seed) * big.to(dtype), _randn(T, heads, V, dtype=dtype, seed=seed + 1)
    F_.cache_write(k, v, kc, vc, _slots(table, lens, page), ks, vs)
    return kc, vc, table, ks, vs


STORES = [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (E4M3, torch.bfloat16), (E4M3, torch.float16)]


@pytest.mark.parametrize("D,V", [(128, 128), (128, 64), (64, 64), (64, 128), (96, 80), (16, 32)])
@pytest.mark.parametrize("G,group", [(2, 1), (3, 7), (2, 16), (1, 32), (1, 33)])
@pytest.mark.parametrize("store,dtype", STORES)
def test_paged_attention(store, dtype, G, group, D, V):
    lens = [0, 1, 15, 16, 17, 63, 64, 200, 0, 777]
    kc, vc, table, ks, vs = _filled(lens, 24, G, D, V, store, dtype)
    q = _randn(len(lens), G * group, D, dtype=dtype, std=1.5, seed=5)
    got = _check(q, kc, vc, table, lens, D ** -0.5, ks, vs)
    assert (got[[0, 8]] == 0).all()


@pytest.mark.parametrize("store,dtype", STORES)
@pytest.mark.parametrize("lens,page,G,group", [
    ([40000], 16, 2, 4), ([1], 1, 1, 1), ([5], 7, 1, 128), ([3000, 2, 9001, 31], 33, 8, 5), ([1] * 300, 64, 2, 8), ([16] * 40 + [0] * 40, 16, 4, 4),
    ([100000, 1], 128, 1, 64),
])
def test_paged_attention_lengths(lens, page, G, group, store, dtype):
    kc, vc, table, ks, vs = _filled(lens, page, G, 128, 128, store, dtype)
    q = _randn(len(lens), G * group, 128, dtype=dtype, seed=5)
    _check(q, kc, vc, table, lens, 0.11, ks, vs)


@pytest.mark.parametrize("store,dtype", STORES)
@pytest.mark.parametrize("scale", [-0.3, 0.0, 4.0])
def test_paged_attention_scales(scale, store, dtype):
    lens = [70, 300]
    kc, vc, table, ks, vs = _filled(lens, 16, 2, 64, 64, store, dtype)
    _check(_randn(2, 8, 64, dtype=dtype, seed=5), kc, vc, table, lens, scale, ks, vs)


def test_paged_attention_powers_far_apart():
    """Rows of a quantised cache whose powers differ by 2^40, the weight on the small ones, and query heads of any size."""
    lens, page = [90], 16
    table, pages = _tables(lens, page)
    (kc, ks), (vc, vs) = _blank(pages, page, 1, 64, E4M3), _blank(pages, page, 1, 64, E4M3)
    power = torch.logspace(-20, 20, 90, base=2, device="cuda")[:, None, None]
    k, v = _randn(90, 1, 64, dtype=torch.float32), _randn(90, 1, 64, dtype=torch.float32, seed=1) * power
    k = (k - 3 * torch.arange(90, device="cuda")[:, None, None] / 90 * torch.ones(64, device="cuda") * 0.2).to(torch.bfloat16)
    F_.cache_write(k, v.to(torch.bfloat16), kc, vc, _slots(table, lens, page), ks, vs)
    q = (torch.ones(1, 8, 64, device="cuda") * torch.logspace(-30, 30, 8, base=2, device="cuda")[:, None]).to(torch.bfloat16)
    for head in range(8):
        _check(q[:, head:head + 1].contiguous(), kc, vc, table, lens, 0.5 / 2.0 ** (-30 + 60 * head / 7), ks, vs)


def test_paged_attention_of_latent_rows():
    """Values that are the first columns of the key rows, one key head for all, and queries that are columns of something wider."""
    lens, page = [100, 33, 500], 32
    table, pages = _tables(lens, page)
    kc = torch.full((pages, page, 1, 128), math.nan, dtype=torch.bfloat16, device="cuda")
    F_.cache_write(_randn(633, 1, 128), None, kc, None, _slots(table, lens, page))
    q = _randn(3, 32, 256, seed=2)[..., 64:192]
    _check(q, kc, kc[..., :64], table, lens, 0.09)


@pytest.mark.parametrize("store", [torch.bfloat16, E4M3])
def test_paged_attention_of_a_cache_behind_32_bits(store):
    """Rows more than 2^32 bytes (and 2^31 elements) into the cache."""
    page, G, D = 64, 8, 128
    pages = 70000 if store == E4M3 else 35000
    kc, vc = (torch.empty(pages, page, G, D, dtype=torch.uint8 if store == E4M3 else store, device="cuda") for _ in range(2))
    ks = vs = None
    if store == E4M3:
        kc, vc = kc.view(E4M3), vc.view(E4M3)
        ks, vs = (torch.full((pages, page, G), 127, dtype=torch.uint8, device="cuda") for _ in range(2))
    lens = [150]
    table = _i32([[pages - 1, 0, pages - 2]])
    F_.cache_write(_randn(150, G, D), _randn(150, G, D, seed=1), kc, vc, _slots(table, lens, page), ks, vs)
    _check(_randn(1, 32, D, seed=2), kc, vc, table, lens, D ** -0.5, ks, vs)
    got = F_.cache_read(kc, vc, table, _i32([0, 150]), 150, ks, vs)
    assert all(torch.equal(a, b) for a, b in zip(got, ref.cache_read(kc, vc, table, _i32([0, 150]), 150, ks, vs, torch.bfloat16)))


@pytest.mark.parametrize("form", ["long pages", "places first"])
def test_places_of_a_page_far_apart(form):
    """Tokens of one page more than 2^31 bytes apart: pages of a million tokens, and a cache laid out [page, pages, heads, width]."""
    G, D = 8, 128
    if form == "long pages":
        page, pages = 1050000, 2
        kc, vc = (torch.empty(pages, page, G, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        lens, ends, table, first = [page + 70], [0, page + 70], _i32([[1, 0]]), page - 100
    else:
        page, pages = 32, 70000
        kc, vc = (torch.empty(page, pages, G, D, dtype=torch.bfloat16, device="cuda").transpose(0, 1) for _ in range(2))
        lens, ends, table, first = [100], [0, 100], _i32([[pages - 1, 0, 3, pages - 2]]), 0
    assert (page - 1) * kc.stride(1) * 2 > 2 ** 31
    n = lens[0] - first                                       # the tokens that are written; the others hold zeros
    if first:
        kc.zero_()
        vc.zero_()
    k, v = _randn(n, G, D), _randn(n, G, D, seed=1)
    pos = torch.arange(first, lens[0], device="cuda")
    F_.cache_write(k, v, kc, vc, table[0].long()[pos // page] * page + pos % page)
    got = F_.cache_read(kc, vc, table, _i32(ends), lens[0])
    assert torch.equal(got[0][first:], k) and torch.equal(got[1][first:], v) and not got[0][:first].any()
    q = _randn(1, 32, D, seed=2)
    o = F_.paged_attention(q, kc, vc, table, _i32(lens), 0.5)
    (k_all, v_all), heads = (t.double() for t in got), q[0].double().view(G, 4, D)
    for g in range(G):
        s = heads[g] @ k_all[:, g].T * 0.5
        p = torch.softmax(s, 1)
        e = 2 * ((D + 8) * 2.0 ** -23 * (heads[g].abs() @ k_all[:, g].abs().T * 0.5)).amax(1, keepdim=True) + 2.0 ** -19 + lens[0] * 2.0 ** -23
        want, size = p @ v_all[:, g], p @ v_all[:, g].abs()
        assert ((o[0].view(G, 4, D)[g].double() - want).abs() <= (2.0 ** -8 + e) * 2 * size + 2.0 ** -8 * want.abs()).all()


def test_paged_attention_same_bits_and_other_stream():
    lens = [5000, 12, 900]
    kc, vc, table, ks, vs = _filled(lens, 16, 4, 128, 128, E4M3, torch.bfloat16)
    q, n = _randn(3, 32, 128), _i32(lens)
    want = F_.paged_attention(q, kc, vc, table, n, 0.1, ks, vs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            assert torch.equal(F_.paged_attention(q, kc, vc, table, n, 0.1, ks, vs), want)
    torch.cuda.current_stream().wait_stream(side)


def test_a_step_of_generation_captured_and_replayed():
    """Write and attention in one graph, replayed for tokens and lengths that change in place; two graphs take turns."""
    page, G, H, D, most = 16, 2, 8, 64, 80
    table = torch.randperm(3 * 5, device="cuda").int().view(3, 5)
    (kc, ks), (vc, vs) = _blank(15, page, G, D, E4M3), _blank(15, page, G, D, E4M3)
    lens, slots = _i32([0, 7, 30]), torch.zeros(3, dtype=torch.int64, device="cuda")
    start = [_randn(30, G, D, seed=s) for s in (50, 51)]
    where = _slots(table, [0, 7, 30], page)
    pick = torch.cat([torch.arange(7), torch.arange(30)]).cuda()
    F_.cache_write(start[0][pick], start[1][pick], kc, vc, where, ks, vs)
    state = [{"q": _randn(3, H, D, seed=s), "k": _randn(3, G, D, seed=s + 1), "v": _randn(3, G, D, seed=s + 2)} for s in (10, 20)]

    def step(x):
        slots.copy_(table.gather(1, (lens // page).long()[:, None])[:, 0].long() * page + lens % page)
        lens.add_(1)
        F_.cache_write(x["k"], x["v"], kc, vc, slots, ks, vs)
        return F_.paged_attention(x["q"], kc, vc, table, lens, 0.125, ks, vs)

    keep = lens.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(state[0])
    torch.cuda.current_stream().wait_stream(side)
    lens.copy_(keep)
    graphs = []
    for x in state:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(x)
        graphs.append((g, out))
    lens.copy_(keep)
    for i in range(40):
        x, (g, out) = state[i % 2], graphs[i % 2]
        for n, t in enumerate(("q", "k", "v")):
            x[t].copy_(_randn(*x[t].shape, seed=100 * i + n))
        g.replay()
        got = out.clone()
        _check(x["q"], kc, vc, table, lens.tolist(), 0.125, ks, vs, got=got)
    assert int(lens.max()) == 70 <= most


def test_calls_of_nothing():
    for store in (torch.bfloat16, E4M3):
        (kc, ks), (vc, vs) = _blank(3, 16, 2, 64, store), _blank(3, 16, 2, 64, store)
        none = torch.zeros(0, 3, dtype=torch.int32, device="cuda")
        F_.cache_write(_randn(0, 2, 64), _randn(0, 2, 64), kc, vc, torch.zeros(0, dtype=torch.int64, device="cuda"), ks, vs)
        assert F_.cache_read(kc, vc, none, _i32([0]), 0, ks, vs)[0].shape == (0, 2, 64)
        assert all((t == 0).all() for t in F_.cache_read(kc, vc, none, _i32([0]), 70, ks, vs))
        assert F_.paged_attention(_randn(0, 4, 64), kc, vc, none, _i32([]), 0.1, ks, vs).shape == (0, 4, 64)
        assert (F_.paged_attention(_randn(2, 4, 64), kc, vc, none.new_zeros(2, 0), _i32([0, 0]), 0.1, ks, vs) == 0).all()
        assert (F_.paged_attention(_randn(2, 4, 64), kc, vc, none.new_zeros(2, 3), _i32([0, 0]), 0.1, ks, vs) == 0).all()
    from cppmega_b200.ops import cuda as cu
    cu.check_errors()


def test_sequences_that_share_pages():
    """One table row for several sequences (a common beginning), broadcast, at different lengths."""
    kc, vc, table, _, _ = _filled([300], 16, 2, 128, 128, torch.bfloat16, torch.bfloat16)
    lens = [300, 17, 300, 16]
    _check(_randn(4, 8, 128, seed=9), kc, vc, table.expand(4, -1), lens, 0.09)
    k, v = F_.cache_read(kc, vc, table.expand(2, -1), _i32([0, 300, 317]), 317)
    assert torch.equal(k[300:], k[:17]) and torch.equal(v[300:], v[:17])


def test_two_calls_at_once():
    lens = [3000, 1, 700]
    kc, vc, table, ks, vs = _filled(lens, 16, 4, 128, 128, E4M3, torch.bfloat16)
    qs, n = [_randn(3, 32, 128, seed=s) for s in (5, 6)], _i32(lens)
    want = [F_.paged_attention(q, kc, vc, table, n, 0.1, ks, vs) for q in qs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(30):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, F_.paged_attention(qs[i], kc, vc, table, n, 0.1, ks, vs)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i, o in got)


def test_a_cache_that_was_saved_for_a_gradient_and_written():
    kc, vc, table, _, _ = _filled([20], 16, 2, 64, 64, torch.bfloat16, torch.bfloat16)
    q = _randn(1, 4, 64).requires_grad_()
    o = F_.paged_attention(q, kc, vc, table, _i32([20]), 0.1)
    before = kc._version
    F_.cache_write(_randn(1, 2, 64), _randn(1, 2, 64), kc, vc, torch.tensor([3], device="cuda"))
    assert kc._version == before + 1 and o.isfinite().all()
    with torch.inference_mode():
        a, b = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
        F_.cache_write(_randn(1, 2, 64), _randn(1, 2, 64), a, b, torch.tensor([3], device="cuda"))
        assert a.abs().sum() > 0
    F_.cache_write(_randn(1, 2, 64), _randn(1, 2, 64), a, b, torch.tensor([9], device="cuda"))       # and outside of that mode
    assert a.view(32, -1).abs().sum(1).nonzero().flatten().tolist() == [3, 9]
    q = _randn(1, 4, 64)
    assert F_.paged_attention(q, a, b, _i32([[0]]), _i32([10]), 0.1).isfinite().all()


@pytest.mark.parametrize("scale", [math.inf, math.nan])
def test_scales_that_are_not_finite_run_the_definition(scale):
    kc, vc, table, _, _ = _filled([20], 16, 2, 64, 64, torch.bfloat16, torch.bfloat16)
    F_.reset_counters()
    assert F_.paged_attention(_randn(1, 4, 64), kc, vc, table, _i32([20]), scale).isnan().any()
    assert F_.fallback_counts() == {"paged_attention(shape/dtype)": 1}


def test_paged_attention_for_a_gradient_is_the_definition():
    lens = [20, 3]
    kc, vc, table, _, _ = _filled(lens, 16, 2, 64, 64, torch.bfloat16, torch.bfloat16)
    q = _randn(2, 4, 64).requires_grad_()
    F_.reset_counters()
    o = F_.paged_attention(q, kc, vc, table, _i32(lens), 0.1)
    assert F_.fallback_counts() == {"paged_attention(shape/dtype)": 1} and torch.autograd.grad(o.sum(), q)[0].abs().max() > 0


# ---- calls that are reported --------------------------------------------------------------------------------------------

def _reported():
    from cppmega_b200.ops import cuda as cu
    with pytest.raises(cu.KernelError, match="bad argument"):
        cu.check_errors()
    cu.check_errors()


@pytest.mark.parametrize("bad", [-1, 5, 2 ** 31 - 1, -2 ** 31])
def test_pages_outside_the_cache_are_left_out_and_reported(bad):
    kc, vc = _randn(5, 16, 2, 64), _randn(5, 16, 2, 64, seed=1)
    table = _i32([[1, bad, 3], [0, 2, 4]])
    got = F_.paged_attention(_randn(2, 4, 64), kc, vc, table, _i32([40, 48]), 0.1)
    _reported()
    assert got.isfinite().all()
    k, _ = F_.cache_read(kc, vc, table, _i32([0, 40, 88]), 88)
    _reported()
    assert (k[16:32] == 0).all() and torch.equal(k[:16], kc[1]) and torch.equal(k[32:40], kc[3, :8]) and torch.equal(k[40:56], kc[0])


@pytest.mark.parametrize("n", [-1, 49, 2 ** 31 - 1, -2 ** 31])
def test_lengths_outside_the_table_are_reported(n):
    kc, vc = _randn(5, 16, 2, 64), _randn(5, 16, 2, 64, seed=1)
    got = F_.paged_attention(_randn(2, 4, 64), kc, vc, _i32([[1, 4, 3], [0, 2, 4]]), _i32([n, 48]), 0.1)
    _reported()
    assert got.isfinite().all()


@pytest.mark.parametrize("ends", [[0, 40, 30], [0, 40, 89], [1, 40, 80], [-3, 40, 80], [0, 2 ** 31 - 1, 80], [0, 40, -2 ** 31]])
def test_read_with_ends_that_do_not_hold_is_reported(ends):
    kc, vc = _randn(5, 16, 2, 64), _randn(5, 16, 2, 64, seed=1)
    k, v = F_.cache_read(kc, vc, _i32([[1, 4, 3], [0, 2, 4]]), _i32(ends), 88)
    _reported()
    assert k.isfinite().all() and v.isfinite().all()


@pytest.mark.parametrize("slot", [32, 2 ** 40])
def test_slots_behind_the_cache_are_skipped_and_reported(slot):
    kc = torch.zeros(2, 16, 1, 8, dtype=torch.bfloat16, device="cuda")
    F_.cache_write(torch.ones(3, 1, 8, dtype=torch.bfloat16, device="cuda"), None, kc, None, torch.tensor([3, slot, 31], device="cuda"))
    _reported()
    assert kc.view(32, 8).sum(1).nonzero().flatten().tolist() == [3, 31]


def test_forms_without_a_kernel_run_the_definition():
    lens = [20, 3]
    table, pages = _tables(lens, 16)
    kc, vc = (torch.zeros(pages, 16, 2, 12, device="cuda") for _ in range(2))
    k = _randn(23, 2, 12, dtype=torch.float32)
    F_.reset_counters()
    F_.cache_write(k, -k, kc, vc, _slots(table, lens, 16))
    rk, rv = F_.cache_read(kc, vc, table, _i32([0, 20, 23]), 23)
    assert torch.equal(rk, k) and torch.equal(rv, -k)
    o = F_.paged_attention(_randn(2, 2, 12, dtype=torch.float32), kc, vc, table, _i32(lens), 0.1)
    assert o.isfinite().all() and sum(F_.fallback_counts().values()) == 3 and not F_.launch_counts()
