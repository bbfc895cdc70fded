"""The paged key-value cache and the attentions beside it on the CPU: calls at the edges of what they take.  Where the kernels would be reached, a
library of Python functions stands in for them and sees what it is given."""
import ctypes
import types

import pytest
import torch

from cppmega_b200.ops import functional as F_
from cppmega_b200.ops import reference as ref
from cppmega_b200.ops.cuda import packed, paged


def _i32(*values):
    return torch.tensor(values, dtype=torch.int32)


def _randn(*shape, dtype=torch.bfloat16, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.fixture
def kernels(monkeypatch):
    """The wrappers on CPU tensors; ``kernels.name = function`` stands in for an entry of the library."""
    library = types.SimpleNamespace()
    for module in (paged, packed):
        monkeypatch.setattr(module._cu, "lib", lambda: library)
        monkeypatch.setattr(module._cu, "err_word", lambda dev=None: torch.zeros(1, dtype=torch.int32))
        monkeypatch.setattr(module._cu, "stream_ptr", lambda: 0)
    monkeypatch.setattr(F_, "_cuda", lambda name, t: {"cache_write": paged.cache_write, "cache_read": paged.cache_read,
                                                      "paged_attention": paged.paged_attention, "packed_attention": packed.packed_attention}[name])
    monkeypatch.setattr(paged, "_plans", {})
    return library


def _bits_at(pointer, like):
    """The bits of a packed tensor of ``like``'s shape that begins at an address."""
    return torch.frombuffer(bytearray(ctypes.string_at(pointer, like.numel() * like.element_size())), dtype=like.dtype).view(like.shape)


# ---- rows that lie in the cache they are written to ----------------------------------------------------------------------

@pytest.mark.parametrize("case", ["k in k_cache", "v in k_cache", "k in v_cache", "v in v_cache", "apart", "no values"])
def test_rows_of_the_cache_are_copied_before_it_is_written(kernels, case):
    kc, vc = _randn(4, 8, 2, 16), _randn(4, 8, 2, 16, seed=1)
    k, v = _randn(16, 2, 16, seed=2), _randn(16, 2, 16, seed=3)
    k = {"k in k_cache": kc, "k in v_cache": vc, "no values": kc}[case].view(32, 2, 16)[3:19] if case[0] == "k" or case == "no values" else k
    v = {"v in k_cache": kc, "v in v_cache": vc}[case].view(32, 2, 16)[3:19] if case[0] == "v" else v
    if case == "no values":
        v = vc = None
    seen = []

    def write(kp, vp, kcp, vcp, *rest):
        seen.append((kp, vp))
        assert torch.equal(_bits_at(kp, k), k) and (v is None or torch.equal(_bits_at(vp, v), v))
        return 0

    kernels.cm_cache_write = write
    F_.cache_write(k, v, kc, vc, torch.arange(16))
    (kp, vp), = seen
    ranges = [(t.data_ptr(), t.data_ptr() + t.numel() * 2) for t in (kc, vc) if t is not None]
    for p in (kp, vp):
        assert p is None or not any(a - 16 * 32 * 2 < p < b for a, b in ranges) or case == "apart"
    if case == "apart":
        assert (kp, vp) == (k.data_ptr(), v.data_ptr())


@pytest.mark.parametrize("swap", [False, True])
def test_the_definition_takes_rows_of_the_cache_as_they_were(swap):
    kc, vc = _randn(4, 8, 2, 16), _randn(4, 8, 2, 16, seed=1)
    was = [t.clone().view(32, 2, 16) for t in (kc, vc)]
    k, v = (t.view(32, 2, 16)[:31] for t in ((vc, kc) if swap else (kc, vc)))
    F_.cache_write(k, v, kc, vc, torch.arange(1, 32))
    for got, rows, old in zip((kc, vc), reversed(was) if swap else was, was):
        assert torch.equal(got.view(32, 2, 16)[1:], rows[:31]) and torch.equal(got.view(32, 2, 16)[0], old[0])


# ---- caches whose rows share memory ----------------------------------------------------------------------------------------

def _bytes_of(t):
    """Every byte that a tensor's elements hold, as often as they hold it."""
    at = torch.zeros(1, dtype=torch.long)
    for n, s in zip(t.shape, t.stride()):
        at = (at[:, None] + torch.arange(n) * s).view(-1)
    es = t.element_size()
    return (t.data_ptr() + at[:, None] * es + torch.arange(es)).view(-1).tolist()


def test_memory_that_two_tensors_share():
    """Against the bytes themselves, for views of one buffer with any steps: nothing that shares memory is missed, and views whose axes have the
    same steps, or lie in one piece inside each other's, are told exactly."""
    g = torch.Generator().manual_seed(5)
    buffers = {torch.int16: torch.zeros(600, dtype=torch.int16), torch.uint8: torch.zeros(1200, dtype=torch.uint8)}
    nested = same = 0
    for _ in range(4000):
        dtype = torch.int16 if torch.rand(1, generator=g) < 0.7 else torch.uint8
        views = []
        steps = [int(torch.randint(0, 40, (1,), generator=g)) for _ in range(3)] + [1]
        for i in range(2):
            if i and torch.rand(1, generator=g) < 0.5:
                steps = [int(torch.randint(0, 40, (1,), generator=g)) for _ in range(3)] + [1]
            shape = torch.randint(1, 5, (4,), generator=g).tolist()
            views.append(buffers[dtype].as_strided(shape, steps, int(torch.randint(0, 150, (1,), generator=g))))
        a, b = views
        for t in views:
            held = _bytes_of(t)
            if F_._nested(t):
                nested += 1
                assert len(set(held)) == len(held)
        meet = bool(set(_bytes_of(a)) & set(_bytes_of(b)))
        if F_._nested(a) and F_._nested(b):
            same += meet
            assert F_._share_memory(a, b) == meet and F_._share_memory(b, a) == meet
    assert nested > 500 and same > 50


@pytest.mark.parametrize("case", ["heads overlap", "tokens overlap", "one cache for both", "columns of one another", "shifted by a row", "scales of both",
                                  "scale broadcast"])
def test_caches_that_share_memory_are_refused(case):
    e4m3 = torch.float8_e4m3fn
    k = v = torch.ones(3, 2, 16)
    kc, vc, ks, vs = torch.zeros(4, 8, 2, 16), torch.zeros(4, 8, 2, 16), None, None
    if case == "heads overlap":
        kc = torch.zeros(600).as_strided((4, 8, 2, 16), (128, 16, 8, 1))
    elif case == "tokens overlap":
        kc = torch.zeros(4000).as_strided((4, 8, 2, 16), (512, 24, 16, 1))
    elif case == "one cache for both":
        vc = kc
    elif case == "columns of one another":
        v, vc = v[..., :8], kc[..., 8:]
    elif case == "shifted by a row":
        both = torch.zeros(5, 8, 2, 16)
        kc, vc = both[:4], both.view(40, 2, 16)[1:33].view(4, 8, 2, 16)
    else:
        kc, vc = (torch.zeros(4, 8, 2, 16, dtype=torch.uint8).view(e4m3) for _ in range(2))
        ks = vs = torch.zeros(4, 8, 2, dtype=torch.uint8)
        if case == "scale broadcast":
            ks, vs = torch.zeros(4, 8, 1, dtype=torch.uint8).expand(4, 8, 2), vs.clone()
    for _ in range(2):
        with pytest.raises(ValueError, match="overlap|share memory"):
            F_.cache_write(k, v, kc, vc, torch.tensor([0, 5, 7]), ks, vs)


@pytest.mark.parametrize("case", ["stacked in a page", "columns side by side", "heads side by side", "blocks of a page in two orders", "places first",
                                  "one buffer, two halves"])
def test_caches_that_lie_between_one_another_are_taken(case):
    k, v = torch.ones(3, 2, 16), torch.full((3, 2, 16), 2.0)
    if case == "stacked in a page":
        both = torch.zeros(4, 2, 8, 2, 16)
        kc, vc = both[:, 0], both[:, 1]
    elif case == "columns side by side":
        both = torch.zeros(4, 8, 2, 40)
        kc, vc = both[..., :16], both[..., 24:]
    elif case == "heads side by side":
        both = torch.zeros(4, 8, 5, 16)
        kc, vc = both[:, :, :2], both[:, :, 3:]
    elif case == "blocks of a page in two orders":
        both = torch.zeros(4, 512)
        kc, vc = both[:, :256].view(4, 8, 2, 16), both[:, 256:].view(4, 2, 8, 16).transpose(1, 2)
    elif case == "places first":
        both = torch.zeros(8, 4, 2, 2, 16)
        kc, vc = both[:, :, 0].transpose(0, 1), both[:, :, 1].transpose(0, 1)
    else:
        both = torch.zeros(8, 8, 2, 16)
        kc, vc = both[:4], both[4:]
    for _ in range(2):
        F_.cache_write(k, v, kc, vc, torch.tensor([0, 9, 31]))
    assert float(kc.sum()) == k.numel() and float(vc.sum()) == 2 * v.numel() and float(both.sum()) == 3 * k.numel()


# ---- attention over packed sequences -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("wanted", [[0, 1, 2], [1], [0, 2]])
def test_batched_upstream_gradients_of_the_packed_attention(kernels, wanted):
    """Under ``is_grads_batched`` the upstream gradient has no memory that a kernel could read: the definition's gradients, one row of the batch
    after the other."""
    kernels.cm_packed_attention_ws = lambda at: 0
    kernels.cm_packed_attention_fwd = lambda *args: 0
    ends, ends_k = _i32(0, 5, 9), _i32(0, 7, 11)
    leaves = [_randn(n, h, 16, seed=s).requires_grad_(s in wanted) for s, n, h in ((0, 9, 4), (1, 11, 2), (2, 11, 2))]
    some = [leaves[i] for i in wanted]
    go = _randn(3, 9, 4, 16, seed=3)
    o = F_.packed_attention(*leaves, ends, 0.25, ends_k)
    got = torch.autograd.grad(o, some, go, is_grads_batched=True)
    for i in range(3):
        want = torch.autograd.grad(ref.packed_attention(*leaves, ends, 0.25, ends_k), some, go[i])
        # the same sums in another order in fp32, then one rounding
        assert all(((a[i].double() - b.double()).abs() <= 2.0 ** -7 * b.double().abs() + 2.0 ** -16).all() for a, b in zip(got, want))


# ---- caches and calls of nothing ---------------------------------------------------------------------------------------------

def test_paged_attention_over_a_cache_of_no_pages_names_memory_that_is_there(kernels):
    seen = []
    kernels.cm_paged_attention_ws = lambda *sizes: 0
    kernels.cm_paged_attention = lambda *args: seen.append(args) or 0
    q, none = _randn(2, 4, 16), torch.zeros(0, 8, 2, 16, dtype=torch.bfloat16)
    F_.paged_attention(q, none, none, torch.zeros(2, 3, dtype=torch.int32), _i32(5, 0), 0.25)
    assert seen[0][:3] == (q.data_ptr(),) * 3


@pytest.mark.parametrize("store", [torch.float32, torch.float8_e4m3fn])
def test_the_definitions_over_a_cache_of_no_pages(store):
    """No page is looked up, in a table that has columns either."""
    kc, vc = (torch.zeros(0, 8, 2, n, dtype=torch.uint8).view(store) if store != torch.float32 else torch.zeros(0, 8, 2, n) for n in (16, 24))
    ks = vs = None if store == torch.float32 else torch.zeros(0, 8, 2, dtype=torch.uint8)
    table = torch.tensor([[0, -1, 3], [5, 5, 5]], dtype=torch.int32)
    q = _randn(2, 4, 16, dtype=torch.float32).requires_grad_()
    o = F_.paged_attention(q, kc, vc, table, _i32(0, 0), 1.0, ks, vs)
    assert o.shape == (2, 4, 24) and (o == 0).all() and (torch.autograd.grad(o.sum(), q)[0] == 0).all()
    k, v = F_.cache_read(kc, vc, table, _i32(0, 0, 0), 5, ks, vs)
    assert k.shape == (5, 2, 16) and v.shape == (5, 2, 24) and not k.any() and not v.any()
    F_.cache_write(torch.ones(3, 2, 16), torch.ones(3, 2, 24), kc, vc, torch.full((3,), -1), ks, None if vs is None else vs.clone())
    with pytest.raises(ValueError, match="outside the cache"):
        F_.paged_attention(q, kc, vc, table, _i32(0, 1), 1.0, ks, vs)


@pytest.mark.parametrize("shape", [(0, 4), (3, 0), (0, 0), (2, 4)])
def test_tables_whose_entries_lie_apart(kernels, shape):
    """Every other column of a wider table: copied, and where it has no entries there is nothing to copy."""
    seen = []
    kernels.cm_paged_attention_ws = lambda *sizes: 0
    kernels.cm_paged_attention = lambda *args: seen.append(args) or 0
    kernels.cm_cache_read = lambda *args: seen.append(args) or 0
    kc = _randn(4, 8, 2, 16)
    n, columns = shape
    table = torch.arange(4 * 10, dtype=torch.int32).view(4, 10)[:n, :2 * columns:2]
    assert F_.paged_attention(_randn(n, 4, 32)[..., 8:24], kc, kc, table, torch.zeros(2 * n, dtype=torch.int32)[::2], 0.25).shape == (n, 4, 16)
    ends = torch.zeros(n + 1, dtype=torch.int32)
    assert F_.cache_read(kc, kc, table, ends, 3)[0].shape == (3, 2, 16)
    assert len(seen) == 2


def test_a_number_of_rows_that_changes_in_place(kernels):
    """A tensor of no axes may say how many rows are read: its value at the call counts, not the tensor."""
    seen = []
    kernels.cm_cache_read = lambda *args: seen.append((ctypes.c_longlong * 11).from_address(args[8])[10]) or 0
    kc, total = _randn(4, 8, 2, 16), torch.tensor(3)
    for rows in (3, 7):
        total.fill_(rows)
        assert F_.cache_read(kc, None, torch.zeros(1, 2, dtype=torch.int32), _i32(0, 2), total)[0].shape == (rows, 2, 16)
    assert seen == [3, 7]                                       # the rows that the kernel is told to write
    with pytest.raises(TypeError):
        F_.cache_read(kc, None, torch.zeros(1, 2, dtype=torch.int32), _i32(0, 2), 3.0)


@pytest.mark.parametrize("T,Tk,H", [(0, 0, 4), (0, 7, 4), (7, 0, 4), (7, 7, 0)])
def test_packed_attention_of_nothing_looks_at_its_ends_on_the_device(kernels, monkeypatch, T, Tk, H):
    """No rows of queries, of keys, or no heads: one look at the ends, zeros, and nothing that waits for their values."""
    seen = []
    kernels.cm_packed_attention_ends = lambda *args: seen.append(args) or 0
    monkeypatch.setattr(F_.ref, "packed_attention", None)
    cu, cu_k = torch.tensor([0, -9, 0, -9, T], dtype=torch.int32)[::2], _i32(0, 0, Tk)
    leaves = [_randn(n, h, 16, seed=s).requires_grad_() for s, n, h in ((0, T, H), (1, Tk, 2), (2, Tk, 2))]
    o = F_.packed_attention(*leaves, cu, -0.5, cu_k)
    assert len(seen) == 1 and seen[0][2:5] == (2, T, Tk) and o.shape == (T, H, 16) and not o.any()
    assert all(g.shape == t.shape and not g.any() for g, t in zip(torch.autograd.grad(o.sum(), leaves), leaves))


@pytest.mark.parametrize("wanted", [[0], [1], [2], [0, 2], [0, 1, 2]])
def test_packed_gradients_that_nobody_asks_for_have_no_memory(kernels, wanted):
    seen = []
    kernels.cm_packed_attention_ws = lambda at: 0
    kernels.cm_packed_attention_fwd = lambda *args: 0
    kernels.cm_packed_attention_bwd = lambda *args: seen.append(args[10:13]) or 0
    leaves = [_randn(9, h, 16, seed=s).requires_grad_(s in wanted) for s, h in ((0, 4), (1, 2), (2, 2))]
    o = F_.packed_attention(*leaves, _i32(0, 5, 9), 0.25)
    grads = torch.autograd.grad(o, [leaves[i] for i in wanted], torch.ones_like(o))
    (dq, dk, dv), = seen
    assert (dq is not None) == (0 in wanted) and (dk is not None) == (dv is not None) == bool({1, 2} & set(wanted))
    assert [g.shape for g in grads] == [leaves[i].shape for i in wanted]


def test_interleaved_caches_are_looked_at_once_for_a_distance(kernels, monkeypatch):
    """Keys and values in one buffer: their memory is compared once for each way that two tensors of these shapes lie, and again where they lie another
    way, with the kernels as with the definition."""
    compared = []
    share = F_._share_memory
    monkeypatch.setattr(F_, "_share_memory", lambda a, b: compared.append(1) or share(a, b))
    kernels.cm_cache_write = lambda *args: 0
    both, k = torch.zeros(4, 8, 3, 2, 16, dtype=torch.bfloat16), _randn(3, 2, 16)
    slots = torch.tensor([0, 9, 31])
    for _ in range(3):
        F_.cache_write(k, k, both[:, :, 0], both[:, :, 1], slots)
    assert len(compared) == 1
    for _ in range(3):
        F_.cache_write(k, k, both[:, :, 0], both[:, :, 2], slots)
    assert len(compared) == 2
    for _ in range(2):
        with pytest.raises(ValueError, match="share memory"):
            F_.cache_write(k, k, both[:, :, 0], both[:, :, 0], slots)
    e4m3 = both.view(torch.uint8).view(torch.float8_e4m3fn)[..., :16]
    one = torch.zeros(4, 8, 2, dtype=torch.uint8)
    for _ in range(2):
        with pytest.raises(ValueError, match="share memory"):
            F_.cache_write(k, k, e4m3[:, :, 0], e4m3[:, :, 1], slots, one, one)
