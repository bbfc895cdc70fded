"""The paged key-value cache and the attentions beside it on the CPU: calls at the edges of what they take.  Where the kernels would be reached, a
library of Python functions stands in for them and sees what it is given."""
import ctypes
import types

import pytest
import torch

from cppmega_b200.ops import functional as F_
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
