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
