"""The operators around a dense block on the CPU: definitions, refusals, and what the GPU wrappers do with strides."""
import pytest
import torch

from cppmega_b200.ops import functional as F_
from cppmega_b200.ops import reference as ref


def _r(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + sum(shape)), dtype=torch.float64)


def test_residual_rmsnorm_definition():
    y, x, w, pw, gate = _r(3, 5, 24), _r(3, 5, 24, seed=1), _r(24), _r(24, seed=2), _r(24, seed=3)
    n, h = (t.double() for t in F_.residual_rmsnorm(y.float(), x.float(), w.float(), pw.float(), gate.float(), 0.5))
    p = y / (y.square().mean(-1, keepdim=True) + 1e-5).sqrt() * pw * gate
    want = x + 0.5 * p
    assert (h - want).abs().max() < 32 * 2 ** -24 * want.abs().max()
    wn = want / (want.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w
    assert (n - wn).abs().max() < 32 * 2 ** -24 * wn.abs().max()


def test_residual_rmsnorm_is_add_and_norm():
    y, x, w = _r(7, 16).float(), _r(7, 16, seed=1).float(), _r(16).float()
    n, h = F_.residual_rmsnorm(y, x, w)
    assert torch.equal(h, x + y) and torch.equal(n, F_.rmsnorm(x + y, w))


@pytest.mark.parametrize("name", ["silu", "gelu_tanh", "relu"])
def test_gated_mlp_definition(name):
    x, w1, w2 = _r(4, 6, 16).float(), _r(40, 16).float(), _r(16, 20).float()
    got = F_.gated_mlp(x, w1, w2, name)
    want = ref.gated_mlp(x, w1, w2, name)
    assert got.shape == (4, 6, 16) and torch.allclose(got, want, rtol=1e-5, atol=1e-4)


def test_zero_rows():
    x, w = torch.zeros(0, 16, requires_grad=True), torch.ones(16)
    for out in (*F_.residual_rmsnorm(x, x, w), F_.rmsnorm_gated(x, w, x), F_.gated_mlp(x, torch.ones(24, 16), torch.ones(16, 12))):
        assert out.shape == (0, 16)
        assert torch.autograd.grad(out.sum(), x, retain_graph=True)[0].shape == (0, 16)


@pytest.mark.parametrize("call", [
    lambda x, w: F_.residual_rmsnorm(x, x[:2], w),
    lambda x, w: F_.residual_rmsnorm(x, x, w[:3]),
    lambda x, w: F_.residual_rmsnorm(x, x, w, post_weight=w[:1]),
    lambda x, w: F_.residual_rmsnorm(x, x, w, gate=x[:, :1]),
    lambda x, w: F_.residual_rmsnorm(x, x, w, gate=x[0, 0]),
    lambda x, w: F_.residual_rmsnorm(x, x, w.to("meta")),
    lambda x, w: F_.gated_mlp(x, torch.ones(24, 15), torch.ones(16, 12)),
    lambda x, w: F_.gated_mlp(x, torch.ones(25, 16), torch.ones(16, 12)),
    lambda x, w: F_.gated_mlp(x, torch.ones(24, 16), torch.ones(16, 24)),
    lambda x, w: F_.gated_mlp(x, torch.ones(24, 16), torch.ones(16, 12), activation="tanh"),
    lambda x, w: F_.gated_mlp(x, torch.ones(2, 24, 16), torch.ones(16, 12)),
    lambda x, w: F_.gated_mlp(x, torch.ones(24, 16), torch.ones(16, 12, device="meta")),
])
def test_refusals(call):
    with pytest.raises(ValueError):
        call(torch.ones(4, 16), torch.ones(16))


def test_rows_view():
    """Rows of any even spacing are taken in place, anything else is copied."""
    from cppmega_b200.ops.cuda.block import _rows
    base = torch.arange(2 * 6 * 20.0).view(2, 6, 20)
    for t, pitch, same in ((base, 20, True), (base[..., 4:12], 20, True), (base[:, ::2, :8], 40, True), (base[:1, :1, 3:9], None, True),
                           (base[:, :3], 20, False), (base.transpose(0, 1), 20, False), (base[..., ::2], 10, False),
                           (base[0, 0].expand(5, 20), 20, False), (base[..., :1], 20, True), (base[0, 0], 20, True)):
        got, p = _rows(t)
        assert torch.equal(got, t)
        assert (got.data_ptr() == t.data_ptr()) == same
        if pitch is not None:
            assert p == (pitch if same else t.shape[-1])
        width = t.shape[-1]
        flat = torch.as_strided(got, (t.numel() // width, width), (p, 1), got.storage_offset())
        assert torch.equal(flat, t.reshape(-1, width))


def test_wide_or_mixed_types_are_left_to_the_definition():
    from cppmega_b200.ops.cuda import block
    x, w = torch.ones(2, 16, dtype=torch.bfloat16), torch.ones(16)
    assert block.residual_rmsnorm(x, x, w, None, None, 1.0, 1e-5) is None
    assert block.rmsnorm_gated(x, w, None, 1e-5, 16, True) is None
    wide = torch.ones(1, 16385, dtype=torch.bfloat16)
    assert block.residual_rmsnorm(wide, wide, wide[0], None, None, 1.0, 1e-5) is None
    assert block.rmsnorm_gated(wide, wide[0], None, 1e-5, 16385, True) is None
    assert block.gated_mlp(x, torch.ones(24, 16), torch.ones(16, 12), "silu") is None
    assert block.gated_mlp(x[:, :12], torch.ones(16, 12).bfloat16(), torch.ones(16, 8).bfloat16(), "silu") is None


def test_kernel_entry_points_refuse():
    """Argument checks of the C entries; nothing is launched."""
    from cppmega_b200.ops.cuda import lib
    L = lib()
    assert L.cm_gated_mlp_fwd(16, 12, 16, 16, None, 16, 16, 16, 4, 12, 8, 8, 0, None, None) == -10        # width of 12
    assert L.cm_gated_mlp_fwd(8, 16, 16, 16, None, 16, 16, 16, 4, 16, 8, 8, 0, None, None) == -10         # base not on 16 bytes
    assert L.cm_gated_mlp_fwd(16, 12, 16, 16, None, 16, 16, 16, 4, 8, 8, 8, 0, None, None) == -10         # row pitch of 12
    assert L.cm_gated_mlp_fwd(16, 16, 16, 16, None, 16, 16, 16, 0, 16, 8, 8, 0, None, None) == 0          # no tokens
    assert L.cm_residual_rmsnorm_fwd(16, 8, 16, 8, 16, None, None, 0, 16, 16, None, None, 2, 8, 1.0, 1e-5, 3, None) == -10     # no such type
    assert L.cm_residual_rmsnorm_fwd(16, 8, 16, 8, 16, None, None, 0, 16, 16, None, None, 2, 40000, 1.0, 1e-5, 0, None) == -10  # too wide
    assert L.cm_rmsnorm_gated_fwd(16, 8, None, 0, 16, 16, None, 2, 8, 3, 0, 1e-5, 0, None) == -10     # groups that do not divide
    assert L.cm_rmsnorm_gated_fwd(16, 8, None, 0, 16, 16, None, 2, 8, 0, 0, 1e-5, 0, None) == -10
    assert L.cm_rmsnorm_gated_fwd(16, 8, None, 0, 16, 16, None, 0, 8, 8, 0, 1e-5, 0, None) == 0


@pytest.mark.parametrize("M,N,K,b_mn", [(4095, 3584, 18944, 0), (4095, 3584, 37888, 1), (512, 1024, 2048, 0), (512, 1024, 4096, 1), (300, 136, 1032, 0),
                                        (16384, 4096, 21504, 0), (1, 8, 8, 0), (2064, 72, 300, 1), (257, 4096, 4096, 1), (20000, 264, 512, 0),
                                        (4096, 1024, 512, 1), (43008, 4096, 16384, 1), (700, 1000, 20000, 1)])
def test_split_plan(M, N, K, b_mn):
    """Every row and every k block is worked on once, by runs that are not empty, and no wave of runs is left over."""
    import ctypes
    from cppmega_b200.ops.cuda import lib
    L = lib()
    out = (ctypes.c_int * 4)()
    floats = L.cm_gemm_split_plan(148, M, N, K, b_mn, out)
    whole, bn, slices, per = out
    if slices == 0:
        assert (whole, floats) == (M, 0)
        return
    nkb = -(-K // 64)
    assert 0 <= whole < M and whole % 256 == 0 and bn in (128, 256) and slices >= 2
    assert slices * per >= nkb > (slices - 1) * per
    assert -(-(M - whole) // 256) * -(-N // bn) * slices <= 74
    assert floats == slices * (M - whole) * N


def test_split_plan_takes_the_products_it_is_for():
    import ctypes
    from cppmega_b200.ops.cuda import lib
    out = (ctypes.c_int * 4)()
    took = []
    for args in ((4095, 3584, 18944, 0), (512, 1024, 4096, 1), (16384, 4096, 21504, 0)):
        lib().cm_gemm_split_plan(148, *args, out)
        took.append(out[2] > 0)
    assert took == [True, True, False]


def _mlp():
    from cppmega_b200.models.common import DenseMLP
    from cppmega_b200.parallel.state import single_process_context
    m = DenseMLP(32, 48, single_process_context(), std=0.1, out_std=0.1, dtype=torch.float32, seed=3)
    return m


def test_dense_mlp_is_the_operator_and_heeds_hooks():
    m, x = _mlp(), _r(2, 5, 32).float()
    want = m.linear_fc2(F_.swiglu(m.linear_fc1(x)))
    assert torch.equal(m(x), want)
    seen = []
    for child in (m.linear_fc1, m.linear_fc2):
        hook = child.register_forward_hook(lambda mod, args, out: seen.append(mod))
        assert torch.equal(m(x), want) and seen[-1] is child
        hook.remove()
    n = len(seen)
    m(x)
    assert len(seen) == n


def test_dense_mlp_leaves_saved_activations_to_the_packer(monkeypatch):
    from cppmega_b200.utils import fp8_activations as fa
    m, x = _mlp(), _r(2, 5, 32).float()
    calls = []
    monkeypatch.setattr(F_, "gated_mlp", lambda *a: calls.append(1) or x)
    with fa.fp8_activation_context():
        assert fa.packing()
        m(x)
        with fa.fp8_quantize_disabled():
            assert not fa.packing()
            m(x)
    assert not fa.packing() and len(calls) == 1
    with fa.fp8_activation_context(enabled=False):
        m(x)
    assert len(calls) == 2


def test_dense_mlp_under_a_recipe_stays_two_linears(monkeypatch):
    m, x = _mlp(), _r(2, 5, 32).float()
    calls = []
    plain = F_.linear
    monkeypatch.setattr(F_, "linear", lambda a, w: (calls.append(F_.precision_recipe()), plain(a, w))[1])
    with F_.precision_scope("mxfp8"):
        m(x)
    assert calls == ["mxfp8", "mxfp8"]


def test_norm_module_with_a_gate():
    from cppmega_b200.models.common import RMSNorm
    m, x, z = RMSNorm(24), _r(3, 24).float(), _r(3, 24, seed=1).float()
    silu = z * torch.sigmoid(z)
    assert torch.allclose(m(x, gate=z), m(x) * silu, rtol=1e-5, atol=1e-6)
    assert torch.allclose(m(x, gate=z, norm_before_gate=False), m(x * silu), rtol=1e-5, atol=1e-6)


def test_calls_go_to_the_device_of_their_tensors(monkeypatch):
    """With another device current, the call runs with the tensors' device current and puts the other one back."""
    from cppmega_b200.ops.cuda import block

    class On:
        is_cuda, device = True, "cuda:1"

        def get_device(self):
            return 1

    class Guard:
        def __init__(self, d):
            seen.append(d)

        def __enter__(self):
            seen.append("in")

        def __exit__(self, *exc):
            seen.append("out")

    seen = []
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch.cuda, "device", Guard)
    assert block._on_device(lambda t, a: seen.append("call") or a)(On(), 5) == 5
    assert seen == ["cuda:1", "in", "call", "out"]
    seen.clear()
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1, raising=False)
    block._on_device(lambda t: seen.append("call"))(On())
    assert seen == ["call"]
