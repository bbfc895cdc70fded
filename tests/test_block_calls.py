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


class _Recorder:
    """Stands in for the kernel library: a backward entry leaves the bytes at each pointer of its arguments that is looked at."""

    def __init__(self, look, sizes):
        self.look, self.sizes, self.seen = look, sizes, None

    def __getattr__(self, name):
        import ctypes

        def call(*args):
            if name == self.look:
                self.seen = {i: ctypes.string_at(args[i], n) for i, n in self.sizes.items()}
            return 64 if name.endswith(("_ws", "_parts", "_kept")) else 0
        return call


def _apart(t):                                   # the same values, every second element of a buffer
    return t.new_empty(*t.shape, 2)[..., 0].copy_(t)


def _wider(t):
    return t.float() if t.dtype == torch.bfloat16 else t


def _offset(t):                                  # packed, but not on 16 bytes
    return t.new_empty(t.numel() + 1)[1:].view(t.shape).copy_(t)


@pytest.mark.parametrize("form", [_apart, _wider, _offset])
@pytest.mark.parametrize("name", ["gated_mlp", "residual_rmsnorm", "rmsnorm_gated"])
def test_backward_reads_saved_tensors_in_any_form(monkeypatch, name, form):
    """A saved-tensor hook may give the values back with other strides, in a wider type or at another address."""
    bf = torch.bfloat16
    r = lambda *s, seed=0: _r(*s, seed=seed, dtype=bf).requires_grad_()  # noqa: E731
    calls = {                                    # call, entry, argument -> saved tensor behind it
        "gated_mlp": (lambda: block.gated_mlp(r(4, 16), r(48, 16), r(16, 24), "silu"), "cm_gated_mlp_bwd", {2: 0, 4: 1, 5: 2, 6: 3, 7: 4}),
        "residual_rmsnorm": (lambda: block.residual_rmsnorm(r(4, 16), r(4, 16, seed=1), r(16), r(16, seed=2), r(16, seed=3), 0.5, 1e-5)[0],
                             "cm_residual_rmsnorm_bwd", {4: 0, 5: 1, 7: 2, 8: 3, 9: 4, 11: 5}),
        "rmsnorm_gated": (lambda: block.rmsnorm_gated(r(4, 16), r(16), r(4, 16, seed=1), 1e-5, 16, True), "cm_rmsnorm_gated_bwd",
                          {0: 0, 4: 1, 2: 2, 7: 3}),
    }
    call, entry, where = calls[name]
    saved = []

    def pack(t):
        saved.append(t.detach().clone())
        return form(t.detach())

    library = _Recorder(entry, {})
    monkeypatch.setattr(block._cu, "lib", lambda: library)
    monkeypatch.setattr(block._cu, "err_word", lambda dev: torch.zeros(1))
    monkeypatch.setattr(block._cu, "stream_ptr", lambda: None)
    block._size.cache_clear()
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        y = call()
    library.sizes = {arg: saved[i].numel() * saved[i].element_size() for arg, i in where.items()}
    y.backward(torch.ones_like(y))
    block._size.cache_clear()
    for arg, i in where.items():
        got, want = torch.frombuffer(bytearray(library.seen[arg]), dtype=saved[i].dtype), saved[i].reshape(-1)
        # no kernel ran: what results hold may be NaN, whose bits a cast changes
        assert torch.equal(got.nan_to_num(), want.nan_to_num()) if got.is_floating_point() else torch.equal(got, want)


def _dense_mlp():
    from cppmega_b200.models.common import DenseMLP
    from cppmega_b200.parallel.state import single_process_context
    return DenseMLP(32, 48, single_process_context(), std=0.1, out_std=0.1, dtype=torch.float32, seed=3)


def test_dense_mlp_calls_a_child_that_is_not_a_stock_linear(monkeypatch):
    """A module in the place of a linear, one with a bias, a forward of its own, a parametrised weight: what it computes counts."""
    class Biased(torch.nn.Module):
        def __init__(self, m):
            super().__init__()
            self.inner, self.weight, self.bias = m, m.weight, torch.ones(m.weight.shape[0])

        def forward(self, x):
            return self.inner(x) + self.bias

    class Nameless(torch.nn.Module):                # no attribute ``weight``
        def __init__(self, m):
            super().__init__()
            self.inner = m

        def forward(self, x):
            return 2 * self.inner(x)

    x = _r(2, 5, 32)
    for name in ("linear_fc1", "linear_fc2"):
        for wrap in (Biased, Nameless):
            m = _dense_mlp()
            setattr(m, name, wrap(getattr(m, name)))
            assert torch.equal(m(x), m.linear_fc2(F_.swiglu(m.linear_fc1(x))))
        m = _dense_mlp()
        child = getattr(m, name)
        monkeypatch.setattr(child, "forward", lambda t, plain=child.forward: 3 * plain(t))
        assert torch.equal(m(x), m.linear_fc2(F_.swiglu(m.linear_fc1(x))))
        m = _dense_mlp()
        want = m.linear_fc2(F_.swiglu(m.linear_fc1(x)))
        torch.nn.utils.parametrize.register_parametrization(getattr(m, name), "weight", torch.nn.Identity())
        assert torch.equal(m(x), want)


def test_dense_mlp_shows_its_linears_to_global_hooks():
    m, x, seen = _dense_mlp(), _r(2, 5, 32), []
    hook = torch.nn.modules.module.register_module_forward_hook(lambda mod, args, out: seen.append(mod))
    try:
        m(x)
    finally:
        hook.remove()
    assert m.linear_fc1 in seen and m.linear_fc2 in seen
    calls = []
    with pytest.MonkeyPatch.context() as patch:     # without hooks it is the operator again
        patch.setattr(F_, "gated_mlp", lambda *a: calls.append(1) or x)
        m(x)
    assert calls == [1]


def _mixers():
    from cppmega_b200.config.model import M2RNNConfig, nam56r_tiny
    from cppmega_b200.models.m2rnn import M2RNNMixer
    from cppmega_b200.models.mamba_variants import VARIANTS, SSDMixer
    from cppmega_b200.parallel.state import single_process_context
    cfg, pc = nam56r_tiny(), single_process_context()
    return {"g_norm": M2RNNMixer(160, M2RNNConfig(), pc, 1),
            "norm": SSDMixer(cfg, pc, 1, VARIANTS["ssd"], dtype=torch.float32, seed=3, out_std=0.1)}


@pytest.mark.parametrize("name", ["g_norm", "norm"])
def test_mixers_call_a_norm_that_is_not_the_stock_one(name):
    """A norm without a gate argument in the place of the mixer's output norm, and hooks on it: called with its input alone."""
    m = _mixers()[name]
    x = _r(1, 64, m.input_projection.weight.shape[1] if name == "g_norm" else m.in_proj.weight.shape[1])
    want, norm, seen = m(x), getattr(m, name), []

    class Plain(torch.nn.Module):
        def forward(self, t):
            seen.append(t)
            return F_.rmsnorm(t, norm.weight, norm.eps)

    setattr(m, name, Plain())
    got = m(x)
    assert len(seen) == 1 and torch.allclose(got, want, rtol=1e-4, atol=1e-5)
    setattr(m, name, norm)
    hook = norm.register_forward_hook(lambda mod, args, out: seen.append(args[0]))
    m(x)
    hook.remove()
    assert torch.allclose(seen[1], seen[0], rtol=1e-4, atol=1e-5)


def test_recomputed_dense_mlp_takes_the_same_operator_in_both_passes(monkeypatch):
    """FP8 storage of saved activations with recomputation: the first pass runs under the context, the replay outside it."""
    from cppmega_b200.utils import fp8_activations as fa
    from cppmega_b200.utils.recompute import checkpoint
    m, x, calls = _dense_mlp(), _r(2, 5, 32).requires_grad_(), []
    plain = F_.gated_mlp
    monkeypatch.setattr(F_, "gated_mlp", lambda *a: calls.append(torch.is_grad_enabled()) or plain(*a))
    with fa.fp8_activation_context():
        y = checkpoint(m, x)
        assert fa.packing()                      # tensors saved here are packed all the same
        with torch.no_grad():
            assert not fa.packing()
    y.sum().backward()
    assert calls == [False, True]


def test_layers_that_stay_bf16_keep_the_fused_dense_mlp(monkeypatch):
    """The first and last layers of a layer-aware storage pack nothing, so that nothing there has to step back for the packer."""
    from cppmega_b200.utils import fp8_activations as fa
    m, x, calls = _dense_mlp(), _r(2, 5, 32), []
    monkeypatch.setattr(F_, "gated_mlp", lambda *a: calls.append(fa.current_layer_idx()) or x)
    try:
        for layer in range(5):
            fa.set_current_layer_idx(layer)
            with fa.fp8_activation_context(n_layers=5, bf16_first=1, bf16_last=2):
                m(x)
                with fa.fp8_activation_context():
                    assert fa.packing()          # the inner context packs every layer
                assert fa.packing() == (layer in (1, 2))
    finally:
        fa.set_current_layer_idx(-1)
    assert calls == [0, 3, 4] and not fa.packing()


@pytest.mark.parametrize("T,H,F,Ho", [(4, 16, 0, 16), (4, 16, 24, 0), (0, 16, 24, 16), (4, 0, 24, 16)])
def test_gated_mlp_of_nothing_is_the_definition(monkeypatch, T, H, F, Ho):
    """A width or a number of tokens of zero never asks for a kernel: the entries return without writing their results."""
    monkeypatch.setattr(F_, "_cuda", lambda name, *t: pytest.fail(f"{name} asked for"))
    leaves = [_r(*s, dtype=torch.bfloat16).requires_grad_() for s in ((T, H), (2 * F, H), (Ho, F))]
    y = F_.gated_mlp(*leaves)
    assert y.shape == (T, Ho) and y.dtype == torch.bfloat16 and (y == 0).all()
    for g, t in zip(torch.autograd.grad(y, leaves, torch.ones_like(y)), leaves):
        assert g.shape == t.shape and (g == 0).all()


def test_residual_rmsnorm_with_a_learnt_scale_is_the_definition():
    """The kernels take the scale as a number: one that wants a gradient would not get it."""
    x, w, scale = _r(4, 16), _r(16), torch.tensor(0.5, requires_grad=True)
    assert block.residual_rmsnorm(x, x, w, None, None, scale, 1e-5) is None
    n, h = F_.residual_rmsnorm(x, x, w, scale=scale)
    assert torch.allclose(torch.autograd.grad(h.sum(), scale)[0], x.sum())


def test_launchers_keep_no_answer_of_one_device_for_all():
    """What a launcher asks the runtime once, it asks per device; a plain static would serve every device and race between threads."""
    import re
    from cppmega_b200.ops.cuda.build import CSRC
    for name in ("residual_norm.cu", "gated_norm.cu", "gated_mlp.cu", "few_rows.cu", "gemm_split.cu", "row_vec.cuh"):
        assert not re.findall(r"\bstatic\s+(?:int|bool|long long|size_t)\s+\w+(?:\[\w+\])?\s*(?:=[^;()]*)?;", (CSRC / name).read_text()), name


def test_function_attributes_are_marked_on_the_device_that_was_set(tmp_path):
    """Two host threads on two devices take turns between asking and marking: neither marks the other's device."""
    import re
    import subprocess
    from cppmega_b200.ops.cuda.build import CSRC
    struct = re.search(r"struct PerDevice \{.*?\n\};", (CSRC / "common.cuh").read_text(), re.S).group(0)
    (tmp_path / "t.cpp").write_text("""#include <atomic>
enum { cudaSuccess = 0 };
static int current = 0;
static int cudaGetDevice(int* d) { *d = current; return cudaSuccess; }
%s
int main() {
  static PerDevice cfg;
  bool a0 = cfg.first();           // thread A, device 0: sets its attribute ...
  current = 1;
  bool b0 = cfg.first();           // ... thread B, device 1, asks meanwhile ...
  current = 0;
  cfg.done();                      // ... and A marks device 0
  bool a1 = cfg.first();
  current = 1;
  bool b1 = cfg.first();           // B has not marked device 1 yet
  cfg.done();
  return a0 && b0 && !a1 && b1 && !cfg.first() ? 0 : 1;
}
""" % struct)
    subprocess.run(["g++", "-std=c++17", "-o", str(tmp_path / "t"), str(tmp_path / "t.cpp")], check=True)
    assert subprocess.run([str(tmp_path / "t")]).returncode == 0


def test_few_row_products_take_what_the_feed_forward_gives_them():
    """The limit of the streamed product is the dispatch's: no range that is accepted but never run."""
    import re
    from cppmega_b200.ops.cuda import lib
    from cppmega_b200.ops.cuda.build import CSRC
    most = int(re.search(r"MAX_ROWS = (\d+);", (CSRC / "few_rows.cuh").read_text()).group(1))
    L, H, F = lib(), 1024, 2048
    ws = [L.cm_gated_mlp_fwd_ws(m, H, F, H) for m in (most - 1, most, most + 1)]
    # up to the limit the work space grows with the tokens: partial tiles, and h's second part of F / 2 floats a token
    assert ws[1] > ws[0] > 0 and ws[2] != ws[1] + (ws[1] - ws[0])


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_norm_entries_refuse_rows_wider_than_the_operators(dtype):
    """The C entries take the widths that the operators do, up to 16384; pointers are never looked at."""
    from cppmega_b200.ops.cuda import lib
    L = lib()
    for W in (16392, 20000, 32768):
        assert L.cm_residual_rmsnorm_fwd(16, W, 16, W, 16, None, None, 0, 16, 16, None, None, 2, W, 1.0, 1e-5, dtype, None) == -10
        assert L.cm_residual_rmsnorm_fwd(16, W, 16, W, 16, 16, 16, 0, 16, 16, None, None, 2, W, 1.0, 1e-5, dtype, None) == -10
        assert L.cm_residual_rmsnorm_bwd(16, W, None, 0, 16, None, 0, 16, None, None, 0, 16, 16, 16, None, None, None, None, None, None, 2, W, 1.0,
                                         dtype, None) == -10
        for gate_first in (0, 1):
            assert L.cm_rmsnorm_gated_fwd(16, W, None, 0, 16, 16, None, 2, W, W, gate_first, 1e-5, dtype, None) == -10
            assert L.cm_rmsnorm_gated_bwd(16, W, None, 0, 16, 16, W, 16, 16, None, None, None, 2, W, W, gate_first, dtype, None) == -10


def _without_kernels(monkeypatch):
    """Forward and backward of the wrappers with a library that computes nothing."""
    library = _Recorder("", {})
    monkeypatch.setattr(block._cu, "lib", lambda: library)
    monkeypatch.setattr(block._cu, "err_word", lambda dev: torch.zeros(1))
    monkeypatch.setattr(block._cu, "stream_ptr", lambda: None)
    monkeypatch.setattr(block, "_size", lambda *a: 64)


@pytest.mark.parametrize("name", ["gated_mlp", "residual_rmsnorm", "rmsnorm_gated"])
def test_second_derivatives_raise_beside_other_terms(monkeypatch, name):
    """A term that needs a second derivative may not go missing from a sum whose other terms have theirs: not with an upstream gradient
    that is a constant, and not where only some leaves are asked for."""
    _without_kernels(monkeypatch)
    call, args = _block_calls()[name]
    leaves = [t.requires_grad_() for t in args]
    for asked in leaves:
        y = call(*leaves)
        y = y[0] if isinstance(y, tuple) else y
        (g,) = torch.autograd.grad(y.sum(), leaves[0], create_graph=True)
        assert g.requires_grad
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum() + asked.sum(), asked)
        with pytest.raises(RuntimeError):
            (g.sum() + asked.sum()).backward()


@pytest.mark.parametrize("name,i", [("gated_mlp", 0), ("residual_rmsnorm", 0), ("rmsnorm_gated", 0), ("rmsnorm_gated", 2)])
def test_second_derivatives_raise_through_an_input_that_was_copied(monkeypatch, name, i):
    """Columns that are not contiguous are copied for the kernels; the copy is still the caller's tensor, here the only one with a gradient."""
    _without_kernels(monkeypatch)
    call, args = _block_calls()[name]
    leaf = args[i].t().contiguous().requires_grad_()
    y = call(*[leaf.t() if j == i else t for j, t in enumerate(args)])
    y = y[0] if isinstance(y, tuple) else y
    (g,) = torch.autograd.grad(y.sum(), leaf, create_graph=True)
    assert g.shape == leaf.shape
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum() + leaf.sum(), leaf)
