"""The operators around a dense block: gated feed-forward (``csrc/gated_mlp.cu``), residual step with its norms
(``csrc/residual_norm.cu``) and gated norm of a mixer's output (``csrc/gated_norm.cu``), with their autograd wrappers.

The wrappers take their tensors as they come: leading dimensions of any number, rows of any pitch (column slices of a wider
projection are read in place), widths that no vector divides.  Work space is allocated per call on the current stream.
A kernel reads memory and gives first derivatives: what needs more than that is left to the definitions, or raises.
"""
from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd import forward_ad

from .. import cuda as _cu
from .. import functional as F_
from .. import reference as ref

ACTIVATIONS = {"silu": 0, "gelu_tanh": 1, "relu": 2}
ROW_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_WIDTH = 16384          # widest normalised row


def declare(L: ctypes.CDLL) -> None:
    vp, i32, i64, f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float
    sig = {
        "cm_gated_mlp_fwd": [vp, i64, vp, vp, vp, vp, vp, vp, i32, i32, i32, i32, i32, vp, vp],
        "cm_gated_mlp_bwd": [vp, i64, vp, i64, vp, vp, vp, vp, vp, vp, vp, i32, i32, vp, i32, i32, vp, i32, i32, i32, i32, i32, vp, vp],
        "cm_gemm_split": [vp, vp, vp, i32, i32, i32, i64, i64, i64, i32, i32, i32, i32, vp, vp, vp],
        "cm_residual_rmsnorm_fwd": [vp, i64, vp, i64, vp, vp, vp, i32, vp, vp, vp, vp, i64, i32, f32, f32, i32, vp],
        "cm_residual_rmsnorm_parts": [i64, i32],
        "cm_rmsnorm_gated_parts": [i64, i32, i32],
        "cm_residual_rmsnorm_bwd": [vp, i64, vp, i64, vp, vp, i64, vp, vp, vp, i32, vp, vp, vp, vp, vp, vp, vp, vp, vp, i64, i32, f32,
                                    i32, vp],
        "cm_rmsnorm_gated_fwd": [vp, i64, vp, i64, vp, vp, vp, i64, i32, i32, i32, f32, i32, vp],
        "cm_rmsnorm_gated_bwd": [vp, i64, vp, i64, vp, vp, i64, vp, vp, vp, vp, vp, i64, i32, i32, i32, i32, vp],
    }
    for name, args in sig.items():
        fn = getattr(L, name, None)
        if fn is not None:
            fn.argtypes = args
            fn.restype = i32
    for name, args in (("cm_gated_mlp_fwd_ws", [i32] * 4), ("cm_gated_mlp_bwd_ws", [i32] * 4), ("cm_gemm_split_plan", [i32] * 5 + [vp]),
                       ("cm_gated_mlp_kept", [i32] * 2)):
        if hasattr(L, name):
            getattr(L, name).argtypes, getattr(L, name).restype = args, i64


def _failed(name: str, rc: int) -> None:
    raise _cu.KernelError(f"{name} failed with code {rc}")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _on_device(fn):
    """Launches go to the device of the tensors (the first argument's), whichever is current."""
    @functools.wraps(fn)
    def call(t, *args):
        if not t.is_cuda or t.get_device() == torch._C._cuda_getDevice():
            return fn(t, *args)
        with torch.cuda.device(t.device):
            return fn(t, *args)
    return call


class _Undifferentiable(torch.autograd.Function):
    """Passes its first ``n`` tensors on as results that depend on all of its tensors and refuse to be differentiated."""

    @staticmethod
    def forward(ctx, n, *tensors):
        return tuple(t.view_as(t) for t in tensors[:n])

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("the kernels around a dense block have first derivatives only; ops.reference has the definitions, which can be "
                           "differentiated again")


def _first_order(fn):
    """``backward`` without a graph of its own.  Under ``create_graph`` its results are tied to everything that they were computed from, so
    that a second derivative raises on every way to it instead of missing a term."""
    def backward(ctx, *grads):
        if not torch.is_grad_enabled():
            return fn(ctx, *grads)
        with torch.no_grad():
            outs = fn(ctx, *grads)
        own = [t for t in outs if t is not None]
        roots = [t for t in (*ctx.saved_tensors, *grads) if t is not None and t.requires_grad]
        tied = iter(_Undifferentiable.apply(len(own), *own, *roots))
        return tuple(None if t is None else next(tied) for t in outs)
    return backward


def _bare(*tensors) -> bool:
    """Whether the tensors are no more than the memory that a kernel reads: one inside a function transform (``vmap``, ``torch.func``)
    has no storage, and the tangent of a forward-mode dual lies beside it."""
    for t in tensors:
        if t is not None and (not torch._C._has_storage(t)
                              or forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None):
            return False
    return True


@functools.lru_cache(maxsize=1024)
def _size(name: str, device: int, *args) -> int:
    """The library's answer to a question about sizes on the current device."""
    return getattr(_cu.lib(), name)(*args)


def _pitch(t: torch.Tensor):
    """Elements between rows of the [rows, width] view of a tensor whose rows are contiguous and evenly spaced; None for any other."""
    if t.is_contiguous():
        return t.shape[-1]
    if t.stride(-1) == 1 or t.shape[-1] == 1:
        pitch = expect = None
        for n, s in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if n == 1:
                continue
            if pitch is None:
                pitch = expect = s
            if s != expect:
                return None
            expect = s * n
        if pitch is None:
            return t.shape[-1]
        if pitch >= t.shape[-1]:
            return pitch
    return None


def _rows(t: torch.Tensor):
    """``(tensor, elements between rows)`` of the [rows, width] view; a tensor without one is copied."""
    pitch = _pitch(t)
    return (t, pitch) if pitch is not None else (_cu.fast_contiguous(t), t.shape[-1])


class _Copied(torch.autograd.Function):
    """A packed copy that stays tied to its original."""

    @staticmethod
    def forward(ctx, t):
        return _cu.fast_copy_(torch.empty(t.shape, dtype=t.dtype, device=t.device), t)

    @staticmethod
    def backward(ctx, g):
        return g


def _readable(t, tma: bool = False):
    """The tensor, or a copy where the kernels cannot read it in place: made before the operator's own function, which saves what it is
    given, so that a second derivative finds its way from there to the original."""
    if t is None:
        return t
    pitch = _pitch(t)
    return t if pitch is not None and not (tma and (pitch % 8 or t.data_ptr() % 16)) else _Copied.apply(t)


def _given_back(t, dtype: torch.dtype, device: torch.device, packed: bool = True, align: int = 1):
    """A saved tensor in the form in which the kernels read it, whatever form a saved-tensor hook gave its values back in."""
    if t is None or (t.dtype == dtype and t.device == device and (not packed or t.is_contiguous() and t.data_ptr() % align == 0)):
        return t
    return torch.empty(t.shape, dtype=dtype, device=device).copy_(t)


def _like(t: torch.Tensor) -> torch.Tensor:
    """A packed tensor of the same shape, type and device."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty_like(t, memory_format=torch.contiguous_format)


# ---------------------------------------------------------------------------
# gated feed-forward block
# ---------------------------------------------------------------------------

def _tma_rows(t: torch.Tensor):
    """As :func:`_rows`, for a bf16 operand that is read through a tensor map: 16-byte rows and base."""
    t, pitch = _rows(t)
    if pitch % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        pitch = t.shape[-1]
    return t, pitch


def _mlp_forward(x, w1, w2, act, keep):
    L = _cu.lib()
    x, ldx = _tma_rows(x)
    H, F, Ho = w1.shape[1], w2.shape[1], w2.shape[0]
    M = x.numel() // H
    y = _like(x) if Ho == H else x.new_empty(*x.shape[:-1], Ho)
    h = x.new_empty(M, F)
    kept = torch.empty(_size("cm_gated_mlp_kept", x.get_device(), M, F), dtype=torch.uint8, device=x.device) if keep else None
    floats = _size("cm_gated_mlp_fwd_ws", x.get_device(), M, H, F, Ho)
    ws = torch.empty(floats, dtype=torch.float32, device=x.device) if floats else None
    rc = L.cm_gated_mlp_fwd(x.data_ptr(), ldx, w1.data_ptr(), w2.data_ptr(), _ptr(kept), h.data_ptr(), y.data_ptr(), _ptr(ws), M, H, F, Ho,
                            act, _cu.err_word(x.device).data_ptr(), _cu.stream_ptr())
    if rc:
        _failed("cm_gated_mlp_fwd", rc)
    F_.count_launch("gated_mlp")
    return y, x, kept, h


class GatedMLPFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, w2, act):
        y, x, kept, h = _mlp_forward(x, w1, w2, act, keep=True)
        ctx.save_for_backward(x, w1, w2, kept, h)
        ctx.act = act
        return y

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        x, p1, p2, kept, h = ctx.saved_tensors
        need_x, need_w1, need_w2, _ = ctx.needs_input_grad
        w1, w2, h = (_given_back(t, torch.bfloat16, dy.device, align=16) for t in (p1, p2, h))
        kept = _given_back(kept, torch.uint8, dy.device, align=16)
        x = _given_back(x, torch.bfloat16, dy.device, packed=False)
        H, F, Ho = w1.shape[1], w2.shape[1], w2.shape[0]
        dy, lddy = _tma_rows(dy)
        x, ldx = _tma_rows(x)
        dx = _like(x) if need_x else None
        into = [(None, 0, 0), (None, 0, 0)]                        # (result, fp32, added to what is there) of each weight

        def target(i, w):
            def run(out, acc):
                t = torch.empty_like(w) if out is None else out
                into[i] = (t.data_ptr(), int(t.dtype == torch.float32), int(acc))
                return t
            return run

        dw1 = _cu.wgrad_into_main_grad(p1, target(0, w1)) if need_w1 else None
        dw2 = _cu.wgrad_into_main_grad(p2, target(1, w2)) if need_w2 else None
        dgu = x.new_empty(h.shape[0], 2 * F) if need_x or need_w1 else None
        L, M = _cu.lib(), h.shape[0]
        floats = _size("cm_gated_mlp_bwd_ws", x.get_device(), M, H, F, Ho)
        ws = torch.empty(floats, dtype=torch.float32, device=x.device) if floats else None
        rc = L.cm_gated_mlp_bwd(dy.data_ptr(), lddy, x.data_ptr(), ldx, w1.data_ptr(), w2.data_ptr(), kept.data_ptr(), h.data_ptr(),
                                _ptr(dgu), _ptr(dx), *into[0], *into[1], _ptr(ws), M, H, F, Ho, ctx.act,
                                _cu.err_word(x.device).data_ptr(), _cu.stream_ptr())
        if rc:
            _failed("cm_gated_mlp_bwd", rc)
        F_.count_launch("gated_mlp_bwd")
        return dx, dw1, dw2, None


@_on_device
def gated_mlp(x, w1, w2, activation):
    """None where the kernels do not apply: they take bf16 throughout and widths that are multiples of 8."""
    if not (_bare(x, w1, w2) and x.dtype == w1.dtype == w2.dtype == torch.bfloat16 and w1.is_contiguous() and w2.is_contiguous() and x.numel() > 0
            and x.shape[-1] % 8 == 0 and w2.shape[0] % 8 == 0 and w2.shape[1] % 8 == 0 and w1.data_ptr() % 16 == 0
            and w2.data_ptr() % 16 == 0 and x.numel() // x.shape[-1] < 2 ** 30):
        return None
    if torch.is_grad_enabled() and (x.requires_grad or w1.requires_grad or w2.requires_grad):
        return GatedMLPFn.apply(_readable(x, tma=True), w1, w2, ACTIVATIONS[activation])
    return _mlp_forward(x, w1, w2, ACTIVATIONS[activation], keep=False)[0]


# ---------------------------------------------------------------------------
# residual step with its norms
# ---------------------------------------------------------------------------

def _residual_forward(y, residual, weight, post, gate, scale, eps, keep):
    y, sy = _rows(y)
    residual, sres = _rows(residual)
    W = y.shape[-1]
    R = y.numel() // W
    n, h = _like(y), _like(y)
    stats = torch.empty(2 * R, dtype=torch.float32, device=y.device) if keep else None         # 1 / rms of y, then of h
    at = stats.data_ptr() if keep else None
    rc = _cu.lib().cm_residual_rmsnorm_fwd(y.data_ptr(), sy, residual.data_ptr(), sres, weight.data_ptr(), _ptr(post), _ptr(gate),
                                           int(gate is not None and gate.dim() > 1), n.data_ptr(), h.data_ptr(), at,
                                           at + 4 * R if keep else None, R, W, scale, eps, ROW_TYPES[y.dtype], _cu.stream_ptr())
    if rc:
        _failed("cm_residual_rmsnorm_fwd", rc)
    F_.count_launch("residual_rmsnorm")
    return n, h, y, stats


class ResidualRMSNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, residual, weight, post, gate, scale, eps):
        n, h, y, stats = _residual_forward(y, residual, weight, post, gate, scale, eps, keep=True)
        # the block's output is read again only where a norm or a gate stands between it and the stream
        ctx.save_for_backward(h, y if post is not None or gate is not None else None, weight, post, gate, stats)
        ctx.scale, ctx.dtype = scale, y.dtype
        ctx.set_materialize_grads(False)
        return n, h

    @staticmethod
    @_first_order
    def backward(ctx, dn, dh):
        if dn is None and dh is None:
            return (None,) * 7
        h, y, weight, post, gate, stats = ctx.saved_tensors
        need_y, _, need_w, need_post, need_gate = ctx.needs_input_grad[:5]
        dt, dev = ctx.dtype, (dh if dn is None else dn).device
        h, weight, post, gate = (_given_back(t, dt, dev) for t in (h, weight, post, gate))
        stats = _given_back(stats, torch.float32, dev)
        y = _given_back(y, dt, dev, packed=False)
        W = h.shape[-1]
        R = h.numel() // W
        sy = sdn = sdh = 0
        if y is not None:
            y, sy = _rows(y)
        if dn is not None:
            dn, sdn = _rows(dn)
        if dh is not None:
            dh, sdh = _rows(dh)
        per_row = gate is not None and gate.dim() > 1
        same = y is None and ctx.scale == 1.0
        dres = torch.empty_like(h)
        dy = torch.empty_like(h) if need_y and not same else None
        dgate = torch.empty_like(gate) if need_gate else None
        dw = torch.empty_like(weight) if need_w else None
        dpost = torch.empty_like(post) if need_post else None
        sums = need_w + need_post + (need_gate and not per_row)
        L = _cu.lib()
        part = torch.empty(sums * _size("cm_residual_rmsnorm_parts", h.get_device(), R, W) * W, dtype=torch.float32, device=h.device) if sums else None
        at = stats.data_ptr()
        rc = L.cm_residual_rmsnorm_bwd(_ptr(dn), sdn, _ptr(dh), sdh, h.data_ptr(), _ptr(y), sy, weight.data_ptr(), _ptr(post), _ptr(gate),
                                       int(per_row), at, at + 4 * R, dres.data_ptr(), _ptr(dy), _ptr(dgate) if per_row else None, _ptr(dw),
                                       _ptr(dpost), None if per_row else _ptr(dgate), _ptr(part), R, W, ctx.scale, ROW_TYPES[h.dtype],
                                       _cu.stream_ptr())
        if rc:
            _failed("cm_residual_rmsnorm_bwd", rc)
        F_.count_launch("residual_rmsnorm_bwd")
        return (dres if same else dy), dres, dw, dpost, dgate, None, None


@_on_device
def residual_rmsnorm(y, residual, weight, post_weight, gate, scale, eps):
    """None where the kernels do not apply: one type for all tensors (bf16, fp16 or fp32), rows of at most 16384, a scale that is a
    number (a tensor may want a gradient)."""
    dt = y.dtype
    if (dt not in ROW_TYPES or residual.dtype != dt or weight.dtype != dt or (post_weight is not None and post_weight.dtype != dt)
            or (gate is not None and gate.dtype != dt) or y.shape[-1] > MAX_WIDTH or y.numel() == 0
            or isinstance(scale, torch.Tensor) or not _bare(y, residual, weight, post_weight, gate)):
        return None
    weight = weight.contiguous()
    if post_weight is not None:
        post_weight = post_weight.contiguous()
    if gate is not None:
        gate = gate.contiguous()
    if torch.is_grad_enabled() and (y.requires_grad or residual.requires_grad or weight.requires_grad
                                    or (post_weight is not None and post_weight.requires_grad) or (gate is not None and gate.requires_grad)):
        return ResidualRMSNormFn.apply(_readable(y), residual, weight, post_weight, gate, float(scale), float(eps))
    return _residual_forward(y, residual, weight, post_weight, gate, float(scale), float(eps), keep=False)[:2]


# ---------------------------------------------------------------------------
# gated norm
# ---------------------------------------------------------------------------

def _gated_forward(x, weight, z, eps, group, gate_first, keep):
    x, sx = _rows(x)
    sz = 0
    if z is not None:
        z, sz = _rows(z)
    W = x.shape[-1]
    R = x.numel() // W
    y = _like(x)
    rstd = torch.empty(R * (W // group), dtype=torch.float32, device=x.device) if keep else None
    rc = _cu.lib().cm_rmsnorm_gated_fwd(x.data_ptr(), sx, _ptr(z), sz, weight.data_ptr(), y.data_ptr(), _ptr(rstd), R, W, group,
                                        int(gate_first), eps, ROW_TYPES[x.dtype], _cu.stream_ptr())
    if rc:
        _failed("cm_rmsnorm_gated_fwd", rc)
    F_.count_launch("rmsnorm_gated")
    return y, x, z, rstd


class GatedRMSNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, z, eps, group, gate_first):
        y, x, z, rstd = _gated_forward(x, weight, z, eps, group, gate_first, keep=True)
        ctx.save_for_backward(x, weight, z, rstd)
        ctx.eps, ctx.group, ctx.gate_first = eps, group, gate_first
        return y

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        x, weight, z, rstd = ctx.saved_tensors
        if not _bare(dy):
            return _gated_by_definition(ctx, x, weight, z, dy)
        _, need_w, need_z = ctx.needs_input_grad[:3]
        weight, rstd = _given_back(weight, dy.dtype, dy.device), _given_back(rstd, torch.float32, dy.device)
        x, z = (_given_back(t, dy.dtype, dy.device, packed=False) for t in (x, z))
        W = x.shape[-1]
        R = x.numel() // W
        x, sx = _rows(x)
        dy, sdy = _rows(dy)
        sz = 0
        if z is not None:
            z, sz = _rows(z)
        dx = _like(x)
        dz = torch.empty_like(dx) if need_z else None
        dw = part = None
        L = _cu.lib()
        if need_w:
            dw = torch.empty_like(weight)
            part = torch.empty(_size("cm_rmsnorm_gated_parts", x.get_device(), R, W, ctx.group) * W, dtype=torch.float32, device=x.device)
        rc = L.cm_rmsnorm_gated_bwd(x.data_ptr(), sx, _ptr(z), sz, weight.data_ptr(), dy.data_ptr(), sdy, rstd.data_ptr(), dx.data_ptr(),
                                    _ptr(dz), _ptr(dw), _ptr(part), R, W, ctx.group, int(ctx.gate_first), ROW_TYPES[x.dtype],
                                    _cu.stream_ptr())
        if rc:
            _failed("cm_rmsnorm_gated_bwd", rc)
        F_.count_launch("rmsnorm_gated_bwd")
        return dx, dw, dz, None, None, None


def _gated_by_definition(ctx, x, weight, z, dy):
    """Gradients for a ``dy`` without memory of its own (a batch of them, under ``is_grads_batched``)."""
    F_._miss("rmsnorm_gated_bwd(batched gradients)", x)
    with torch.enable_grad():
        leaves = [None if t is None else t.detach().requires_grad_(need) for t, need in zip((x, weight, z), ctx.needs_input_grad)]
        y = ref.rmsnorm_gated(*leaves, ctx.eps, ctx.group, not ctx.gate_first)
    wanted = [t for t in leaves if t is not None and t.requires_grad]
    grads = iter(torch.autograd.grad(y, wanted, dy))
    return (*(next(grads) if t is not None and t.requires_grad else None for t in leaves), None, None, None)


@_on_device
def rmsnorm_gated(x, weight, z, eps, group, norm_before_gate):
    """None where the kernels do not apply: one type for all tensors (bf16, fp16 or fp32), groups of at most 16384 channels and at
    most 65535 of them."""
    dt = x.dtype
    if (dt not in ROW_TYPES or weight.dtype != dt or (z is not None and z.dtype != dt) or group > MAX_WIDTH or x.numel() == 0
            or x.shape[-1] // group > 65535 or not _bare(x, weight, z)):
        return None
    weight = weight.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (z is not None and z.requires_grad)):
        return GatedRMSNormFn.apply(_readable(x), weight, _readable(z), float(eps), group, not norm_before_gate)
    return _gated_forward(x, weight, z, float(eps), group, not norm_before_gate, keep=False)[0]


def register() -> None:
    F_.register_cuda("gated_mlp", gated_mlp)
    F_.register_cuda("residual_rmsnorm", residual_rmsnorm)
    F_.register_cuda("rmsnorm_gated", rmsnorm_gated)
