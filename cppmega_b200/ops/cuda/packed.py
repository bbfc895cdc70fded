"""Causal attention over packed sequences (``csrc/packed_attention.cu``) with its autograd wrapper."""
from __future__ import annotations

import ctypes

import torch

from .. import cuda as _cu
from .. import functional as F_
from .block import _Copied, _bare, _failed, _first_order, _given_back, _on_device, _ptr
from .paged import TYPES, _rows_on, _strides, _width_ok


def declare(L: ctypes.CDLL) -> None:
    vp, i32, f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_float
    sig = {
        "cm_packed_attention_fwd": [vp] * 10 + [i32] * 7 + [f32, i32, vp, vp],
        "cm_packed_attention_bwd": [vp] * 17 + [i32] * 7 + [f32, i32, vp, vp],
    }
    for name, args in sig.items():
        if hasattr(L, name):
            getattr(L, name).argtypes, getattr(L, name).restype = args, i32


def _in_place(t: torch.Tensor) -> bool:
    """Whether a tensor map can read the rows where they are: on 16 bytes, and no step of zero."""
    return _rows_on(t, 16) and all(n == 1 or 0 < s < 2 ** 38 for n, s in zip(t.shape[:-1], t.stride()[:-1]))


def _readable(t: torch.Tensor) -> torch.Tensor:
    """The tensor, or a packed copy that stays tied to it."""
    return t if _in_place(t) else _Copied.apply(t)


def _packed(t: torch.Tensor) -> torch.Tensor:
    return t if _in_place(t) else t.clone(memory_format=torch.contiguous_format)


def _forward(q, k, v, cu_q, cu_k, scale, keep):
    T, H, D = q.shape
    o = torch.empty(T, H, v.shape[2], dtype=q.dtype, device=q.device)
    lse = torch.empty(T, H, dtype=torch.float32, device=q.device) if keep else None
    rc = _cu.lib().cm_packed_attention_fwd(
        q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), v.data_ptr(), _strides(v), cu_q.data_ptr(), cu_k.data_ptr(), o.data_ptr(), _ptr(lse),
        cu_q.numel() - 1, T, k.shape[0], H, k.shape[1], D, v.shape[2], scale, TYPES[q.dtype], _cu.err_word(q.device).data_ptr(), _cu.stream_ptr())
    if rc:
        _failed("cm_packed_attention_fwd", rc)
    F_.count_launch("packed_attention")
    return o, lse


class PackedAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, scale):
        o, lse = _forward(q, k, v, cu_q, cu_k, scale, keep=True)
        ctx.save_for_backward(q, k, v, cu_q, cu_k, o, lse)
        ctx.scale, ctx.dtype = scale, q.dtype
        return o

    @staticmethod
    @_first_order
    def backward(ctx, go):
        dt, dev = ctx.dtype, go.device
        q, k, v, cu_q, cu_k, o, lse = ctx.saved_tensors
        q, k, v, o = (_packed(_given_back(t, dt, dev, packed=False)) for t in (q, k, v, o))
        cu_q, cu_k = (_given_back(t, torch.int32, dev) for t in (cu_q, cu_k))
        lse = _given_back(lse, torch.float32, dev)
        go = _packed(go)
        T, H, D = q.shape
        Tk, G, V = v.shape
        dq = torch.empty(T, H, D, dtype=dt, device=dev)
        dk, dv = torch.empty(Tk, G, D, dtype=dt, device=dev), torch.empty(Tk, G, V, dtype=dt, device=dev)
        delta = torch.empty(T * H + 1, dtype=torch.float32, device=dev)
        rc = _cu.lib().cm_packed_attention_bwd(
            q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), v.data_ptr(), _strides(v), o.data_ptr(), _strides(o), go.data_ptr(), _strides(go),
            cu_q.data_ptr(), cu_k.data_ptr(), lse.data_ptr(), delta.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), cu_q.numel() - 1, T, Tk,
            H, G, D, V, ctx.scale, TYPES[dt], _cu.err_word(dev).data_ptr(), _cu.stream_ptr())
        if rc:
            _failed("cm_packed_attention_bwd", rc)
        F_.count_launch("packed_attention_bwd", 2)
        return dq, dk, dv, None, None, None


@_on_device
def packed_attention(q, k, v, cu_q, scale, cu_k):
    """None where the kernels do not apply."""
    if not (q.dtype in TYPES and not isinstance(scale, torch.Tensor) and _bare(q, k, v, cu_q, cu_k) and _width_ok(q, 8, 128) and _width_ok(v, 8, 128)
            and 0 < q.shape[0] < 2 ** 30 and 0 < k.shape[0] < 2 ** 30 and q.shape[1] > 0 and abs(scale) < 2.0 ** 64):
        return None
    cu_q = cu_q.contiguous()
    cu_k = cu_q if cu_k is None else cu_k.contiguous()
    if scale < 0:          # the kernels take the largest product of a row for its reference: the sign goes into q, exactly
        q, scale = -q, -scale
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return PackedAttentionFn.apply(_readable(q), _readable(k), _readable(v), cu_q, cu_k, float(scale))
    return _forward(_packed(q), _packed(k), _packed(v), cu_q, cu_k, float(scale), keep=False)[0]


def register() -> None:
    F_.register_cuda("packed_attention", packed_attention)
