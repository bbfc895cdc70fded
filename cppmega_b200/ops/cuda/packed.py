"""Causal attention over packed sequences (``csrc/packed_attention.cu``) with its autograd wrapper."""
from __future__ import annotations

import ctypes

import torch

from .. import cuda as _cu
from .. import functional as F_
from .. import reference as ref
from .block import _Copied, _bare, _failed, _first_order, _given_back, _on_device, _ptr
from .paged import TYPES, Plan, planned, rows_on, strides, width_ok


def declare(L: ctypes.CDLL) -> None:
    vp, i32, i64, f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float
    sig = {
        "cm_packed_attention_fwd": [vp] * 10 + [f32, vp, vp],
        "cm_packed_attention_bwd": [vp] * 14 + [f32, vp, vp],
        "cm_packed_attention_ends": [vp, vp, i64, i64, i64, vp, vp],
    }
    for name, args in sig.items():
        if hasattr(L, name):
            getattr(L, name).argtypes, getattr(L, name).restype = args, i32
    if hasattr(L, "cm_packed_attention_ws"):
        L.cm_packed_attention_ws.argtypes, L.cm_packed_attention_ws.restype = [vp], ctypes.c_longlong


NOTHING = -1               # work of a call without rows of queries, or of keys, or heads


def _strides_ok(t: torch.Tensor) -> bool:
    """Whether a tensor map can read the rows where they are: on 16 bytes, and no step of zero."""
    return rows_on(t, 16) and all(n == 1 or 0 < s < 2 ** 38 for n, s in zip(t.shape[:-1], t.stride()[:-1]))


def _in_place(t: torch.Tensor) -> bool:
    return t.data_ptr() % 16 == 0 and _strides_ok(t)


def _readable(t: torch.Tensor) -> torch.Tensor:
    """The tensor, or a packed copy that stays tied to it."""
    return t if _in_place(t) else _Copied.apply(t)


def _packed(t: torch.Tensor) -> torch.Tensor:
    return t if _in_place(t) else t.clone(memory_format=torch.contiguous_format)


def _numbers(q, k, v, cu_q, go=None):
    T, H, D = q.shape
    return [*strides(q), *strides(k), *strides(v), *strides(go, 2), cu_q.numel() - 1, T, k.shape[0], H, k.shape[1], D, v.shape[2], TYPES[q.dtype]]


def _plan(q, k, v, cu_q, cu_k):
    if not (q.dtype in TYPES and width_ok(q, 8, 128) and width_ok(v, 8, 128) and q.shape[0] < 2 ** 30 and k.shape[0] < 2 ** 30):
        return False
    if not (q.shape[0] and k.shape[0] and q.shape[1]):
        return Plan([], shape=(q.shape[0], q.shape[1], v.shape[2]), work=NOTHING)
    plan = Plan(_numbers(q, k, v, cu_q), shape=(q.shape[0], q.shape[1], v.shape[2]), like=q.is_contiguous() and q.shape[2] == v.shape[2],
                copy=not (_strides_ok(q) and _strides_ok(k) and _strides_ok(v) and cu_q.is_contiguous() and (cu_k is None or cu_k.is_contiguous())))
    plan.work = _cu.lib().cm_packed_attention_ws(plan.at)
    return plan


def _plan_backward(dt, q, k, v, cu_q, cu_k, o, rest, lse, go):
    """False where a tensor is not in the form in which the forward left it, or an upstream gradient has to be copied."""
    if not (all(t.dtype == dt and t.device == go.device for t in (q, k, v, o, rest, go)) and all(_strides_ok(t) for t in (q, k, v, go))
            and all(t.is_contiguous() and t.device == go.device for t in (cu_q, cu_k, o, rest, lse))
            and cu_q.dtype == cu_k.dtype == torch.int32 and lse.dtype == torch.float32):
        return False
    return Plan(_numbers(q, k, v, cu_q, go), work=lse.numel() if dt == torch.bfloat16 else 2 * (lse.numel() + (cu_q.numel() - 1) * k.shape[1]))


def _forward(plan, q, k, v, cu_q, cu_k, scale, keep):
    dev = q.device
    o = torch.empty_like(q) if plan.like else torch.empty(plan.shape, dtype=q.dtype, device=dev)
    rest = torch.empty_like(o) if keep else None
    lse = torch.empty(plan.shape[:2], dtype=torch.float32, device=dev) if keep else None
    ws = torch.empty(plan.work, dtype=torch.float32, device=dev) if plan.work else None
    rc = _cu.lib().cm_packed_attention_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(), o.data_ptr(), _ptr(rest),
                                           _ptr(lse), _ptr(ws), plan.at, scale, _cu.err_word(dev).data_ptr(), _cu.stream_ptr())
    if rc:
        _failed("cm_packed_attention_fwd", rc)
    F_.count_launch("packed_attention")
    return o, rest, lse


class PackedAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, scale, plan):
        o, rest, lse = _forward(plan, q, k, v, cu_q, cu_k, scale, keep=True)
        ctx.save_for_backward(q, k, v, cu_q, cu_k, o, rest, lse)
        ctx.scale, ctx.dtype = scale, q.dtype
        return o

    @staticmethod
    @_first_order
    def backward(ctx, go):
        saved = ctx.saved_tensors
        if not _bare(go):
            return _by_definition(ctx, *saved[:5], go)
        layout = F_.layout_of("packed_attention_bwd", *saved, go)
        plan = planned(layout, lambda: _plan_backward(ctx.dtype, *saved, go))
        q, k, v, cu_q, cu_k, o, rest, lse = saved
        if not plan or (q.data_ptr() | k.data_ptr() | v.data_ptr() | o.data_ptr() | rest.data_ptr() | go.data_ptr()) & 15:
            dt, dev = ctx.dtype, go.device     # whatever form a saved-tensor hook gave the values back in
            q, k, v = (_packed(_given_back(t, dt, dev, packed=False)) for t in (q, k, v))
            o, rest = (_given_back(t, dt, dev, align=16) for t in (o, rest))
            cu_q, cu_k = (_given_back(t, torch.int32, dev) for t in (cu_q, cu_k))
            lse, go = _given_back(lse, torch.float32, dev), _packed(go)
            plan = _plan_backward(dt, q, k, v, cu_q, cu_k, o, rest, lse, go)
        dev = go.device
        need_q, need_k, need_v = ctx.needs_input_grad[:3]           # dk and dv come from one kernel
        dq, dk, dv = (torch.empty_like(t, memory_format=torch.contiguous_format) if need else None
                      for t, need in ((q, need_q), (k, need_k or need_v), (v, need_k or need_v)))
        delta = torch.empty(plan.work, dtype=torch.float32, device=dev)
        rc = _cu.lib().cm_packed_attention_bwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), rest.data_ptr(), go.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(),
            lse.data_ptr(), delta.data_ptr(), _ptr(dq), _ptr(dk), _ptr(dv), plan.at, ctx.scale,
            _cu.err_word(dev).data_ptr(), _cu.stream_ptr())
        if rc:
            _failed("cm_packed_attention_bwd", rc)
        F_.count_launch("packed_attention_bwd", (1 if ctx.dtype == torch.bfloat16 else 2) + need_q + (need_k or need_v))
        return dq, dk if need_k else None, dv if need_v else None, None, None, None, None


def _nothing(plan, q, k, v, cu_q, cu_k):
    """Zeros that depend on the inputs, whose gradients are zeros too; the ends are checked on the device as those of any call."""
    rc = _cu.lib().cm_packed_attention_ends(cu_q.data_ptr(), cu_k.data_ptr(), cu_q.numel() - 1, q.shape[0], k.shape[0],
                                            _cu.err_word(q.device).data_ptr(), _cu.stream_ptr())
    if rc:
        _failed("cm_packed_attention_ends", rc)
    F_.count_launch("packed_attention")
    return q.new_zeros(plan.shape) + sum(t[:0].sum() for t in (q, k, v))


def _by_definition(ctx, q, k, v, cu_q, cu_k, go):
    """Gradients for a ``go`` without memory of its own (a batch of them, under ``is_grads_batched``)."""
    F_._miss("packed_attention_bwd(batched gradients)", q)
    q, k, v = (_given_back(t, ctx.dtype, go.device, packed=False) for t in (q, k, v))
    cu_q, cu_k = (_given_back(t, torch.int32, go.device, packed=False) for t in (cu_q, cu_k))
    with torch.enable_grad():
        leaves = [t.detach().requires_grad_(need) for t, need in zip((q, k, v), ctx.needs_input_grad)]
        o = ref.packed_attention(*leaves, cu_q, ctx.scale, cu_k)
    grads = iter(torch.autograd.grad(o, [t for t in leaves if t.requires_grad], go))
    return (*(next(grads) if t.requires_grad else None for t in leaves), None, None, None, None)


@_on_device
def packed_attention(q, k, v, cu_q, scale, cu_k, layout):
    """None where the kernels do not apply."""
    plan = planned(layout, lambda: _plan(q, k, v, cu_q, cu_k))
    if not plan or isinstance(scale, torch.Tensor) or not abs(scale) < 2.0 ** 64 or not _bare(q, k, v, cu_q, cu_k):
        return None
    if plan.work == NOTHING:
        return _nothing(plan, q, k, v, cu_q.contiguous(), cu_q.contiguous() if cu_k is None else cu_k.contiguous())
    if scale < 0 or plan.copy or (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15:
        if scale < 0:      # the kernels take the largest product of a row for its reference: the sign goes into q, exactly
            q, scale = -q, -scale
        q, k, v, cu_q = _readable(q), _readable(k), _readable(v), cu_q.contiguous()
        cu_k = None if cu_k is None else cu_k.contiguous()
        return packed_attention(q, k, v, cu_q, scale, cu_k, F_.layout_of("packed_attention", q, k, v, cu_q, cu_k))
    if cu_k is None:
        cu_k = cu_q
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return PackedAttentionFn.apply(q, k, v, cu_q, cu_k, float(scale), plan)
    return _forward(plan, q, k, v, cu_q, cu_k, float(scale), keep=False)[0]


def register() -> None:
    F_.register_cuda("packed_attention", packed_attention)
