"""The paged key-value cache (``csrc/paged_cache.cu``) and the attention of one new token per sequence over it (``csrc/paged_attention.cu``).

Tensors are read where they are: strides of a cache are free as long as a row (the last axis) is contiguous and lies on 16 bytes.
Work space is allocated per call on the current stream, and nothing waits for the device.

A call's sizes and strides, as the library takes them, are worked out once per layout (shapes, strides, types, devices) and kept: a step of
generation makes the same call again and again, and on the host its checks would cost more than its kernels do on the device.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.graph import increment_version

from .. import cuda as _cu
from .. import functional as F_
from .block import _bare, _failed, _on_device, _ptr

TYPES = {torch.bfloat16: 0, torch.float16: 1}
E4M3 = torch.float8_e4m3fn


def declare(L: ctypes.CDLL) -> None:
    vp, i32, i64, f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float
    sig = {
        "cm_cache_write": [vp] * 10,
        "cm_cache_read": [vp] * 11,
        "cm_paged_attention": [vp] * 10 + [f32, vp, vp],
    }
    for name, args in sig.items():
        if hasattr(L, name):
            getattr(L, name).argtypes, getattr(L, name).restype = args, i32
    if hasattr(L, "cm_paged_attention_ws"):
        L.cm_paged_attention_ws.argtypes, L.cm_paged_attention_ws.restype = [i32] * 8, i64


class Plan:
    """What a layout's calls have in common: the library's array of sizes and strides, and what else the wrapper needs."""

    __slots__ = ("numbers", "at", "copy", "shape", "work", "like", "spans", "apart")

    def __init__(self, numbers, copy=False, shape=None, work=0, like=False, spans=None):
        self.numbers = (ctypes.c_longlong * len(numbers))(*numbers)
        self.at = ctypes.addressof(self.numbers)
        self.copy, self.shape, self.work, self.like, self.spans = copy, shape, work, like, spans
        self.apart = set()         # distances at which tensors of this layout have been found not to share memory


_plans: dict = {}


def planned(layout, make):
    """The plan of a layout, or False where the kernels do not apply."""
    plan = _plans.get(layout)
    if plan is None:
        if len(_plans) >= 4096:
            _plans.clear()
        plan = _plans[layout] = make()
    return plan


def strides(t, n=None):
    return list(t.stride()[:-1]) if t is not None else [0] * n


def rows_on(t, align: int) -> bool:
    """Whether every row of the tensor is contiguous and lies on ``align`` bytes, as far as the strides go."""
    if t is None:
        return True
    es = t.element_size()
    return (t.shape[-1] == 1 or t.stride(-1) == 1) and all(s * es % align == 0 for s in t.stride()[:-1]) and near(t)


def near(t) -> bool:
    """Steps between tokens and heads are 32-bit numbers of bytes in the kernels; those between pages are not."""
    return all(s < 2 ** 30 for s in (t.stride()[1:] if t.dim() == 4 else t.stride()))


def width_ok(t, step: int, most: int) -> bool:
    return t is None or (t.shape[-1] % step == 0 and step <= t.shape[-1] <= most)


def _rows_of_pages(table) -> bool:
    """Whether the rows of a block table can be read in place; one without entries never is."""
    return table.numel() == 0 or table.shape[1] == 1 or table.stride(1) == 1


def _scales(t):
    """Exponent bytes are read and written through one index."""
    return t is None or t.is_contiguous()


def _caches_ok(k_cache, v_cache, k_scale, v_scale, align, step, most):
    return (rows_on(k_cache, align) and rows_on(v_cache, align) and width_ok(k_cache, step, most) and width_ok(v_cache, step, most)
            and _scales(k_scale) and _scales(v_scale) and k_cache.shape[0] < 2 ** 31 and k_cache.shape[1] < 2 ** 31)


def _plan_write(k, v, k_cache, v_cache, slots, k_scale, v_scale):
    q = k_cache.dtype == E4M3
    T, heads, dim = k.shape
    if not (k.dtype in TYPES and _caches_ok(k_cache, v_cache, k_scale, v_scale, 8 if q else 16, 8, 256) and T * max(1, heads) < 2 ** 30):
        return False
    return Plan([*strides(k), *strides(v, 2), *strides(k_cache), *strides(v_cache, 3), T, heads, dim, 0 if v is None else v.shape[2],
                 k_cache.shape[0], k_cache.shape[1], TYPES[k.dtype], int(q), int(slots.dtype == torch.int64)],
                copy=not (rows_on(k, 16) and rows_on(v, 16) and slots.is_contiguous()),
                spans=[F_.bytes_spanned(t) for t in (k, v, k_cache, v_cache, k_scale, v_scale)])


@_on_device
def cache_write(k, v, k_cache, v_cache, slots, k_scale, v_scale, layout) -> bool:
    """False where the kernel does not apply."""
    plan = planned(layout, lambda: _plan_write(k, v, k_cache, v_cache, slots, k_scale, v_scale))
    if not plan or not _bare(k, v, k_cache, v_cache, slots, k_scale, v_scale):
        return False
    at, kp, vp, kcp, vcp, ksp, vsp = slots.data_ptr(), k.data_ptr(), _ptr(v), k_cache.data_ptr(), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale)
    if (kcp | (vcp or 0)) & (7 if k_scale is not None else 15):
        return False
    k_bytes, v_bytes, kc_bytes, vc_bytes, ks_bytes, vs_bytes = plan.spans
    inside = -k_bytes < kp - kcp < kc_bytes               # ranges of memory that have bytes in common
    if vp:
        inside = inside or -k_bytes < kp - vcp < vc_bytes or -v_bytes < vp - kcp < kc_bytes or -v_bytes < vp - vcp < vc_bytes
        if -kc_bytes < kcp - vcp < vc_bytes and kcp - vcp not in plan.apart:      # keys and values in one buffer
            F_.check_apart(k_cache, v_cache)
            plan.apart.add(kcp - vcp)
        if vsp and -ks_bytes < ksp - vsp < vs_bytes and (ksp - vsp,) not in plan.apart:
            F_.check_apart(k_scale, v_scale)
            plan.apart.add((ksp - vsp,))
    if plan.copy or inside or (kp | (vp or 0)) & 15:      # a few rows; or rows of the cache itself, read before any is overwritten
        k, v = (None if t is None else t.detach().clone(memory_format=torch.contiguous_format) for t in (k, v))
        slots = slots.contiguous()
        return cache_write(k, v, k_cache, v_cache, slots, k_scale, v_scale, F_.layout_of("cache_write", k, v, k_cache, v_cache, slots, k_scale, v_scale))
    rc = _cu.lib().cm_cache_write(kp, vp, kcp, vcp, ksp, vsp, at, plan.at, _cu.err_word(k.device).data_ptr(), _cu.stream_ptr())
    if rc:
        _failed("cm_cache_write", rc)
    F_.count_launch("cache_write")
    # whoever saved them for a gradient is told (tensors of inference mode cannot be saved and have no count)
    increment_version([t for t in (k_cache, v_cache, k_scale, v_scale) if t is not None and not t.is_inference()])
    return True


def _plan_read(k_cache, v_cache, table, ends, total, k_scale, v_scale, dtype):
    q = k_cache.dtype == E4M3
    heads, dim, vdim = k_cache.shape[2], k_cache.shape[3], 0 if v_cache is None else v_cache.shape[3]
    if not (dtype in TYPES and _caches_ok(k_cache, v_cache, k_scale, v_scale, 8 if q else 16, 8, 256) and total * max(1, heads) < 2 ** 30):
        return False
    return Plan([heads * dim, dim, heads * vdim, vdim, *strides(k_cache), *strides(v_cache, 3), total, heads, dim, vdim, k_cache.shape[0],
                 k_cache.shape[1], TYPES[dtype], int(q), table.stride(0), table.shape[0], table.shape[1]],
                copy=not (_rows_of_pages(table) and ends.is_contiguous()),
                shape=((total, heads, dim), (total, heads, vdim)))


@_on_device
def cache_read(k_cache, v_cache, table, ends, total, k_scale, v_scale, dtype, layout):
    """None where the kernel does not apply."""
    plan = planned(layout, lambda: _plan_read(k_cache, v_cache, table, ends, total, k_scale, v_scale, dtype))
    if (not plan or not _bare(k_cache, v_cache, table, ends, k_scale, v_scale)
            or (torch.is_grad_enabled() and (k_cache.requires_grad or (v_cache is not None and v_cache.requires_grad)))):
        return None
    kcp, vcp = k_cache.data_ptr(), _ptr(v_cache)
    if (kcp | (vcp or 0)) & (7 if k_scale is not None else 15):
        return None
    if plan.copy:
        table, ends = table.contiguous(), ends.contiguous()
        layout = (F_.layout_of("cache_read", k_cache, v_cache, table, ends, k_scale, v_scale), total, dtype)
        return cache_read(k_cache, v_cache, table, ends, total, k_scale, v_scale, dtype, layout)
    dev = k_cache.device
    k = torch.empty(plan.shape[0], dtype=dtype, device=dev)
    v = None if v_cache is None else torch.empty(plan.shape[1], dtype=dtype, device=dev)
    rc = _cu.lib().cm_cache_read(k.data_ptr(), _ptr(v), kcp, vcp, _ptr(k_scale), _ptr(v_scale), table.data_ptr(), ends.data_ptr(), plan.at,
                                 _cu.err_word(dev).data_ptr(), _cu.stream_ptr())
    if rc:
        _failed("cm_cache_read", rc)
    F_.count_launch("cache_read")
    return k, v


def _plan_attention(q, k_cache, v_cache, table, lens, k_scale, v_scale):
    e4m3 = k_cache.dtype == E4M3
    B, H, dim = q.shape
    pages, page, heads, vdim = v_cache.shape
    group, columns = H // heads, table.shape[1]
    if not (q.dtype in TYPES and (e4m3 or k_cache.dtype == q.dtype) and _caches_ok(k_cache, v_cache, k_scale, v_scale, 16, 16 if e4m3 else 8, 128)
            and 0 < group <= 128 and columns * page < 2 ** 31 - 16 and B * H < 2 ** 31):
        return False
    return Plan([*strides(q), *strides(k_cache), *strides(v_cache), table.stride(0), B, heads, group, columns, pages, page, dim, vdim,
                 TYPES[q.dtype], int(e4m3)],
                copy=not (rows_on(q, 16) and _rows_of_pages(table) and lens.is_contiguous()), shape=(B, H, vdim),
                work=_cu.lib().cm_paged_attention_ws(B, heads, group, dim, vdim, columns, page, int(e4m3)) if B else 0,
                like=q.is_contiguous() and vdim == dim)


@_on_device
def paged_attention(q, k_cache, v_cache, table, lens, scale, k_scale, v_scale, layout):
    """None where the kernels do not apply."""
    plan = planned(layout, lambda: _plan_attention(q, k_cache, v_cache, table, lens, k_scale, v_scale))
    if (not plan or isinstance(scale, torch.Tensor) or not abs(scale) < 2.0 ** 64 or not _bare(q, k_cache, v_cache, table, lens, k_scale, v_scale)
            or (torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad))):
        return None
    qp, kp, vp = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    if (kp | vp) & 15:
        return None
    if plan.copy or qp & 15:
        q, table, lens = q.clone(memory_format=torch.contiguous_format), table.contiguous(), lens.contiguous()
        return paged_attention(q, k_cache, v_cache, table, lens, scale, k_scale, v_scale,
                               F_.layout_of("paged_attention", q, k_cache, v_cache, table, lens, k_scale, v_scale))
    dev = q.device
    out = torch.empty_like(q) if plan.like else torch.empty(plan.shape, dtype=q.dtype, device=dev)
    ws = torch.empty(plan.work, dtype=torch.float32, device=dev)
    # a cache of no pages lies nowhere: the copies of no bytes that stand for its rows name the query's memory
    rc = _cu.lib().cm_paged_attention(qp, kp or qp, vp or qp, _ptr(k_scale), _ptr(v_scale), table.data_ptr(), lens.data_ptr(), out.data_ptr(), ws.data_ptr(),
                                      plan.at, float(scale), _cu.err_word(dev).data_ptr(), _cu.stream_ptr())
    if rc:
        _failed("cm_paged_attention", rc)
    F_.count_launch("paged_attention")
    return out


def register() -> None:
    F_.register_cuda("cache_write", cache_write)
    F_.register_cuda("cache_read", cache_read)
    F_.register_cuda("paged_attention", paged_attention)
