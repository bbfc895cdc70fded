"""The paged key-value cache (``csrc/paged_cache.cu``) and the attention of one new token per sequence over it (``csrc/paged_attention.cu``).

Tensors are read where they are: strides of a cache are free as long as a row (the last axis) is contiguous and lies on 16 bytes.
Work space is allocated per call on the current stream, and nothing waits for the device.
"""
from __future__ import annotations

import ctypes

import torch

from .. import cuda as _cu
from .. import functional as F_
from .block import _bare, _failed, _on_device, _ptr

TYPES = {torch.bfloat16: 0, torch.float16: 1}
E4M3 = torch.float8_e4m3fn


def declare(L: ctypes.CDLL) -> None:
    vp, i32, i64, f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float
    sig = {
        "cm_cache_write": [vp] * 11 + [i32] * 9 + [vp, vp],
        "cm_cache_read": [vp] * 11 + [i64, vp] + [i32] * 10 + [vp, vp],
        "cm_paged_attention": [vp] * 9 + [i64, vp, vp, vp] + [i32] * 8 + [f32, i32, i32, vp, vp],
    }
    for name, args in sig.items():
        if hasattr(L, name):
            getattr(L, name).argtypes, getattr(L, name).restype = args, i32
    if hasattr(L, "cm_paged_attention_ws"):
        L.cm_paged_attention_ws.argtypes, L.cm_paged_attention_ws.restype = [i32] * 7, i64


def _strides(t):
    """Strides of all axes but the last, as the library takes them."""
    return None if t is None else (ctypes.c_longlong * (t.dim() - 1))(*t.stride()[:-1])


def _rows_on(t, align: int) -> bool:
    """Whether every row of the tensor is contiguous and begins on ``align`` bytes."""
    if t is None:
        return True
    es = t.element_size()
    return (t.shape[-1] == 1 or t.stride(-1) == 1) and t.data_ptr() % align == 0 and all(s * es % align == 0 for s in t.stride()[:-1])


def _packed_rows(t, align: int = 16):
    """A few rows: copied where the kernels cannot read them in place."""
    return t if t is None or _rows_on(t, align) else t.clone(memory_format=torch.contiguous_format)


def _width_ok(t, step: int, most: int) -> bool:
    return t is None or (t.shape[-1] % step == 0 and step <= t.shape[-1] <= most)


def _scales(t):
    """Exponent bytes are read and written through one index."""
    return t is None or t.is_contiguous()


@_on_device
def cache_write(k, v, k_cache, v_cache, slots, k_scale, v_scale) -> bool:
    """False where the kernel does not apply."""
    q = k_cache.dtype == E4M3
    if not (k.dtype in TYPES and _bare(k, v, k_cache, v_cache, slots) and _width_ok(k, 8, 256) and _width_ok(v, 8, 256)
            and _rows_on(k_cache, 8 if q else 16) and _rows_on(v_cache, 8 if q else 16) and _scales(k_scale) and _scales(v_scale)
            and k.shape[0] * max(1, k.shape[1]) < 2 ** 30 and k_cache.shape[0] < 2 ** 31 and k_cache.shape[1] < 2 ** 31):
        return False
    T, heads, dim = k.shape
    if T == 0 or heads == 0:
        return True
    k, v, slots = _packed_rows(k.detach()), _packed_rows(None if v is None else v.detach()), slots.contiguous()
    rc = _cu.lib().cm_cache_write(
        k.data_ptr(), _strides(k), _ptr(v), _strides(v), k_cache.data_ptr(), _strides(k_cache), _ptr(v_cache), _strides(v_cache),
        _ptr(k_scale), _ptr(v_scale), slots.data_ptr(), int(slots.dtype == torch.int64), T, heads, dim, 0 if v is None else v.shape[2],
        k_cache.shape[0], k_cache.shape[1], TYPES[k.dtype], int(q), _cu.err_word(k.device).data_ptr(), _cu.stream_ptr())
    if rc:
        _failed("cm_cache_write", rc)
    F_.count_launch("cache_write")
    return True


@_on_device
def cache_read(k_cache, v_cache, table, ends, total, k_scale, v_scale, dtype):
    """None where the kernel does not apply."""
    q = k_cache.dtype == E4M3
    heads = k_cache.shape[2]
    if not (dtype in TYPES and _bare(k_cache, v_cache, table, ends) and _width_ok(k_cache, 8, 256) and _width_ok(v_cache, 8, 256)
            and _rows_on(k_cache, 8 if q else 16) and _rows_on(v_cache, 8 if q else 16) and _scales(k_scale) and _scales(v_scale)
            and not (torch.is_grad_enabled() and (k_cache.requires_grad or (v_cache is not None and v_cache.requires_grad)))
            and total * max(1, heads) < 2 ** 30 and k_cache.shape[0] < 2 ** 31):
        return None
    k = torch.empty(total, heads, k_cache.shape[3], dtype=dtype, device=k_cache.device)
    v = None if v_cache is None else torch.empty(total, heads, v_cache.shape[3], dtype=dtype, device=k_cache.device)
    if total == 0 or heads == 0:
        return k, v
    if table.stride(-1) != 1:
        table = table.contiguous()
    ends = ends.contiguous()
    rc = _cu.lib().cm_cache_read(
        k.data_ptr(), _strides(k), _ptr(v), _strides(v), k_cache.data_ptr(), _strides(k_cache), _ptr(v_cache), _strides(v_cache),
        _ptr(k_scale), _ptr(v_scale), table.data_ptr(), table.stride(0), ends.data_ptr(), table.shape[0], table.shape[1], total, heads,
        k.shape[2], 0 if v is None else v.shape[2], k_cache.shape[0], k_cache.shape[1], TYPES[dtype], int(q),
        _cu.err_word(k.device).data_ptr(), _cu.stream_ptr())
    if rc:
        _failed("cm_cache_read", rc)
    F_.count_launch("cache_read")
    return k, v


@_on_device
def paged_attention(q, k_cache, v_cache, table, lens, scale, k_scale, v_scale):
    """None where the kernels do not apply."""
    e4m3 = k_cache.dtype == E4M3
    B, H, dim = q.shape
    pages, page, heads, vdim = v_cache.shape
    step = 16 if e4m3 else 8
    if not (q.dtype in TYPES and (e4m3 or k_cache.dtype == q.dtype) and not isinstance(scale, torch.Tensor)
            and _bare(q, k_cache, v_cache, table, lens) and _width_ok(k_cache, step, 128) and _width_ok(v_cache, step, 128)
            and H // heads <= 128 and _rows_on(k_cache, 16) and _rows_on(v_cache, 16) and _scales(k_scale) and _scales(v_scale)
            and table.shape[1] * page < 2 ** 31 - 16 and B * H < 2 ** 31 and pages < 2 ** 31):
        return None
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        return None
    out = torch.empty(B, H, vdim, dtype=q.dtype, device=q.device)
    if B == 0 or H == 0:
        return out
    q, lens = _packed_rows(q), lens.contiguous()
    if table.stride(-1) != 1:
        table = table.contiguous()
    L, group, columns = _cu.lib(), H // heads, table.shape[1]
    ws = torch.empty(L.cm_paged_attention_ws(B, heads, group, dim, vdim, columns, page), dtype=torch.float32, device=q.device)
    rc = L.cm_paged_attention(
        q.data_ptr(), _strides(q), k_cache.data_ptr(), _strides(k_cache), v_cache.data_ptr(), _strides(v_cache), _ptr(k_scale), _ptr(v_scale),
        table.data_ptr(), table.stride(0), lens.data_ptr(), out.data_ptr(), ws.data_ptr(), B, heads, group, columns, pages, page, dim, vdim,
        float(scale), TYPES[q.dtype], int(e4m3), _cu.err_word(q.device).data_ptr(), _cu.stream_ptr())
    if rc:
        _failed("cm_paged_attention", rc)
    F_.count_launch("paged_attention")
    return out


def register() -> None:
    F_.register_cuda("cache_write", cache_write)
    F_.register_cuda("cache_read", cache_read)
    F_.register_cuda("paged_attention", paged_attention)
