"""Operator front door.

Every model calls the functions here.  On a CUDA tensor they run the sm_100a
kernels from :mod:`cppmega_b200.ops.cuda` (wrapped in autograd Functions); on a CPU
tensor they run the PyTorch definitions in :mod:`cppmega_b200.ops.reference`.  A CUDA call
for which no kernel is registered is counted in :func:`fallback_counts` and runs
the PyTorch definition on the GPU, so a training log can prove "zero fallbacks"
(the reference keeps equivalent counters for its MXFP8 routing,
scripts/cppmega_fp8_shim.py:445-500).  If the extension failed to load on a machine
that has a GPU, the first CUDA call raises instead of silently falling back.
"""
from __future__ import annotations

import collections
import operator
from typing import Callable, Dict, Optional

import torch
import torch.nn.functional as F

from . import reference as ref
from . import mimo_scan_ref

_CUDA_IMPL: Dict[str, Callable] = {}
_FALLBACKS: "collections.Counter[str]" = collections.Counter()
_LAUNCHES: "collections.Counter[str]" = collections.Counter()
_DISABLED: set = set()
_ext_checked = False


def register_cuda(name: str, fn: Callable) -> None:
    _CUDA_IMPL[name] = fn


def disable_cuda(*names: str) -> None:
    """Route the named ops through the PyTorch definitions (used by A/B benchmarks)."""
    _DISABLED.update(names)


def enable_cuda(*names: str) -> None:
    for n in names:
        _DISABLED.discard(n)


# kernels whose reductions use floating-point atomics (the order of the additions, hence the last bits, varies from run to run)
ATOMIC_REDUCTION_OPS = ("embedding", "ngram_hash_embed", "causal_conv1d_silu", "head_linear", "sparse_mla", "mimo_scan_bwd",
                        "causal_attention")
_deterministic = False


def set_deterministic(on: bool = True) -> None:
    """Bitwise-reproducible reruns for debugging: the operators in ``ATOMIC_REDUCTION_OPS`` go through their PyTorch
    definitions and the tensor library is put in deterministic mode (it then refuses or replaces its own atomic kernels).
    Slower; meant for comparing two runs of a few steps, e.g. when hunting a race in a new kernel."""
    global _deterministic
    _deterministic = bool(on)
    if on:
        disable_cuda(*ATOMIC_REDUCTION_OPS)
    else:
        enable_cuda(*ATOMIC_REDUCTION_OPS)
    torch.use_deterministic_algorithms(bool(on), warn_only=True)


def is_deterministic() -> bool:
    return _deterministic


def fallback_counts() -> Dict[str, int]:
    return dict(_FALLBACKS)


def launch_counts() -> Dict[str, int]:
    """Number of calls that reached one of this package's own CUDA kernels, per op."""
    return dict(_LAUNCHES)


def reset_counters() -> None:
    _FALLBACKS.clear()
    _LAUNCHES.clear()


def count_launch(name: str, n: int = 1) -> None:
    _LAUNCHES[name] += n


def _ensure_ext() -> None:
    global _ext_checked
    if _ext_checked:
        return
    _ext_checked = True
    from . import cuda  # noqa: F401  (registers kernels; raises if the .so is missing on a GPU box)


def _miss(name: str, t: torch.Tensor) -> None:
    """A CUDA call that ends in a PyTorch / library kernel instead of one of this package's kernels."""
    if t.is_cuda:
        _FALLBACKS[name] += 1


def _cuda(name: str, *tensors) -> Optional[Callable]:
    t = tensors[0]
    if not t.is_cuda:
        return None
    _ensure_ext()
    fn = _CUDA_IMPL.get(name)
    if fn is None or name in _DISABLED:
        _FALLBACKS[name] += 1
        return None
    return fn


def _same_device(name: str, first: torch.Tensor, *others) -> None:
    dev = first.device
    for t in others:
        if t is not None and t.device != dev:
            raise ValueError(f"{name}: tensors on {dev} and {t.device}")


# ---- dense ---------------------------------------------------------------

_PRECISION_RECIPE = "bf16"
RECIPES = ("bf16", "mxfp8", "tensorwise")


def set_precision_recipe(name: str) -> None:
    """Precision of the linear layers (2-D bf16 weight, all three dims multiples of 32) and the expert GEMMs:

    * ``bf16``: bf16 operands;
    * ``mxfp8``: operands rounded to E4M3 with one E8M0 scale per 32 values along the reduced dimension; the activation
      saved for the weight gradient is kept in that form;
    * ``tensorwise``: E4M3 with ONE power-of-two scale per tensor, measured from the tensor at every use (current
      scaling) - the reference's production FP8 recipe (docs/production_status.md:13-18) on the same kernels.

    This is the process-wide default; :func:`precision_scope` and :func:`install_precision_rules` narrow it to modules."""
    global _PRECISION_RECIPE
    if name not in RECIPES:
        raise ValueError(f"unknown precision recipe {name!r}")
    _PRECISION_RECIPE = name


def precision_recipe() -> str:
    return _PRECISION_RECIPE


class precision_scope:
    """``with precision_scope("mxfp8"): ...`` - the recipe of every linear called inside (forward; each op remembers its
    recipe for its backward)."""

    def __init__(self, name: str):
        if name not in RECIPES:
            raise ValueError(f"unknown precision recipe {name!r}")
        self.name = name

    def __enter__(self):
        self.prev = _PRECISION_RECIPE
        set_precision_recipe(self.name)
        return self

    def __exit__(self, *exc):
        set_precision_recipe(self.prev)
        return False


def install_precision_rules(model, rules, default: str = "bf16"):
    """Per-module precision selection.  ``rules``: sequence of ``(glob pattern, recipe)`` matched against the qualified
    module names of ``model`` (first match wins; e.g. ``("*.mixer.in_proj", "mxfp8")`` or ``("decoder.layers.*.mlp",
    "tensorwise")``); modules that match run their forward under that recipe, everything else under ``default``.
    Counterpart of the reference's layer-selective FP8 (cppmega/megatron/selective_fp8_moe_patch.py:60-149: FP8 on MoE
    layers only) and of its per-module precision file (configs/te_precision/mamba_mxfp8_eval_bf16.yaml:1-29: MXFP8 on
    the Mamba in / out projections only).  Returns ``(handles, matched module names)``; ``h.remove()`` undoes a hook."""
    import fnmatch
    set_precision_recipe(default)
    handles, matched = [], []
    for name, mod in model.named_modules():
        recipe = next((r for pat, r in rules if fnmatch.fnmatchcase(name, pat)), None)
        if recipe is None:
            continue
        if recipe not in RECIPES:
            raise ValueError(f"unknown precision recipe {recipe!r} for pattern matching {name!r}")
        stack = []

        def pre(_m, _args, recipe=recipe, stack=stack):
            stack.append(_PRECISION_RECIPE)
            set_precision_recipe(recipe)

        def post(_m, _args, _out, stack=stack):
            set_precision_recipe(stack.pop())

        handles.append(mod.register_forward_pre_hook(pre))
        handles.append(mod.register_forward_hook(post, always_call=True))
        matched.append(name)
    return handles, matched


def linear(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """``x @ w^T``; w is [out, in]."""
    if _PRECISION_RECIPE != "bf16" and x.is_cuda:
        _ensure_ext()
        from .cuda import mxfp8
        y = mxfp8.linear(x, w, tensorwise=_PRECISION_RECIPE == "tensorwise")
        if y is not None:
            return y
        _FALLBACKS["fp8_linear(shape)"] += 1
    fn = _cuda("linear", x)
    if fn is not None:
        y = fn(x, w)
        if y is not None:
            return y
        _miss("linear(shape/dtype)", x)
    return F.linear(x, w.to(x.dtype) if w.dtype != x.dtype else w)


def linear_fp32out(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """fp32 ``x @ weight.T`` for an fp32 parameter.  On the GPU with bf16 activations the products run on the tensor
    cores (bf16 operands, fp32 accumulation and output); elsewhere plain fp32."""
    fn = _cuda("linear_fp32out", x) if x.is_cuda and x.dtype == torch.bfloat16 else None
    if fn is not None:
        y = fn(x, weight)
        if y is not None:
            return y
    _miss("linear_fp32out(shape/dtype)", x)
    return F.linear(x.float(), weight.float())


def grouped_linear(x: torch.Tensor, w: torch.Tensor, counts: torch.Tensor, counts_host=None) -> torch.Tensor:
    """Rows of x sorted by expert; w [E, out, in]; counts [E] rows per expert."""
    fn = _cuda("grouped_linear", x)
    if fn is not None:
        y = fn(x, w, counts, counts_host)
        if y is not None:
            return y
        _miss("grouped_linear(shape)", x)
    ch = counts_host if counts_host is not None else counts.tolist()
    return ref.grouped_gemm(x, w.transpose(1, 2).to(x.dtype), ch)


def moe_experts(x_sorted: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, counts: torch.Tensor, counts_host=None):
    """SwiGLU expert MLP over expert-sorted rows: ``fc2(swiglu(fc1(x)))`` with per-expert weights
    ``w1`` [E, 2F, H] and ``w2`` [E, H, F]."""
    fn = _cuda("moe_experts", x_sorted)
    if fn is not None:
        y = fn(x_sorted, w1, w2, counts)
        if y is not None:
            return y
    h = grouped_linear(x_sorted, w1, counts, counts_host)
    return grouped_linear(swiglu(h), w2, counts, counts_host)


# ---- norms / activations ---------------------------------------------------

def rmsnorm(x, weight, eps: float = 1e-5):
    fn = _cuda("rmsnorm", x)
    if fn is not None:
        return fn(x, weight, eps)
    return ref.rmsnorm(x, weight, eps)


def rmsnorm_gated(x, weight, z=None, eps: float = 1e-5, group_size=None, norm_before_gate=True):
    """RMS norm of a mixer's output with a SiLU gate: ``rms(x) * weight * silu(z)``, or ``rms(x * silu(z)) * weight`` with
    ``norm_before_gate=False``; every ``group_size`` channels normalise apart (default: the whole row).  ``x``, ``z`` [..., D] of
    one type, rows of any pitch (column slices of a projection are read in place), ``weight`` [D].  The kernels have first derivatives;
    forward mode, function transforms and batches of upstream gradients run the definition, ``reference.rmsnorm_gated``."""
    D = x.shape[-1]
    group = int(group_size) if group_size else D
    fn = _cuda("rmsnorm_gated", x)
    if fn is not None:
        y = None
        if weight.shape == (D,) and (z is None or z.shape == x.shape) and D % group == 0:
            _same_device("rmsnorm_gated", x, weight, z)
            y = fn(x, weight, z, eps, group, norm_before_gate)
        if y is not None:
            return y
        _miss("rmsnorm_gated(shape/dtype)", x)
    return ref.rmsnorm_gated(x, weight, z, eps, group_size, norm_before_gate)


def residual_rmsnorm(y, residual, weight, post_weight=None, gate=None, scale: float = 1.0, eps: float = 1e-5):
    """The step between two blocks: ``h = residual + scale * gate * p`` with ``p = rms(y) * post_weight`` (``y`` itself without a
    post norm), and the norm the next block reads, ``n = rms(h) * weight``.  Returns ``(n, h)``, both in the type of ``y``; ``n``
    is the norm of ``h`` as rounded to that type.  ``y``, ``residual`` [..., D]; ``gate`` [D] (one per channel, shared by all
    rows) or the shape of ``y``; ``weight``, ``post_weight`` [D].  The kernels take ``scale`` as a number and have first derivatives; a
    scale that is a tensor, forward mode and function transforms run the definition, ``reference.residual_rmsnorm``."""
    row = y.shape[-1:]
    if residual.shape != y.shape:
        raise ValueError(f"residual_rmsnorm: block output {tuple(y.shape)}, residual {tuple(residual.shape)}")
    if weight.shape != row or (post_weight is not None and post_weight.shape != row):
        raise ValueError(f"residual_rmsnorm: weight {tuple(weight.shape)}, post_weight "
                         f"{None if post_weight is None else tuple(post_weight.shape)} for rows of {tuple(row)}")
    if gate is not None and gate.shape != row and gate.shape != y.shape:
        raise ValueError(f"residual_rmsnorm: gate {tuple(gate.shape)} is neither {tuple(row)} nor {tuple(y.shape)}")
    _same_device("residual_rmsnorm", y, residual, weight, post_weight, gate)
    fn = _cuda("residual_rmsnorm", y)
    if fn is not None:
        out = fn(y, residual, weight, post_weight, gate, scale, eps)
        if out is not None:
            return out
        _miss("residual_rmsnorm(shape/dtype)", y)
    return ref.residual_rmsnorm(y, residual, weight, post_weight, gate, scale, eps)


def head_linear(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """Per-head product ``y[..., h, :] = x[..., h, :] @ w[h]^T`` with ``x`` [..., H, in] and ``w`` [H, out, in] (the
    absorbed MLA up-projections of the sparse-attention path).  64-wide heads in bf16 run on the streaming tcgen05 kernel;
    anything else is a batched library GEMM and is counted."""
    fn = _cuda("head_linear", x)
    if fn is not None:
        y = fn(x, w)
        if y is not None:
            return y
    _miss("head_linear(library bmm)", x)
    return torch.einsum("...hi,hoi->...ho", x, w.to(x.dtype))


def gated_mlp(x, w1, w2, activation: str = "silu"):
    """Gated feed-forward block ``(act(x Wg^T) * (x Wu^T)) W2^T``: ``x`` [..., H], ``w1`` [2F, H] (the gate rows, then the up rows),
    ``w2`` [Ho, F]; ``activation`` is ``silu``, ``gelu_tanh`` or ``relu``.  In bf16 with widths that are multiples of 8 the
    projections, the activation and the product are one kernel, and so are their gradients (first derivatives); under an FP8 recipe,
    and for anything else, it is :func:`linear`, activation, :func:`linear`."""
    if activation not in ref.GATED_ACTIVATIONS:
        raise ValueError(f"gated_mlp: unknown activation {activation!r}, one of {sorted(ref.GATED_ACTIVATIONS)}")
    if w1.dim() != 2 or w2.dim() != 2 or x.dim() < 1 or w1.shape[1] != x.shape[-1] or w1.shape[0] != 2 * w2.shape[1]:
        raise ValueError(f"gated_mlp: x {tuple(x.shape)}, w1 {tuple(w1.shape)}, w2 {tuple(w2.shape)}")
    _same_device("gated_mlp", x, w1, w2)
    if x.numel() == 0 or w1.numel() == 0 or w2.numel() == 0:       # a sum over nothing is zero: no kernel has anything to read
        return ref.gated_mlp(x, w1, w2, activation)
    fn = _cuda("gated_mlp", x) if _PRECISION_RECIPE == "bf16" else None
    if fn is not None:
        y = fn(x, w1, w2, activation)
        if y is not None:
            return y
        _miss("gated_mlp(shape/dtype)", x)
    gate_up = linear(x, w1)
    return linear(swiglu(gate_up) if activation == "silu" else ref.gated_activation(gate_up, activation), w2)


def swiglu(gate_up):
    fn = _cuda("swiglu", gate_up)
    if fn is not None:
        return fn(gate_up)
    return ref.swiglu(gate_up)


def apply_rope(x, cos, sin):
    fn = _cuda("apply_rope", x)
    if fn is not None:
        y = fn(x, cos, sin)
        if y is not None:
            return y
        _miss("apply_rope(shape)", x)
    return ref.apply_rope(x, cos, sin)


# ---- embeddings --------------------------------------------------------------

def ngram_hash_embed(token_ids, table, mults, bias, table_sizes, table_offsets, order_of_table):
    fn = _cuda("ngram_hash_embed", table)
    if fn is not None:
        out = fn(token_ids, table, mults, bias, table_sizes, table_offsets, order_of_table)
        if out is not None:
            return out
        _miss("ngram_hash_embed(shape)", table)
    return ref.ngram_hash_embed(token_ids, table, mults, bias, table_sizes, table_offsets, order_of_table)


# ---- sequence mixers ----------------------------------------------------------

def mimo_scan(Q, K, V, ADT, DT, Trap, Q_bias, K_bias, Psi, Zeta, Phi, angles, D, Z,
              rotary_dim_divisor: int = 4, chunk_size: int = 16):
    fn = _cuda("mimo_scan", V)
    if fn is not None:
        return fn(Q, K, V, ADT, DT, Trap, Q_bias, K_bias, Psi, Zeta, Phi, angles, D, Z,
                  rotary_dim_divisor, chunk_size)
    if V.is_cuda and None not in (Zeta, Phi, D, Z):
        from .mimo_scan_lean import mimo_scan_lean     # PyTorch on GPU, one head group at a time
        return mimo_scan_lean(Q, K, V, ADT, DT, Trap, Q_bias, K_bias, Psi, Zeta, Phi, angles, D, Z,
                              rotary_dim_divisor, 64)
    return mimo_scan_ref.mimo_scan_chunked(Q, K, V, ADT, DT, Trap, Q_bias, K_bias, Psi, Zeta, Phi,
                                           angles, D, Z, rotary_dim_divisor, chunk_size)


def angle_cumsum(angles_raw, dt):
    fn = _cuda("angle_cumsum", angles_raw)
    if fn is not None:
        out = fn(angles_raw, dt)
        if out is not None:
            return out
        _miss("angle_cumsum(shape)", angles_raw)
    return mimo_scan_ref.angle_cumsum(angles_raw, dt)


def m2rnn_scan(q, k, v, W, f):
    fn = _cuda("m2rnn_scan", v)
    if fn is not None:
        return fn(q, k, v, W, f)
    return ref.m2rnn_scan(q, k, v, W, f)[0]


# ---- DSA ---------------------------------------------------------------------

def indexer_topk(q_idx, k_idx, w, topk: int, q_offset: Optional[int] = None):
    """``q_offset``: sequence position of query 0 when the keys cover more than the queries (context parallelism: the
    keys are gathered over the group, the queries are this rank's chunk); ``None``: queries are the last positions."""
    plain = q_offset is None or (q_offset == 0 and k_idx.shape[1] == q_idx.shape[1])
    fn = _cuda("indexer_topk", q_idx) if plain else None
    if fn is not None:
        with torch.no_grad():
            out = fn(q_idx, k_idx, w, topk)
        if out is not None:
            return out
        _FALLBACKS["indexer_topk(shape)"] += 1
    elif not plain:
        _miss("indexer_topk(query offset)", q_idx)
    with torch.no_grad():
        return ref.indexer_topk(q_idx, k_idx, w, topk, q_offset)


def sparse_mla(q, kv, indices, scale: float, d_v: int):
    fn = _cuda("sparse_mla", q)
    if fn is not None:
        out = fn(q, kv, indices, scale, d_v)
        if out is not None:
            return out
        _FALLBACKS["sparse_mla(shape)"] += 1
    return ref.sparse_mla(q, kv, indices, scale, d_v)[0]


def causal_attention(q, k, v, scale: float):
    """Dense causal attention, q/k [B,S,H,Dqk], v [B,S,H,Dv]."""
    fn = _cuda("causal_attention", q)
    if fn is not None:
        return fn(q, k, v, scale)
    return causal_attention_library(q, k, v, scale)


def causal_attention_library(q, k, v, scale: float):
    """The library path (``scaled_dot_product_attention``): CPU, and shapes the kernel does not take."""
    dq, dv = q.shape[-1], v.shape[-1]
    if q.is_cuda and dv < dq:          # library flash kernels want one head size: zero-pad V
        v = F.pad(v, (0, dq - dv))
    o = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2),
                                       is_causal=True, scale=scale)
    return o.transpose(1, 2)[..., :dv]


_CHECKED: set = set()


def layout_of(name: str, *tensors):
    """Everything about a call's tensors but their addresses and values: what its checks and its plan go by."""
    return (name, *[None if t is None else (t.shape, t.stride(), t.dtype, t.device) for t in tensors])


def _checked(layout) -> None:
    """Calls of this layout pass their checks."""
    if len(_CHECKED) >= 4096:
        _CHECKED.clear()
    _CHECKED.add(layout)


def bytes_spanned(t) -> int:
    """Bytes from a tensor's first element to the end of its last one."""
    if t is None or t.numel() == 0:
        return 0
    return (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _axes(t) -> list:
    """(bytes of a step, steps) of the axes that have any, the widest first."""
    return sorted(((s * t.element_size(), n) for n, s in zip(t.shape, t.stride()) if n > 1), reverse=True)


def _nested(t) -> bool:
    """Whether every axis steps over all that the narrower ones reach: no two elements share memory."""
    reach = t.element_size()
    for step, n in reversed(_axes(t)):
        if step < reach:
            return False
        reach += (n - 1) * step
    return True


def _share_memory(a, b) -> bool:
    """Whether two nested tensors have bytes in common.  Their axes are gone through from the widest in; where that would take long (steps that
    do not match, lying in one another many times) they count as if they had."""
    budget = 4096

    def meet(x, y, off) -> bool:               # elements of x from 0 on, of y from `off` on
        nonlocal budget
        budget -= 1
        x_reach, y_reach = (sum((n - 1) * s for s, n in axes) + e for axes, e in ((x, a.element_size()), (y, b.element_size())))
        if off >= x_reach or off + y_reach <= 0:
            return False
        if not (x or y) or budget < 0:
            return True
        if x and y and x[0][0] == y[0][0]:     # a step of one against a step of the other: only their difference counts
            (step, nx), (_, ny) = x[0], y[0]
            x_in, y_in = x_reach - (nx - 1) * step, y_reach - (ny - 1) * step
            first, last = max(1 - nx, (-off - y_in) // step + 1), min(ny - 1, -((off - x_in) // step) - 1)
            return any(meet(x[1:], y[1:], off + i * step) for i in range(first, last + 1))
        if not y or (x and x[0] > y[0]):
            step, n = x[0]
            inside = x_reach - (n - 1) * step
            first, last = max(0, (off - inside) // step + 1), min(n - 1, -((-off - y_reach) // step) - 1)
            return any(meet(x[1:], y, off - i * step) for i in range(first, last + 1))
        step, n = y[0]
        inside = y_reach - (n - 1) * step
        first, last = max(0, (-off - inside) // step + 1), min(n - 1, -((off - x_reach) // step) - 1)
        return any(meet(x, y[1:], off + i * step) for i in range(first, last + 1))

    return a.numel() > 0 and b.numel() > 0 and meet(_axes(a), _axes(b), b.data_ptr() - a.data_ptr())


def _sequence_ends(name: str, ends, like: torch.Tensor) -> None:
    if ends.dtype != torch.int32 or ends.dim() != 1 or ends.numel() < 1:
        raise ValueError(f"{name}: sequence ends are int32 [sequences + 1], got {ends.dtype} {tuple(ends.shape)}")
    _same_device(name, like, ends)


def _check_packed(q, k, v, cu_seqlens, cu_seqlens_k) -> None:
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3 or k.shape[:2] != v.shape[:2] or q.shape[2] != k.shape[2]:
        raise ValueError(f"packed_attention: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if k.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise ValueError(f"packed_attention: {q.shape[1]} query heads over {k.shape[1]} key heads")
    if q.dtype != k.dtype or q.dtype != v.dtype:
        raise ValueError(f"packed_attention: q {q.dtype}, k {k.dtype}, v {v.dtype}")
    _same_device("packed_attention", q, k, v)
    _sequence_ends("packed_attention", cu_seqlens, q)
    if cu_seqlens_k is not None:
        _sequence_ends("packed_attention", cu_seqlens_k, q)
        if cu_seqlens_k.shape != cu_seqlens.shape:
            raise ValueError(f"packed_attention: {cu_seqlens.numel() - 1} sequences of queries, {cu_seqlens_k.numel() - 1} of keys")
    elif k.shape[0] != q.shape[0]:
        raise ValueError(f"packed_attention: {q.shape[0]} queries and {k.shape[0]} keys without cu_seqlens_k")


def packed_attention(q, k, v, cu_seqlens, scale: float, cu_seqlens_k=None):
    """Causal attention over sequences of different lengths packed into one buffer, with grouped heads:
    ``o[i] = sum_j softmax_j(scale q[i] . k[j]) v[j]`` over the keys of the query's own sequence up to its position.

    ``q`` [T, H, D], ``k`` [Tk, G, D], ``v`` [Tk, G, Dv], ``H`` a multiple of ``G``; result [T, H, Dv].  ``cu_seqlens`` int32 [n + 1]
    on the tensors' device: sequence ``s`` is the rows ``cu_seqlens[s] .. cu_seqlens[s + 1] - 1``, from row 0 on.  ``cu_seqlens_k`` gives the keys
    their own ends: a sequence's queries are then its last positions (the continuation of a prompt whose keys were read back from a cache).  A
    query without keys gives zeros, and so do the rows behind the last sequence, whatever they hold.  Within a sequence a key that is not finite
    reaches earlier queries too where it shares a tile with them (a weight of zero times infinity).

    bf16 and fp16 with ``D`` and ``Dv`` multiples of 8 up to 128 run on the kernels, in training with their gradients (first
    derivatives; the same call gives the same bits); strided tensors are read in place where rows lie on 16 bytes.
    Anything else, forward mode and function transforms run the definition, ``reference.packed_attention``, which reads the ends on the host.  A CUDA
    graph takes forward and backward together, while no eager graph of the same leaves is alive (autograd would add to those on the eager stream).  The
    kernels' calls, those without queries, keys or heads among them, wait for nothing: ends that fall or run over the buffer are reported by
    ``ops.cuda.check_errors``."""
    layout = layout_of("packed_attention", q, k, v, cu_seqlens, cu_seqlens_k)
    if layout not in _CHECKED:
        _check_packed(q, k, v, cu_seqlens, cu_seqlens_k)
        _checked(layout)
    fn = _cuda("packed_attention", q)
    if fn is not None:
        o = fn(q, k, v, cu_seqlens, scale, cu_seqlens_k, layout)
        if o is not None:
            return o
        _miss("packed_attention(shape/dtype)", q)
    return ref.packed_attention(q, k, v, cu_seqlens, scale, cu_seqlens_k)


def _check_cache(name: str, k_cache, v_cache, k_scale, v_scale) -> None:
    if k_cache.dim() != 4 or (v_cache is not None and (v_cache.dim() != 4 or v_cache.shape[:3] != k_cache.shape[:3])):
        raise ValueError(f"{name}: caches {tuple(k_cache.shape)} and {None if v_cache is None else tuple(v_cache.shape)} are not "
                         "[pages, page, heads, width]")
    if k_cache.shape[1] < 1:
        raise ValueError(f"{name}: pages of no tokens")
    if v_cache is not None and v_cache.dtype != k_cache.dtype:
        raise ValueError(f"{name}: caches of {k_cache.dtype} and {v_cache.dtype}")
    quantised = k_cache.dtype == torch.float8_e4m3fn
    for cache, scale in ((k_cache, k_scale), (v_cache, v_scale)):
        if (scale is not None) != (quantised and cache is not None):
            raise ValueError(f"{name}: a float8_e4m3fn cache, and no other, comes with its exponent bytes")
        if scale is not None and (scale.dtype != torch.uint8 or scale.shape != cache.shape[:3]):
            raise ValueError(f"{name}: exponent bytes {scale.dtype} {tuple(scale.shape)} for a cache of {tuple(cache.shape)}")
    _same_device(name, k_cache, v_cache, k_scale, v_scale)


def _check_table(name: str, table, sequences: int, k_cache) -> None:
    if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != sequences:
        raise ValueError(f"{name}: block table {table.dtype} {tuple(table.shape)} for {sequences} sequences (int32 [sequences, pages])")
    _same_device(name, k_cache, table)


def _check_write(k, v, k_cache, v_cache, slots, k_scale, v_scale) -> None:
    if (v is None) != (v_cache is None):
        raise ValueError("cache_write: values and their cache come together")
    _check_cache("cache_write", k_cache, v_cache, k_scale, v_scale)
    if slots.dim() != 1 or slots.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"cache_write: slots {slots.dtype} {tuple(slots.shape)}")
    for x, cache, scale in ((k, k_cache, k_scale), (v, v_cache, v_scale)):
        if x is None:
            continue
        for t in (cache, scale):
            if t is not None and t.numel() and not _nested(t):
                raise ValueError(f"cache_write: the rows of a cache are written once each, those of {tuple(t.shape)} with strides {t.stride()} overlap")
        if x.dim() != 3 or x.shape[0] != slots.shape[0] or x.shape[1:] != cache.shape[2:]:
            raise ValueError(f"cache_write: rows {tuple(x.shape)} and slots {tuple(slots.shape)} for a cache of {tuple(cache.shape)}")
        if x.dtype != cache.dtype and cache.dtype != torch.float8_e4m3fn:
            raise ValueError(f"cache_write: rows of {x.dtype} into a cache of {cache.dtype}")
    if v is not None and v.dtype != k.dtype:
        raise ValueError(f"cache_write: k {k.dtype}, v {v.dtype}")
    _same_device("cache_write", k, v, k_cache, slots)


def check_apart(a, b) -> None:
    """The keys' memory is not the values'.  That goes by addresses too, so every call looks; the kernels' wrapper asks only where the ranges meet."""
    if b is not None and torch._C._has_storage(a) and torch._C._has_storage(b) and _share_memory(a, b):
        raise ValueError(f"cache_write: keys {tuple(a.shape)} and values {tuple(b.shape)} share memory")


def cache_write(k, v, k_cache, v_cache, slots, k_scale=None, v_scale=None) -> None:
    """Writes the keys ``k`` [T, G, D] and values ``v`` [T, G, Dv] of new tokens into a paged cache ``k_cache`` [pages, page, G, D], ``v_cache``
    [pages, page, G, Dv], in place.  ``slots`` [T] (int32 or int64): page number times page size plus place in the page; a negative slot is
    left out (padding), of equal slots the last token's row stays.  ``v`` and ``v_cache`` may both be None (values that are columns of the
    key rows).  ``k`` and ``v`` may lie in the cache itself (tokens moved inside it): they count as they were before the call.

    A ``float8_e4m3fn`` cache holds each row divided by a power of two, whose exponent byte (127 + exponent, as in MXFP8) goes to ``k_scale``,
    ``v_scale`` (uint8 [pages, page, G]): the smallest with which the row's largest finite magnitude is at most 448; values that are not
    finite become NaN.  A 16-bit cache holds the rows as they are.  Values only: no gradient passes through a cache.  A slot behind the
    cache's end is skipped and reported by ``ops.cuda.check_errors``.  Caches whose rows overlap one another, or the other cache's, are refused."""
    layout = layout_of("cache_write", k, v, k_cache, v_cache, slots, k_scale, v_scale)
    if layout not in _CHECKED:
        _check_write(k, v, k_cache, v_cache, slots, k_scale, v_scale)
        _checked(layout)
    if k_cache.requires_grad or (v_cache is not None and v_cache.requires_grad):
        raise ValueError("cache_write: a cache has no gradient")
    fn = _cuda("cache_write", k)
    if fn is not None:
        if fn(k, v, k_cache, v_cache, slots, k_scale, v_scale, layout):
            return
        _miss("cache_write(shape/dtype)", k)
    check_apart(k_cache, v_cache)
    check_apart(k_scale, v_scale)
    with torch.no_grad():
        ref.cache_write(k, v, k_cache, v_cache, slots, k_scale, v_scale)


def cache_read(k_cache, v_cache, block_table, cu_seqlens, total: int, k_scale=None, v_scale=None, dtype=None):
    """Reads the first tokens of each sequence back out of a paged cache into packed rows: ``(k [total, G, D], v [total, G, Dv])``.  Sequence
    ``s`` gives its tokens ``0 .. cu_seqlens[s + 1] - cu_seqlens[s] - 1`` to the rows from ``cu_seqlens[s]`` on (int32 [n + 1], from 0),
    token ``p`` from place ``p % page`` of page ``block_table[s, p // page]`` (int32 [n, columns]); rows behind the last sequence are zeros.
    ``v_cache`` may be None (then so is the second result).  ``dtype``: type of the rows (bf16 by default out of an E4M3 cache, whose
    rows are multiplied by their powers of two; a 16-bit cache keeps its own).  Pages outside the cache give rows of zeros; they, and ends
    that do not rise from 0 to at most ``total``, are reported by ``ops.cuda.check_errors``."""
    layout = layout_of("cache_read", k_cache, v_cache, block_table, cu_seqlens, k_scale, v_scale)
    if layout not in _CHECKED:
        _check_cache("cache_read", k_cache, v_cache, k_scale, v_scale)
        _sequence_ends("cache_read", cu_seqlens, k_cache)
        _check_table("cache_read", block_table, cu_seqlens.numel() - 1, k_cache)
        _checked(layout)
    total = operator.index(total)              # a number: plans are kept by it
    if total < 0:
        raise ValueError(f"cache_read: {total} rows")
    if dtype is None:
        dtype = torch.bfloat16 if k_cache.dtype == torch.float8_e4m3fn else k_cache.dtype
    elif k_cache.dtype != torch.float8_e4m3fn and dtype != k_cache.dtype:
        raise ValueError(f"cache_read: a cache of {k_cache.dtype} read as {dtype}")
    fn = _cuda("cache_read", k_cache)
    if fn is not None:
        out = fn(k_cache, v_cache, block_table, cu_seqlens, total, k_scale, v_scale, dtype, (layout, total, dtype))
        if out is not None:
            return out
        _miss("cache_read(shape/dtype)", k_cache)
    return ref.cache_read(k_cache, v_cache, block_table, cu_seqlens, total, k_scale, v_scale, dtype)


def _check_paged(q, k_cache, v_cache, block_table, seq_lens, k_scale, v_scale) -> None:
    _check_cache("paged_attention", k_cache, v_cache, k_scale, v_scale)
    if v_cache is None or q.dim() != 3 or q.shape[2] != k_cache.shape[3]:
        raise ValueError(f"paged_attention: q {tuple(q.shape)} over caches {tuple(k_cache.shape)}, {None if v_cache is None else tuple(v_cache.shape)}")
    if k_cache.shape[2] == 0 or q.shape[1] % k_cache.shape[2]:
        raise ValueError(f"paged_attention: {q.shape[1]} query heads over {k_cache.shape[2]} key heads")
    _check_table("paged_attention", block_table, q.shape[0], k_cache)
    if seq_lens.dtype != torch.int32 or seq_lens.shape != q.shape[:1]:
        raise ValueError(f"paged_attention: lengths {seq_lens.dtype} {tuple(seq_lens.shape)} for {q.shape[0]} sequences (int32)")
    _same_device("paged_attention", q, k_cache, seq_lens)


def paged_attention(q, k_cache, v_cache, block_table, seq_lens, scale: float, k_scale=None, v_scale=None):
    """Attention of one new token per sequence over a paged cache: ``q`` [n, H, D], caches as in :func:`cache_write`, ``block_table`` int32
    [n, columns], ``seq_lens`` int32 [n] (tokens in the cache, the new one's own row among them once it is written); result [n, H, Dv].
    ``H`` is a multiple of the cache's heads ``G``; ``v_cache`` may be a view of the key rows.  A sequence of no tokens gives zeros.  What the
    pages hold behind a sequence's length is not read.

    bf16 and fp16 queries with a cache of the same type or of E4M3, widths that are multiples of 8 (E4M3: 16) up to 128 and up to 128 heads a
    group run on the kernels; anything else, and calls that need a gradient, run the definition, ``reference.paged_attention``.
    Lengths outside the table and pages outside the cache are left out and reported by ``ops.cuda.check_errors``."""
    layout = layout_of("paged_attention", q, k_cache, v_cache, block_table, seq_lens, k_scale, v_scale)
    if layout not in _CHECKED:
        _check_paged(q, k_cache, v_cache, block_table, seq_lens, k_scale, v_scale)
        _checked(layout)
    fn = _cuda("paged_attention", q)
    if fn is not None:
        o = fn(q, k_cache, v_cache, block_table, seq_lens, scale, k_scale, v_scale, layout)
        if o is not None:
            return o
        _miss("paged_attention(shape/dtype)", q)
    return ref.paged_attention(q, k_cache, v_cache, block_table, seq_lens, scale, k_scale, v_scale)


def embedding(ids, weight):
    """Row gather ``weight[ids]``; on the GPU the backward adds the gradient rows into the weight's gradient buffer with
    vector atomics instead of building a dense [vocab, hidden] gradient."""
    fn = _cuda("embedding", weight)
    if fn is not None:
        y = fn(ids, weight)
        if y is not None:
            return y
    return F.embedding(ids, weight)


def causal_conv1d_silu(x, weight, bias=None):
    """``silu(depthwise causal conv1d over the sequence)`` on a channels-last tensor: x [B, S, C], weight [C, k] (or the
    [C, 1, k] parameter of ``nn.Conv1d(groups=C)``), bias [C].  Output [B, S, C]."""
    if weight.dim() == 3:
        weight = weight.squeeze(1)
    fn = _cuda("causal_conv1d_silu", x)
    if fn is not None:
        y = fn(x, weight, bias)
        if y is not None:
            return y
    return ref.causal_conv1d_silu(x, weight, bias)


# ---- loss --------------------------------------------------------------------

def linear_cross_entropy(hidden, weight, labels, ignore_index: int = -100, reduction: str = "none"):
    fn = _cuda("linear_cross_entropy", hidden)
    if fn is not None:
        return fn(hidden, weight, labels, ignore_index, reduction)
    return ref.linear_cross_entropy(hidden, weight, labels, ignore_index, reduction)


def linear_cross_entropy_weighted(hidden, weight, labels, row_weights, ignore_index: int = -100):
    """Returns ``(sum_t row_weights[t] * CE_t, per-token CE)``; the second output carries no
    gradient.  This is the form the model uses: main and MTP heads are one call whose row
    weights hold mask / token-count / depth scaling."""
    fn = _cuda("linear_cross_entropy_weighted", hidden)
    if fn is not None:
        out = fn(hidden, weight, labels, row_weights, ignore_index)
        if out is not None:
            return out
        _miss("linear_cross_entropy(shape)", hidden)
    per_tok = ref.linear_cross_entropy(hidden, weight, labels, ignore_index, "none")
    return (per_tok * row_weights.to(per_tok.dtype)).sum(), per_tok.detach()


# ---- MoE ---------------------------------------------------------------------

def router_topk(logits, topk, score_function="sigmoid", expert_bias=None, norm_topk_prob=True):
    fn = _cuda("router_topk", logits)
    if fn is not None:
        out = fn(logits, topk, score_function, expert_bias, norm_topk_prob)
        if out is not None:
            return out
        _miss("router_topk(shape)", logits)
    return ref.router_topk(logits, topk, score_function, expert_bias, norm_topk_prob)
