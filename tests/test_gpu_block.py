"""The operators around a dense block on the GPU, against their formulas in 64 bits.

Every tolerance is a worst-case bound: u = eps / 2 of the type for each rounding to it, and C * 2^-24 of the sum of the magnitudes for
sums and products in fp32 (C counts the additions that one value passes through)."""
import math

import pytest
import torch

from cppmega_b200.ops import functional as F_

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24
EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _randn(*shape, dtype=torch.bfloat16, std=1.0, mean=0.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 7919 * sum(shape))
    return torch.empty(shape, device="cuda").normal_(mean, std, generator=g).to(dtype)


def _within(got, want, bound, what):
    """|got - want| <= bound element by element (with the smallest normal number of the type: results below it lose bits)."""
    assert torch.isfinite(got.double()).all(), what
    over = (got.double() - want).abs() - (bound + torch.finfo(got.dtype).tiny)
    assert over.max().item() <= 0, (what, over.max().item(), want.abs().max().item())


def _check_errors():
    from cppmega_b200.ops import cuda as cu
    torch.cuda.synchronize()
    cu.check_errors()


# ---- residual step ----------------------------------------------------------------------------------------------------

def _residual_inputs(rows, width, dtype, post, gate, seed=0):
    ins = dict(y=_randn(*rows, width, dtype=dtype, std=0.7, seed=seed), residual=_randn(*rows, width, dtype=dtype, std=2.0, seed=seed + 1),
               weight=_randn(width, dtype=dtype, mean=1.0, std=0.1, seed=seed + 2))
    if post:
        ins["post_weight"] = _randn(width, dtype=dtype, mean=1.0, std=0.1, seed=seed + 3)
    if gate != "none":
        ins["gate"] = _randn(*((width,) if gate == "channel" else (*rows, width)), dtype=dtype, mean=0.5, std=0.2, seed=seed + 4)
    return ins


def _check_residual(ins, scale, n, h, grads=None, dn=None, dh=None):
    """``grads``: name -> gradient, for upstream gradients ``dn`` / ``dh`` (None: zero)."""
    d = {k: t.detach().double().reshape(-1, t.shape[-1]) if t.dim() > 1 else t.detach().double() for k, t in ins.items()}
    W, dtype = n.shape[-1], n.dtype
    u = _u(dtype)
    C = (64 + W / 64) * E32                        # a row's sum: W / threads additions in a thread, then the team's tree
    y, w, post, gate = d["y"], d["weight"], d.get("post_weight"), d.get("gate")
    r = (y.square().mean(-1, keepdim=True) + EPS).rsqrt() if post is not None else torch.ones_like(y[:, :1])
    hat = y * r
    p = hat * post if post is not None else y
    gs = scale * (gate if gate is not None else torch.ones_like(w))
    want = d["residual"] + gs * p
    _within(h.detach().reshape(want.shape), want, u * want.abs() + C * (d["residual"].abs() + (gs * p).abs()), "h")
    hk = h.detach().double().reshape(want.shape)   # n and the gradients are those of the h that the stream holds
    rho = (hk.square().mean(-1, keepdim=True) + EPS).rsqrt()
    hh = hk * rho
    _within(n.detach().reshape(want.shape), hh * w, (u + C) * (hh * w).abs(), "n")
    if grads is None:
        return
    zero = torch.zeros_like(want)
    dn = zero if dn is None else dn.double().reshape(want.shape)
    dh = zero if dh is None else dh.double().reshape(want.shape)
    g = dn * w
    m1, m1a = (g * hh).mean(-1, keepdim=True), (g * hh).abs().mean(-1, keepdim=True)
    full = rho * (g - hh * m1) + dh
    e_full = C * (rho * (g.abs() + 2 * hh.abs() * m1a) + dh.abs())               # fp32 error of dh before its rounding
    out = {"residual": (full, u * full.abs() + e_full)}
    dp = gs * full
    e_dp = gs.abs() * e_full + C * dp.abs()
    R = want.shape[0]
    CR = (64 + R) * E32
    col = lambda t, e: (t.sum(0), u * t.sum(0).abs() + CR * t.abs().sum(0) + e.sum(0))  # noqa: E731
    out["weight"] = col(dn * hh, C * (dn * hh).abs())
    if post is None:
        out["y"] = (dp, u * dp.abs() + e_dp)
    else:
        a = gs * post
        q = dp * post
        m2 = (q * hat).mean(-1, keepdim=True)
        # the mean from the three sums: (S2 - rho m1 S3) / W, each in fp32
        m2a = ((a * hat) * (rho * g.abs() + dh.abs())).abs().mean(-1, keepdim=True) + rho * m1a * (a * hat * hh).abs().mean(-1, keepdim=True)
        dy = r * (q - hat * m2)
        out["y"] = (dy, u * dy.abs() + r * (e_dp * post.abs() + C * q.abs() + 4 * C * hat.abs() * m2a + C * (hat * m2).abs()))
        out["post_weight"] = col(dp * hat, e_dp * hat.abs() + C * (dp * hat).abs())
    if gate is not None:
        dg = scale * full * p
        e_dg = abs(scale) * e_full * p.abs() + C * dg.abs()
        out["gate"] = col(dg, e_dg) if gate.dim() == 1 else (dg, u * dg.abs() + e_dg)
    for name, got in grads.items():
        ref, bound = out[name]
        _within(got.reshape(ref.shape), ref, bound, "d" + name)


def _run_residual(ins, scale, dn, dh):
    leaves = {k: t.requires_grad_() for k, t in ins.items()}
    n, h = F_.residual_rmsnorm(leaves["y"], leaves["residual"], leaves["weight"], leaves.get("post_weight"), leaves.get("gate"), scale, EPS)
    outs = [(o, g) for o, g in ((n, dn), (h, dh)) if g is not None]
    grads = torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [g for _, g in outs], allow_unused=True)
    return n, h, dict(zip(leaves, grads))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,width", [((1,), 8), ((3,), 1), ((2, 5), 40), ((33,), 64), ((5,), 200), ((130,), 256), ((7,), 333), ((64,), 512),
                                        ((9,), 1001), ((19,), 1024), ((301,), 2048), ((4,), 3584), ((700,), 4096), ((3,), 8192), ((2,), 16384),
                                        ((2,), 12345)])
@pytest.mark.parametrize("post,gate,scale", [(False, "none", 1.0), (False, "none", 0.22), (True, "channel", 0.5), (True, "token", -0.5),
                                             (False, "token", 1.0), (True, "none", 1.0)])
def test_residual_rmsnorm(dtype, rows, width, post, gate, scale):
    dt = DTYPES[dtype]
    ins = _residual_inputs(rows, width, dt, post, gate)
    dn, dh = (_randn(*rows, width, dtype=dt, std=0.1, seed=s) for s in (11, 12))
    before = F_.launch_counts().get("residual_rmsnorm", 0)
    n, h, grads = _run_residual(ins, scale, dn, dh)
    assert F_.launch_counts()["residual_rmsnorm"] == before + 1
    _check_residual(ins, scale, n, h, grads, dn, dh)
    with torch.no_grad():                          # the call without gradients gives the same bits
        n2, h2 = F_.residual_rmsnorm(ins["y"], ins["residual"], ins["weight"], ins.get("post_weight"), ins.get("gate"), scale, EPS)
    assert torch.equal(n, n2) and torch.equal(h, h2)


def test_residual_rmsnorm_one_upstream_gradient():
    ins = _residual_inputs((37,), 136, torch.bfloat16, True, "channel")
    dn, dh = (_randn(37, 136, std=0.1, seed=s) for s in (1, 2))
    for a, b in ((dn, None), (None, dh)):
        n, h, grads = _run_residual({k: t.detach().clone() for k, t in ins.items()}, 0.5, a, b)
        _check_residual(ins, 0.5, n, h, grads, a, b)


def test_residual_rmsnorm_is_the_add_and_the_norm():
    """Without gate and post norm: the bits of the add, and the norm kernel's result to a step of the type (the two sum a row in
    different orders, so their fp32 values differ by a few 2^-24 and may lie on two sides of a rounding border: one step, 2 u)."""
    y, x, w = _randn(300, 4096), _randn(300, 4096, seed=3), _randn(4096, mean=1.0, std=0.1, seed=4)
    n, h = F_.residual_rmsnorm(y, x, w)
    assert torch.equal(h, x + y)
    norm = F_.rmsnorm(x + y, w, EPS).double()
    _within(n, norm, 2 * _u(n.dtype) * norm.abs(), "n")
    assert (n.double() == norm).double().mean() > 0.99


def test_residual_rmsnorm_reads_strided_rows():
    wide = _randn(50, 3 * 96 + 5)
    y, x = wide[:, 5:101], wide[:, 101:197]        # odd offset: no 16-byte rows
    even = _randn(2, 25, 400, seed=5)
    ins = _residual_inputs((50,), 96, torch.bfloat16, True, "channel")
    for a, b in ((y, x), (even[..., 96:192], even[..., 192:288]), (even.transpose(0, 1)[..., :96], even.transpose(0, 1)[..., 96:192])):
        cur = dict(ins, y=a.detach(), residual=b.detach())
        g = _randn(*a.shape, std=0.1, seed=9)
        n, h, grads = _run_residual(cur, 0.5, g, g)
        _check_residual(cur, 0.5, n, h, grads, g, g)


def test_residual_rmsnorm_broadcast_gradients():
    """The expanded gradient of a sum."""
    ins = _residual_inputs((21,), 72, torch.float32, True, "channel")
    leaves = {k: t.requires_grad_() for k, t in ins.items()}
    n, h = F_.residual_rmsnorm(leaves["y"], leaves["residual"], leaves["weight"], leaves["post_weight"], leaves["gate"], 0.5, EPS)
    grads = torch.autograd.grad(n.sum() + h.sum(), list(leaves.values()))
    one = torch.ones(21, 72, device="cuda")
    _check_residual(ins, 0.5, n, h, dict(zip(leaves, grads)), one, one)


def test_residual_rmsnorm_special_values():
    """Infinities and NaN stay in their row; a row of zeros has finite results."""
    ins = _residual_inputs((6,), 64, torch.bfloat16, True, "none")
    ins["y"][1, 3], ins["y"][2, 5] = float("inf"), float("nan")
    ins["y"][3], ins["residual"][3] = 0, 0
    g = _randn(6, 64, std=0.1, seed=4)
    n, h, grads = _run_residual(ins, 1.0, g, g)
    good = [0, 3, 4, 5]
    for t in (n, h, grads["y"], grads["residual"]):
        assert torch.isfinite(t[good].float()).all()
        assert torch.isnan(t[2].float()).any()


def test_residual_rmsnorm_same_bits_twice():
    ins = _residual_inputs((999,), 520, torch.bfloat16, True, "channel")
    g = _randn(999, 520, std=0.1, seed=4)
    a, b = (_run_residual({k: t.detach().clone() for k, t in ins.items()}, 0.5, g, g) for _ in range(2))
    assert all(torch.equal(a[2][k], b[2][k]) for k in a[2])


def test_residual_rmsnorm_same_tensor_as_both():
    """The block's output is the residual itself: the two gradients add up."""
    x = _randn(40, 128, dtype=torch.float32).requires_grad_()
    w = _randn(128, dtype=torch.float32, mean=1.0, std=0.1, seed=1)
    n, h = F_.residual_rmsnorm(x, x, w)
    g = _randn(40, 128, dtype=torch.float32, seed=2)
    (got,) = torch.autograd.grad(h, x, g)
    assert torch.equal(got, 2 * g)


# ---- gated norm -------------------------------------------------------------------------------------------------------

def _check_gated(x, w, z, group, before, y, grads=None, dy=None):
    shape, dtype = y.shape, y.dtype
    D = shape[-1]
    u = _u(dtype)
    C = (64 + group / 16) * E32
    x, w, dy = x.detach().double().reshape(-1, D), w.detach().double(), None if dy is None else dy.double().reshape(-1, D)
    split = lambda t: t.reshape(t.shape[0], -1, group)  # noqa: E731
    if z is None:
        a, slope, zz = torch.ones_like(x), torch.zeros_like(x), torch.zeros_like(x)
    else:
        zz = z.detach().double().reshape(-1, D)
        q = torch.sigmoid(zz)
        a, slope = zz * q, q * (1 + zz * (1 - q))
    ca = C * (1 + zz.abs())                        # the exponent's rounding: |z| 2^-24 of the sigmoid
    v = split(x if before else x * a)
    r = (v.square().mean(-1, keepdim=True) + EPS).rsqrt()
    hat = (v * r).reshape(x.shape)
    worst = split(ca).amax(-1, keepdim=True).expand(v.shape).reshape(x.shape)       # error of a group's norm
    want = hat * w * a if before else hat * w
    _within(y.detach().reshape(want.shape), want, (u + 2 * ca + 2 * worst) * want.abs(), "y")
    if grads is None:
        return
    dn = dy * a if before else dy
    g = dn * w
    mean = lambda t: split(t).mean(-1, keepdim=True).expand(v.shape).reshape(x.shape)  # noqa: E731
    rr = r.expand(v.shape).reshape(x.shape)
    m, ma = mean(g * hat), mean((g * hat).abs())
    du = rr * (g - hat * m)
    e_du = rr * ((2 * ca + 2 * worst) * g.abs() + 6 * worst * hat.abs() * ma)
    out = {}
    slope_err = ca * (q + (zz * q * (1 - q)).abs()) if z is not None else torch.zeros_like(x)
    if before:
        out["x"] = (du, u * du.abs() + e_du)
        dz = dy * hat * w * slope
        out["z"] = (dz, u * dz.abs() + 4 * worst * dz.abs() + (dy * hat * w).abs() * 4 * slope_err)
    else:
        dx = du * a
        out["x"] = (dx, u * dx.abs() + e_du * a.abs() + 2 * ca * dx.abs())
        dz = du * x * slope
        out["z"] = (dz, u * dz.abs() + e_du * (x * slope).abs() + 4 * (du * x).abs() * slope_err + C * dz.abs())
    t = dn * hat
    CR = (64 + t.shape[0]) * E32
    out["w"] = (t.sum(0), u * t.sum(0).abs() + (CR + 4 * worst) .mul(t.abs()).sum(0))
    for name, got in grads.items():
        ref, bound = out[name]
        _within(got.reshape(ref.shape), ref, bound, "d" + name)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,group,groups", [((1,), 8, 1), ((5,), 1, 3), ((2, 9), 24, 2), ((33,), 64, 5), ((17,), 136, 1), ((130,), 256, 3),
                                               ((40,), 333, 2), ((21,), 512, 1), ((600,), 816, 1), ((60,), 1024, 8), ((6,), 2049, 1),
                                               ((31,), 4096, 2), ((3,), 8192, 1), ((2,), 16384, 1)])
@pytest.mark.parametrize("before", [True, False])
def test_rmsnorm_gated(dtype, rows, group, groups, before):
    dt, D = DTYPES[dtype], group * groups
    x, w = _randn(*rows, D, dtype=dt).requires_grad_(), _randn(D, dtype=dt, mean=1.0, std=0.1, seed=1).requires_grad_()
    z = _randn(*rows, 2 * D, dtype=dt, std=2.0, seed=2)[..., D:].requires_grad_()          # a column slice, read in place
    dy = _randn(*rows, D, dtype=dt, std=0.1, seed=3)
    before_count = F_.launch_counts().get("rmsnorm_gated", 0)
    y = F_.rmsnorm_gated(x, w, z, EPS, group, before)
    assert F_.launch_counts()["rmsnorm_gated"] == before_count + 1
    dx, dw, dz = torch.autograd.grad(y, [x, w, z], dy)
    _check_gated(x, w, z, group, before, y, dict(x=dx, w=dw, z=dz), dy)
    with torch.no_grad():
        assert torch.equal(y, F_.rmsnorm_gated(x, w, z, EPS, group, before))


@pytest.mark.parametrize("before", [True, False])
def test_rmsnorm_gated_without_gate(before):
    x, w = _randn(70, 256).requires_grad_(), _randn(256, mean=1.0, std=0.1, seed=1).requires_grad_()
    dy = _randn(70, 256, std=0.1, seed=3)
    y = F_.rmsnorm_gated(x, w, None, EPS, 64, before)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    _check_gated(x, w, None, 64, before, y, dict(x=dx, w=dw), dy)


def test_rmsnorm_gated_large_gates():
    """Gates far out on both sides: silu is 0 or the gate itself, no overflow on the way."""
    z = torch.tensor([-3e38, -1e4, -200.0, -90.0, 90.0, 200.0, 1e4, 3.0], device="cuda").repeat(4, 2).bfloat16().requires_grad_()
    x, w = _randn(4, 16).requires_grad_(), torch.ones(16, device="cuda", dtype=torch.bfloat16)
    y = F_.rmsnorm_gated(x, w, z, EPS, None, True)
    dx, dz = torch.autograd.grad(y, [x, z], torch.ones_like(y))
    assert all(torch.isfinite(t.float()).all() for t in (y, dx, dz))
    assert (y[:, [0, 1, 2]] == 0).all() and (dz[:, [0, 1, 2]] == 0).all()


# ---- dense products with shared last tiles --------------------------------------------------------------------------

@pytest.mark.parametrize("a_mn,b_mn", [(False, False), (False, True), (True, True), (True, False)])
@pytest.mark.parametrize("M,N,K", [(512, 1024, 4096), (304, 136, 1032), (2064, 520, 8200), (5000, 1032, 4104), (256, 256, 16384), (40, 8, 2000)])
@pytest.mark.parametrize("fp32,accumulate", [(False, False), (True, True), (False, True)])
def test_gemm_split(a_mn, b_mn, M, N, K, fp32, accumulate):
    import ctypes
    from cppmega_b200.ops import cuda as cu
    L = cu.lib()
    a, b = _randn(*((K, M) if a_mn else (M, K))), _randn(*((K, N) if b_mn else (N, K)), seed=1)
    c0 = _randn(M, N, dtype=torch.float32 if fp32 else torch.bfloat16, seed=2)
    plan = (ctypes.c_int * 4)()
    floats = L.cm_gemm_split_plan(torch.cuda.get_device_properties(0).multi_processor_count, M, N, K, int(b_mn), plan)
    ws = torch.full((max(floats, 1),), float("nan"), dtype=torch.float32, device="cuda")
    c = c0.clone()
    rc = L.cm_gemm_split(a.data_ptr(), b.data_ptr(), c.data_ptr(), M, N, K, a.stride(0), b.stride(0), N, int(a_mn), int(b_mn), int(fp32),
                         int(accumulate), ws.data_ptr(), cu.err_word().data_ptr(), cu.stream_ptr())
    assert rc == 0
    _check_errors()
    x, y = (a.t() if a_mn else a).double(), (b if b_mn else b.t()).double()
    want = x @ y + (c0.double() if accumulate else 0)
    size = x.abs() @ y.abs() + c0.double().abs()
    _within(c, want, (0 if fp32 else 2 ** -8) * want.abs() + (64 + K) * E32 * size, "C")


# ---- gated feed-forward -----------------------------------------------------------------------------------------------

@torch.enable_grad()
def _act(name, g):
    """act, slope and the largest |g d slope / dg|."""
    t = g.detach().clone().requires_grad_()
    f = {"silu": lambda v: v * torch.sigmoid(v), "relu": lambda v: v.clamp_min(0),
         "gelu_tanh": lambda v: v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))) / 2}[name]
    a = f(t)
    (slope,) = torch.autograd.grad(a.sum(), t)
    if name == "relu":
        return a.detach(), slope, 0.0
    s = torch.linspace(-20, 20, 40001, dtype=torch.float64, device=g.device, requires_grad=True)
    (d1,) = torch.autograd.grad(f(s).sum(), s, create_graph=True)
    (d2,) = torch.autograd.grad(d1.sum(), s)
    return a.detach(), slope, (s * d2).abs().max().item()


def _check_mlp(x, w1, w2, name, y, grads=None, dy=None, h_rounded=True):
    u = 2.0 ** -8
    H, F = w1.shape[1], w2.shape[1]
    x, w1, w2 = x.detach().double().reshape(-1, H), w1.detach().double(), w2.detach().double()
    T, Ho = x.shape[0], w2.shape[0]
    acc = lambda k: (64 + k) * E32  # noqa: E731     # a product of k terms in fp32
    gu = x @ w1.t()
    e_gu = acc(H) * (x.abs() @ w1.abs().t())
    g, up, e_g, e_u = gu[:, :F], gu[:, F:], e_gu[:, :F], e_gu[:, F:]
    a, slope, curve = _act(name, g)
    e_a = 1.2 * e_g + 64 * E32 * (a.abs() + g.abs())          # |slope| < 1.2 everywhere
    h = a * up
    e_h = e_a * up.abs() + a.abs() * e_u + (u if h_rounded else u * u) * h.abs()       # h in one bf16, or in two
    want = h @ w2.t()
    size = h.abs() @ w2.abs().t()
    _within(y.detach().reshape(want.shape), want, u * want.abs() + acc(F) * size + 1.02 * (e_h @ w2.abs().t()), "y")
    if grads is None:
        return
    dy = dy.detach().double().reshape(T, Ho)
    dh = dy @ w2
    e_dh = acc(Ho) * (dy.abs() @ w2.abs())
    # g and u are kept with 11 bits under a power of two per row and 32 columns: half a step is 2^-11 of the value, or 2^-25 under the
    # power, which is 2^-39 of the group's largest (bounded here by the row's); |slope(g') - slope(g)| <= curve |g' - g| / |g|
    k = 2.0 ** -11
    tiny = lambda t: 2.0 ** -39 * t.abs().amax(1, keepdim=True)  # noqa: E731
    e_s = (curve * k + 64 * E32) * torch.ones_like(g) + 1.2 * (e_g + tiny(g))
    if name == "relu":
        e_s = (g.abs() <= e_g + tiny(g)).double()               # a gate whose sign the fp32 sum does not settle
    dg, du = dh * up * slope, dh * a
    e_up = k * up.abs() + e_u + tiny(up)
    e_dg = e_dh * (up * slope).abs() + dh.abs() * (e_up * slope.abs() + (up.abs() + e_up) * e_s) + u * dg.abs()
    e_du = e_dh * a.abs() + dh.abs() * (1.2 * (k * g.abs() + e_g + tiny(g)) + 64 * E32 * (a.abs() + g.abs())) + u * du.abs()
    dgu, e = torch.cat([dg, du], 1), torch.cat([e_dg, e_du], 1)
    out = {"x": (dgu @ w1, acc(2 * F) * (dgu.abs() @ w1.abs()) + 1.02 * (e @ w1.abs())),
           "w1": (dgu.t() @ x, acc(T) * (dgu.abs().t() @ x.abs()) + 1.02 * (e.t() @ x.abs())),
           "w2": (dy.t() @ h, acc(T) * (dy.abs().t() @ h.abs()) + 1.02 * (dy.abs().t() @ e_h))}
    for n, got in grads.items():
        ref, bound = out[n]
        _within(got.reshape(ref.shape), ref, bound + u * ref.abs(), "d" + n)


def _mlp_inputs(lead, H, F, Ho, seed=0):
    return (_randn(*lead, H, seed=seed), _randn(2 * F, H, std=H ** -0.5, seed=seed + 1), _randn(Ho, F, std=F ** -0.5, seed=seed + 2))


@pytest.mark.parametrize("name", ["silu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("lead,H,F,Ho", [((1,), 8, 8, 8), ((2, 3), 64, 72, 64), ((16,), 520, 264, 40), ((33,), 256, 512, 256), ((129,), 264, 200, 264),
                                         ((300,), 72, 1032, 136), ((2, 200), 1024, 2048, 1024), ((1000,), 200, 136, 328)])
def test_gated_mlp(name, lead, H, F, Ho):
    x, w1, w2 = (t.requires_grad_() for t in _mlp_inputs(lead, H, F, Ho))
    dy = _randn(*lead, Ho, std=0.1, seed=9)
    before = F_.launch_counts().get("gated_mlp", 0)
    y = F_.gated_mlp(x, w1, w2, name)
    assert F_.launch_counts()["gated_mlp"] == before + 1 and y.shape == (*lead, Ho)
    dx, dw1, dw2 = torch.autograd.grad(y, [x, w1, w2], dy)
    _check_errors()
    _check_mlp(x, w1, w2, name, y, dict(x=dx, w1=dw1, w2=dw2), dy)


# More tiles than CTA pairs, so that a pair takes several, on both sides of the width at which the backward changes how it reads g and u.
@pytest.mark.parametrize("name", ["silu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("T,H,F,Ho", [(2100, 40, 2344, 136), (2100, 40, 2344, 2560), (2100, 40, 2344, 2568), (5000, 264, 1000, 72), (200, 16, 40, 4104)])
def test_gated_mlp_several_tiles_a_pair(name, T, H, F, Ho):
    test_gated_mlp(name, (T,), H, F, Ho)


@pytest.mark.parametrize("T", [1, 2, 3, 7, 8, 9, 15, 16, 17, 24, 31, 32, 33, 48, 63, 64, 65, 100, 128, 200, 256, 257])
@pytest.mark.parametrize("H,F,Ho", [(1024, 2048, 1024), (520, 1000, 248), (24, 40, 16)])
def test_gated_mlp_without_gradients(T, H, F, Ho):
    x, w1, w2 = _mlp_inputs((T,), H, F, Ho, seed=T)
    with torch.no_grad():
        for name in ("silu", "gelu_tanh", "relu"):
            y = F_.gated_mlp(x, w1, w2, name)
            _check_errors()
            _check_mlp(x, w1, w2, name, y, h_rounded=T > 64)


def test_gated_mlp_parts_of_the_gradient():
    args = _mlp_inputs((70,), 128, 136, 128)
    dy = _randn(70, 128, std=0.1, seed=9)
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1)):
        leaves = [t.detach().clone().requires_grad_(bool(n)) for t, n in zip(args, need)]
        y = F_.gated_mlp(*leaves)
        names = [k for k, n in zip(("x", "w1", "w2"), need) if n]
        grads = torch.autograd.grad(y, [t for t in leaves if t.requires_grad], dy)
        _check_mlp(*leaves, "silu", y, dict(zip(names, grads)), dy)


def test_gated_mlp_strided_input_and_gradient():
    wide = _randn(90, 400)
    _, w1, w2 = _mlp_inputs((90,), 128, 136, 128)
    for x in (wide[:, 8:136], wide[:, 3:131], wide[::2, 16:144], wide.t()[:128].t()):
        x = x.detach().requires_grad_()
        y = F_.gated_mlp(x, w1, w2)
        dy = _randn(y.shape[0], 256, std=0.1, seed=9)[:, 64:192]
        (dx,) = torch.autograd.grad(y, [x], dy)
        _check_mlp(x, w1, w2, "silu", y, dict(x=dx), dy)
    y = F_.gated_mlp(wide[:, 8:136].detach().requires_grad_(), w1, w2)
    y.sum().backward()                              # an expanded gradient


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_gated_mlp_adds_into_main_grad(kind):
    x, w1, w2 = _mlp_inputs((150,), 128, 136, 128)
    leaves = [torch.nn.Parameter(w) for w in (w1, w2)]
    for p in leaves:
        p.main_grad = torch.zeros(p.shape, dtype=kind, device="cuda")
        p.fuse_wgrad_accumulation = True
    dy = _randn(150, 128, std=0.1, seed=9)
    F_.gated_mlp(x, *leaves).backward(dy)
    assert all(p.grad_added_to_main_grad for p in leaves)
    once = [p.main_grad.clone() for p in leaves]
    y = F_.gated_mlp(x, *leaves)
    _check_mlp(x, w1, w2, "silu", y, dict(w1=once[0], w2=once[1]), dy)
    y.backward(dy)
    for p, o in zip(leaves, once):                  # the same products added: exactly twice in fp32, one more rounding in bf16
        _within(p.main_grad, 2 * o.double(), (2 ** -8 if kind == torch.bfloat16 else 2 * E32) * (2 * o.double().abs()) + 1e-6, "main_grad")


@pytest.mark.parametrize("T", [40, 300])
def test_gated_mlp_gradients_of_far_apart_magnitudes(T):
    """Columns of w1 scaled by up to 2^+-30 and rows of x by 2^+-20: the kept values have one power of two per row and 32 columns."""
    x, w1, w2 = _mlp_inputs((T,), 64, 136, 64)
    g = torch.Generator(device="cuda").manual_seed(5)
    x = x * torch.exp2(torch.randint(-20, 21, (T, 1), device="cuda", generator=g).float()).bfloat16()
    rows = torch.exp2(torch.randint(-30, 31, (272, 1), device="cuda", generator=g).float())
    rows[:136].clamp_(max=2.0 ** -22)               # gates in the range where the activation bends
    w1 = (w1.float() * rows).bfloat16()
    leaves = [t.requires_grad_() for t in (x, w1, w2)]
    dy = _randn(T, 64, std=0.1, seed=9)
    for name in ("silu", "gelu_tanh"):
        y = F_.gated_mlp(*leaves, name)
        grads = torch.autograd.grad(y, leaves, dy)
        _check_mlp(*leaves, name, y, dict(zip(("x", "w1", "w2"), grads)), dy)


@pytest.mark.parametrize("name", ["silu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("T", [20, 90])
def test_gated_mlp_nan_stays_in_its_row(T, name):
    x, w1, w2 = _mlp_inputs((T,), 64, 72, 64)
    for grad in (False, True):
        xx = x.clone()
        xx[4, 7] = float("nan")
        y = F_.gated_mlp(xx.requires_grad_(grad), w1, w2, name).detach()
        assert torch.isnan(y[4].float()).all()
        keep = [i for i in range(T) if i != 4]
        assert torch.isfinite(y[keep].float()).all()


@pytest.mark.parametrize("name", ["silu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("T", [20, 90])
def test_gated_mlp_far_out(T, name):
    """Gates of 1e3 to 1e18 on both sides: the activation is 0 or the gate, its slope 0 or 1, and nothing overflows on the way."""
    x = torch.ones(T, 8, device="cuda", dtype=torch.bfloat16).requires_grad_()
    size = torch.tensor([1e3, 1e6, 1e10, 1e14, 1e18, 30.0, 200.0, 1e5], device="cuda")
    w1 = torch.zeros(32, 8, device="cuda")
    w1[:8, 0], w1[8:16, 0] = size, -size
    w1[16:, 0] = 1.0
    w1, w2 = w1.bfloat16(), torch.full((8, 16), 2.0 ** -70, device="cuda", dtype=torch.bfloat16)
    y = F_.gated_mlp(x, w1, w2, name)
    (dx,) = torch.autograd.grad(y, x, torch.full_like(y, 2.0 ** 70))
    kept = w1[:8, 0].double()
    # y is the sum of the positive gates; dx[0] is 8 times that sum twice over: once through the slopes, once through act(g)
    total = kept.sum() * 2.0 ** -70
    assert ((y.double() - total).abs() <= 3 * 2 ** -8 * total).all()
    want = 8 * 2 * kept.sum()
    assert ((dx[:, 0].double() - want).abs() <= 5 * 2 ** -8 * want).all() and torch.isfinite(dx.float()).all()


def test_gated_mlp_against_differences():
    """The gradient along a random direction against the forward's own difference, relu away from its kink and silu."""
    x, w1, w2 = _mlp_inputs((64,), 64, 64, 64)
    v = _randn(64, 64, std=1.0, seed=5)
    dy = _randn(64, 64, std=1.0, seed=6)
    leaf = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(F_.gated_mlp(leaf, w1, w2), leaf, dy)
    e = 2.0 ** -3
    up, down = (x.double() + s * e * v.double() for s in (1, -1))

    def exact(t):
        gu = t @ w1.double().t()
        return ((gu[:, :64] * torch.sigmoid(gu[:, :64]) * gu[:, 64:]) @ w2.double().t() * dy.double()).sum()

    want = (exact(up) - exact(down)) / (2 * e)
    got = (dx.double() * v.double()).sum()
    # central difference: third derivative along v times e^2 / 6 (measured from a half step); gradient: four roundings of 2^-8
    half = (exact(x.double() + e / 2 * v.double()) - exact(x.double() - e / 2 * v.double())) / e
    assert abs(got - want) <= 2 * abs(want - half) + 4 * 2 ** -8 * (dx.double().abs() * v.double().abs()).sum()


# ---- together, on streams, in graphs ----------------------------------------------------------------------------------

def _step(x, y, p):
    """residual step -> feed-forward -> residual step -> gated norm, as a layer runs them."""
    n, h = F_.residual_rmsnorm(y, x, p["w"], p["post"], p["gate"], 0.5)
    m = F_.gated_mlp(n, p["w1"], p["w2"])
    n2, h2 = F_.residual_rmsnorm(m, h, p["w"])
    return F_.rmsnorm_gated(n2, p["w"], h2, EPS, 64, True), h2


def _step_params(H=256, F=264):
    p = dict(w=_randn(H, mean=1.0, std=0.1), post=_randn(H, mean=1.0, std=0.1, seed=1), gate=_randn(H, mean=0.5, std=0.1, seed=2),
             w1=_randn(2 * F, H, std=H ** -0.5, seed=3), w2=_randn(H, F, std=F ** -0.5, seed=4))
    return {k: t.requires_grad_() for k, t in p.items()}


def test_block_together_matches_the_definitions():
    p = _step_params()
    x, y = (_randn(3, 50, 256, seed=s).requires_grad_() for s in (5, 6))
    g = _randn(3, 50, 256, std=0.1, seed=7)
    names = ("residual_rmsnorm", "gated_mlp", "rmsnorm_gated")
    res = []
    for own in (True, False):
        (F_.enable_cuda if own else F_.disable_cuda)(*names)
        try:
            o, h = _step(x, y, p)
            res.append([o, h, *torch.autograd.grad([o, h], [x, y, *p.values()], [g, g])])
        finally:
            F_.enable_cuda(*names)
    _check_errors()
    for a, b in zip(*res):                          # both round about eight times to bf16 on the longest path
        assert (a.double() - b.double()).norm() <= 8 * 2 ** -8 * b.double().norm()


def test_block_in_a_graph_and_on_two_streams():
    p = {k: t.detach() for k, t in _step_params().items()}
    x, y = (_randn(70, 256, seed=s) for s in (5, 6))
    with torch.no_grad():
        want = _step(x, y, p)
        graphs = []
        for _ in range(2):
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                _step(x, y, p)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = _step(x, y, p)
            graphs.append((graph, out))
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        for _ in range(3):                          # both graphs at the same time
            for s, (graph, _) in zip(streams, graphs):
                with torch.cuda.stream(s):
                    graph.replay()
        _check_errors()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
        x.copy_(_randn(70, 256, seed=50))           # other inputs through the same graph
        want = _step(x, y, p)
        graphs[0][0].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(graphs[0][1], want))


def test_block_backward_in_a_graph():
    """Forward and backward captured together replay with the eager bits."""
    p = {k: t.detach().requires_grad_() for k, t in _step_params().items()}
    x, y = (_randn(70, 256, seed=s).requires_grad_() for s in (5, 6))
    g = _randn(70, 256, std=0.1, seed=7)
    leaves = [x, y, *p.values()]

    def run():
        o, h = _step(x, y, p)
        return [o.detach(), h.detach(), *torch.autograd.grad([o, h], leaves, [g, g])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    graph.replay()
    _check_errors()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_residual_gradients_are_separate_tensors():
    """Without gate and scale one gradient serves both inputs: what accumulates in one must not show in the other."""
    y, x = (_randn(33, 64, dtype=torch.float32, seed=s).requires_grad_() for s in (1, 2))
    w = _randn(64, dtype=torch.float32, mean=1.0, std=0.1, seed=3)
    n, h = F_.residual_rmsnorm(y, x, w)
    (n.sum() + h.sum()).backward()
    assert torch.equal(y.grad, x.grad)
    before = x.grad.clone()
    y.grad.add_(1)
    assert torch.equal(x.grad, before)
    n, h = F_.residual_rmsnorm(y, x, w)
    (n.sum() + h.sum()).backward()
    assert torch.equal(x.grad, 2 * before) and torch.equal(y.grad, (before + 1) + before)


def _dense_mlp(hidden=256, ffn=520):
    from cppmega_b200.models.common import DenseMLP
    from cppmega_b200.parallel.state import single_process_context
    return DenseMLP(hidden, ffn, single_process_context(), std=hidden ** -0.5, out_std=ffn ** -0.5, dtype=torch.bfloat16, seed=3).cuda()


def test_dense_mlp_module():
    m = _dense_mlp()
    x, dy = _randn(2, 60, 256), _randn(2, 60, 256, std=0.1, seed=1)
    leaf = x.clone().requires_grad_()
    F_.reset_counters()
    y = m(leaf)
    y.backward(dy)
    assert F_.launch_counts() == {"gated_mlp": 1, "gated_mlp_bwd": 1} and not F_.fallback_counts()
    _check_mlp(x, m.linear_fc1.weight, m.linear_fc2.weight, "silu", y, dict(x=leaf.grad, w1=m.linear_fc1.weight.grad, w2=m.linear_fc2.weight.grad), dy)


def test_dense_mlp_module_captured():
    """The module as a captured callable (the ``mlp`` scope of the graph option): replays give the eager bits."""
    m = _dense_mlp()
    x, dy = _randn(90, 256).requires_grad_(), _randn(90, 256, std=0.1, seed=1)
    y = m(x)
    want = [y.detach().clone(), *torch.autograd.grad(y, [x, *m.parameters()], dy)]
    del y
    graphed = torch.cuda.make_graphed_callables(_dense_mlp(), (torch.randn_like(x).requires_grad_(),))
    for _ in range(2):
        y = graphed(x)
        got = [y.detach().clone(), *torch.autograd.grad(y, [x, *graphed.parameters()], dy)]
        _check_errors()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_fastmtp_block():
    """The shared block: attention, residual step, feed-forward - against the same block on its PyTorch definitions."""
    from cppmega_b200.models.fastmtp import SharedMTPBlock
    torch.manual_seed(0)
    b = SharedMTPBlock(256, 2, 512, torch.bfloat16).cuda()
    x, dy = _randn(2, 128, 256), _randn(2, 128, 256, std=0.1, seed=1)
    res = []
    for own in (True, False):
        names = ("residual_rmsnorm", "gated_mlp")
        (F_.enable_cuda if own else F_.disable_cuda)(*names)
        try:
            leaf = x.clone().requires_grad_()
            y = b(leaf)
            res.append([y.detach(), *torch.autograd.grad(y, [leaf, *b.parameters()], dy)])
        finally:
            F_.enable_cuda(*names)
    _check_errors()
    for p, q in zip(*res):                          # some ten roundings to bf16 on the longest path of either
        assert (p.double() - q.double()).norm() <= 10 * 2 ** -8 * q.double().norm()


def test_mixer_norm_reads_its_gate_in_place():
    """The gate of the M2RNN mixer is a column slice of the projection whose rows are not a multiple of 16 bytes apart from it."""
    from cppmega_b200.models.common import RMSNorm
    norm = RMSNorm(136, dtype=torch.bfloat16).cuda()
    proj = _randn(2, 30, 600).requires_grad_()
    y, dy = _randn(2, 30, 136, seed=2).requires_grad_(), _randn(2, 30, 136, std=0.1, seed=3)
    gate = proj[..., 451:587]
    F_.reset_counters()
    out = norm(y, gate=gate, norm_before_gate=False)
    dx, dp, dw = torch.autograd.grad(out, [y, proj, norm.weight], dy)
    assert set(F_.launch_counts()) == {"rmsnorm_gated", "rmsnorm_gated_bwd"} and not F_.fallback_counts()
    assert (dp[..., :451] == 0).all() and (dp[..., 587:] == 0).all()
    _check_gated(y, norm.weight, gate, 136, False, out, dict(x=dx, w=dw, z=dp[..., 451:587]), dy)


def test_block_calls_from_two_threads():
    """Two host threads, each on its own stream, get what one alone gets."""
    import threading
    p = {k: t.detach() for k, t in _step_params().items()}
    ins = [[_randn(40 + 30 * i, 256, seed=5 + i), _randn(40 + 30 * i, 256, seed=9 + i)] for i in range(2)]
    with torch.no_grad():
        want = [_step(*i, p) for i in ins]
    torch.cuda.synchronize()
    got, failed = [None, None], []

    def work(k):
        try:
            with torch.no_grad(), torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[k] = _step(*ins[k], p)
                torch.cuda.current_stream().synchronize()
        except Exception as e:                      # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    _check_errors()
    for a, b in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_rows_behind_the_last_one_are_left_alone():
    """Results that end inside a larger buffer: the feed-forward's products write whole tiles, clipped at their last row and column."""
    from cppmega_b200.ops import cuda as cu
    L, T, H, F = cu.lib(), 70, 64, 72
    x, w1, w2 = _mlp_inputs((T,), H, F, H)
    for tokens in (T, 9):                           # tiles, and the path for few tokens
        y = torch.full((tokens + 8, H), 7.0, dtype=torch.bfloat16, device="cuda")
        h = torch.full((tokens + 8, F), 7.0, dtype=torch.bfloat16, device="cuda")
        size = L.cm_gated_mlp_kept(tokens, F)
        kept = torch.full((size + 64,), 99, dtype=torch.uint8, device="cuda")
        floats = L.cm_gated_mlp_fwd_ws(tokens, H, F, H)
        ws = torch.full((floats + 64,), 5.0, device="cuda")
        assert L.cm_gated_mlp_fwd(x.data_ptr(), H, w1.data_ptr(), w2.data_ptr(), kept.data_ptr(), h.data_ptr(), y.data_ptr(), ws.data_ptr(), tokens,
                                  H, F, H, 0, cu.err_word().data_ptr(), cu.stream_ptr()) == 0
        _check_errors()
        assert (y[tokens:] == 7).all() and (h[tokens:] == 7).all() and (kept[size:] == 99).all() and (ws[floats:] == 5).all()
        _check_mlp(x[:tokens], w1, w2, "silu", y[:tokens])


def test_offsets_beyond_32_bits():
    """Tensors of more than 2^31 elements: their last rows are those of a small call on the same rows."""
    R, W, tail = 530000, 4096, 300
    y = torch.empty(R, W, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    w = _randn(W, mean=1.0, std=0.1)
    with torch.no_grad():
        n, h = F_.residual_rmsnorm(y, y, w, post_weight=w, gate=w)
        n1, h1 = F_.residual_rmsnorm(y[-tail:], y[-tail:], w, post_weight=w, gate=w)
        assert torch.equal(n[-tail:], n1) and torch.equal(h[-tail:], h1)
        del h
        g = F_.rmsnorm_gated(y, w, n, EPS, 512, False)
        assert torch.equal(g[-tail:], F_.rmsnorm_gated(y[-tail:], w, n[-tail:], EPS, 512, False))
    del g, n
    leaf = y.requires_grad_()
    grads = []
    for t in (leaf, leaf[-tail:]):
        out, h = F_.residual_rmsnorm(t, t, w)
        grads.append(torch.autograd.grad([out, h], leaf, [t.detach(), t.detach()])[0][-tail:].clone())
        del out, h
    assert torch.equal(*grads)
    del leaf, y
    T, H, F = 66000, 64, 16400                      # 2 T F kept values
    x, w1, w2 = _mlp_inputs((T,), H, F, H)
    dy = _randn(T, H, std=0.1, seed=9)
    out = []
    for k in (T, 512):
        leaf = x[-k:].detach().requires_grad_()
        res = F_.gated_mlp(leaf, w1, w2)
        out.append([res.detach()[-tail:], torch.autograd.grad(res, leaf, dy[-k:])[0][-tail:]])
        del res
    _check_errors()
    # the two calls may cut their reductions differently: one fp32 sum against another, rounded once (2 u for values at a border)
    for a, b in zip(*out):
        assert (a.double() - b.double()).abs().max() <= 2 * 2 ** -8 * b.double().abs().max()


def test_first_derivatives_only():
    """Gradients under ``create_graph`` are right; differentiating them again raises."""
    x = _randn(30, 64).requires_grad_()
    w1, w2 = _randn(144, 64, std=0.1, seed=1).requires_grad_(), _randn(64, 72, std=0.1, seed=2)
    w = _randn(64, mean=1.0, std=0.1, seed=3)
    for call in (lambda: F_.gated_mlp(x, w1, w2), lambda: F_.residual_rmsnorm(x, x, w)[0], lambda: F_.rmsnorm_gated(x, w, x)):
        (plain,) = torch.autograd.grad(call().sum(), x)
        (g,) = torch.autograd.grad(call().sum(), x, create_graph=True)
        assert torch.equal(plain, g)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), x)
