"""The operators around a dense block on the GPU: calls that reach them in less usual ways."""
import pytest
import torch
from torch.autograd import forward_ad

from cppmega_b200.ops import functional as F_
from cppmega_b200.ops import reference as ref

pytestmark = pytest.mark.gpu

EPS = 1e-5


def _randn(*shape, dtype=torch.bfloat16, std=1.0, mean=0.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 7919 * sum(shape))
    return torch.empty(shape, device="cuda").normal_(mean, std, generator=g).to(dtype)


def _norm_calls():
    f32 = torch.float32
    x, z, w = _randn(6, 64, dtype=f32), _randn(6, 64, dtype=f32, seed=1), _randn(64, dtype=f32, mean=1.0, std=0.1, seed=2)
    return {"rmsnorm_gated": (F_.rmsnorm_gated, ref.rmsnorm_gated, (x, w, z)),
            "residual_rmsnorm": (lambda *a: F_.residual_rmsnorm(*a)[0], lambda *a: ref.residual_rmsnorm(*a)[0], (x, z, w, w, w))}


@pytest.mark.parametrize("name", ["rmsnorm_gated", "residual_rmsnorm"])
def test_norms_carry_tangents_and_transforms(name):
    """Forward mode, ``vmap`` and ``torch.func.grad`` give what the definition gives (it is what runs)."""
    call, plain, args = _norm_calls()[name]
    tangents = tuple(torch.full_like(t, 0.5) for t in args)
    with forward_ad.dual_level():
        got, want = (forward_ad.unpack_dual(f(*[forward_ad.make_dual(t, d) for t, d in zip(args, tangents)])).tangent for f in (call, plain))
    assert torch.equal(got, want) and got.abs().max() > 0
    for t in (torch.func.jvp(call, args, tangents)[1],):
        assert torch.equal(t, want)
    many = args[0].expand(3, 6, 64)
    assert torch.equal(torch.func.vmap(lambda t: call(t, *args[1:]))(many), torch.func.vmap(lambda t: plain(t, *args[1:]))(many))
    assert torch.equal(*(torch.func.grad(lambda t: f(t, *args[1:]).sum())(args[0]) for f in (call, plain)))


def test_gated_mlp_refuses_tangents():
    """The products have no forward-mode derivative, so that a call with tangents raises instead of losing them."""
    x, w1, w2 = _randn(6, 64), _randn(48, 64), _randn(64, 24)
    with forward_ad.dual_level():
        for i in range(3):
            args = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate((x, w1, w2))]
            with pytest.raises(RuntimeError):
                F_.gated_mlp(*args)


@pytest.mark.parametrize("before", [True, False])
def test_gated_norm_takes_a_batch_of_upstream_gradients(before):
    """Each gradient of a batch is the one that the definition gives alone: the same fp32 expressions over another batch of rows."""
    x, w, z = (t.requires_grad_() for t in _norm_calls()["rmsnorm_gated"][2])
    many = _randn(3, 6, 64, dtype=torch.float32, seed=4)
    got = torch.autograd.grad(F_.rmsnorm_gated(x, w, z, EPS, 16, before), [x, w, z], many, is_grads_batched=True)
    y = ref.rmsnorm_gated(x, w, z, EPS, 16, before)
    for i, dy in enumerate(many):
        for g, t in zip(got, torch.autograd.grad(y, [x, w, z], dy, retain_graph=True)):
            assert (g[i] - t).abs().max() <= 64 * 2 ** -24 * t.abs().max()


@pytest.mark.parametrize("form", ["apart", "wider", "offset"])
@pytest.mark.parametrize("name", ["gated_mlp", "residual_rmsnorm", "rmsnorm_gated"])
def test_saved_tensors_given_back_in_another_form(name, form):
    """Hooks that return the saved values every second element of a buffer, in fp32, or off the 16-byte grid."""
    x, z, w = _randn(40, 64).requires_grad_(), _randn(40, 64, seed=1).requires_grad_(), _randn(64, mean=1.0, std=0.1, seed=2).requires_grad_()
    w1, w2 = _randn(144, 64, std=0.1, seed=3).requires_grad_(), _randn(64, 72, std=0.1, seed=4).requires_grad_()
    call, leaves = {"gated_mlp": (lambda: F_.gated_mlp(x, w1, w2), [x, w1, w2]),
                    "residual_rmsnorm": (lambda: F_.residual_rmsnorm(x, z, w, w, w, 0.5)[0], [x, z, w]),
                    "rmsnorm_gated": (lambda: F_.rmsnorm_gated(x, w, z, EPS, 16, False), [x, w, z])}[name]
    dy = _randn(40, 64, std=0.1, seed=5)
    want = torch.autograd.grad(call(), leaves, dy)

    def pack(t):
        if form == "apart":
            return t.new_empty(*t.shape, 2)[..., 0].copy_(t.detach())
        if form == "wider":
            return t.detach().float() if t.dtype == torch.bfloat16 else t.detach()
        return t.new_empty(t.numel() + 1)[1:].view(t.shape).copy_(t.detach())

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        y = call()
    for a, b in zip(torch.autograd.grad(y, leaves, dy), want):
        if form == "offset" and name != "gated_mlp":      # rows off the grid are summed in another order: one step of bf16, and fp32 sums
            assert ((a.double() - b.double()).abs() <= 2 * 2 ** -8 * b.double().abs() + 2 ** -14 * b.double().abs().max()).all()
        else:
            assert torch.equal(a, b)


@pytest.mark.parametrize("T,H,F,Ho", [(4, 16, 0, 16), (4, 16, 24, 0), (0, 16, 24, 16), (4, 0, 24, 16), (300, 64, 0, 64)])
def test_gated_mlp_of_nothing(T, H, F, Ho):
    """A width or a number of tokens of zero: sums over nothing are zero, and so are their gradients."""
    leaves = [_randn(*s).requires_grad_() for s in ((T, H), (2 * F, H), (Ho, F))]
    junk = [torch.full((1 << 16,), float("nan"), device="cuda") for _ in range(8)]      # what unwritten results would hold
    del junk
    y = F_.gated_mlp(*leaves)
    grads = torch.autograd.grad(y, leaves, torch.ones_like(y))
    with torch.no_grad():
        again = F_.gated_mlp(*leaves)
    assert y.shape == (T, Ho) and all(g.shape == t.shape for g, t in zip(grads, leaves))
    assert all((t == 0).all() for t in (y, again, *grads))


def test_residual_rmsnorm_with_a_learnt_scale():
    """The gradient of a scale given as a tensor: sum of dh y over everything, 4096 fp32 products and their sum."""
    y, x, w = _randn(64, 64, dtype=torch.float32), _randn(64, 64, dtype=torch.float32, seed=1), _randn(64, dtype=torch.float32, mean=1.0, std=0.1)
    scale = torch.tensor(0.5, device="cuda", requires_grad=True)
    dh = _randn(64, 64, dtype=torch.float32, seed=2)
    _, h = F_.residual_rmsnorm(y, x, w, scale=scale)
    (got,) = torch.autograd.grad(h, scale, dh)
    terms = dh.double() * y.double()
    assert abs(got.double() - terms.sum()) <= (64 + 4096) * 2 ** -24 * terms.abs().sum()


@pytest.mark.parametrize("before", [True, False])
def test_gated_norm_in_fp32_far_out_gates(before):
    """The gate's relative error does not grow with its distance from zero.  In units of 2^-24: the exponential 4 (2 ulp), 1 + e and the
    quotient 1 each, the reciprocal root 5, products 1 each.  Rows of +-1 (with the gate first +-1 / silu(z)) have a mean square of one,
    and 16 terms are summed without error (15 roundings with the gate first)."""
    U = 2.0 ** -24
    z = torch.linspace(-80, 2 if before else -1, 4096 * 16, device="cuda").reshape(4096, 16)
    zd = z.double()
    q = torch.sigmoid(zd)
    a, slope = zd * q, q + zd * q * (1 - q)
    sign = torch.where(torch.arange(16, device="cuda") % 2 == 0, 1.0, -1.0).expand(4096, 16)
    x = (sign if before else sign / a.float()).contiguous().requires_grad_()
    z, w = z.requires_grad_(), torch.ones(16, device="cuda")
    dy = _randn(*z.shape, dtype=torch.float32, std=0.1, seed=3)
    y = F_.rmsnorm_gated(x, w, z, EPS, None, before)
    (dz,) = torch.autograd.grad(y, z, dy)
    xd, e_slope = x.detach().double(), U * (7 * q + 16 * (zd * q).abs())
    v = xd if before else xd * a
    r = (v.square().mean(1, keepdim=True) + EPS).rsqrt()
    if before:
        want, bound = xd * r * a, 16 * U
        wz = dy.double() * xd * r * slope
        ez = 10 * U * wz.abs() + (dy.double() * xd * r).abs() * e_slope
    else:
        hat, g = v * r, dy.double()
        want, bound = hat, 40 * U
        m = (g * hat).mean(1, keepdim=True)
        du = r * (g - hat * m)
        wz = du * xd * slope
        e_du = 60 * U * r * (g.abs() + 2 * hat.abs() * (g * hat).abs().mean(1, keepdim=True))
        ez = 10 * U * wz.abs() + (du * xd).abs() * e_slope + e_du * (xd * slope).abs()
    assert ((y.detach().double() - want).abs() <= bound * want.abs()).all()
    assert ((dz.double() - wz).abs() <= ez).all()


@pytest.mark.parametrize("T", [20, 300])
@pytest.mark.parametrize("ffn", [72, 200])
@pytest.mark.parametrize("name,weight", [("relu", -3e38), ("relu", -1e12), ("silu", -1e30), ("silu", -1e12), ("gelu_tanh", -1e30)])
def test_gated_mlp_closed_gate_leaves_its_neighbours_alone(T, ffn, name, weight):
    """A gate far out on the negative side (the first overflows to -inf) is closed: results and gradients are those with a gate that is
    closed at a moderate value, in its own column and in the 31 others that share its power of two."""
    x, w1, w2 = _randn(T, 64), _randn(2 * ffn, 64, std=0.125, seed=1), _randn(64, ffn, std=0.1, seed=2)
    x[:, 0] = 4.0
    cols = [3, 40, ffn - 1]
    w1[:ffn, 0] = 0.0
    dy = _randn(T, 64, std=0.1, seed=3)
    res = []
    for closed in (weight, -256.0):                 # 4 * -256 and at most 64 * 4 * 0.6 beside it
        w1[cols, 0] = closed
        leaves = [t.detach().clone().requires_grad_() for t in (x, w1, w2)]
        y = F_.gated_mlp(*leaves, name)
        res.append([y.detach(), *torch.autograd.grad(y, leaves, dy)])
    (y, dx, dw1, dw2), (y2, *want) = res
    assert torch.equal(y, y2) and torch.equal(dw1, want[1]) and torch.equal(dw2, want[2])
    assert torch.equal(dx, want[0]) and want[1].abs().max() > 0


@pytest.mark.parametrize("name", ["silu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("T", [20, 90])
def test_gated_mlp_gradients_of_a_nan_row(T, name):
    """A token that is NaN has gradients that are, and leaves the others' as they are."""
    x, w1, w2 = _randn(T, 64), _randn(144, 64, std=0.125, seed=1), _randn(64, 72, std=0.1, seed=2)
    dy, grads = _randn(T, 64, std=0.1, seed=3), []
    for bad in (False, True):
        leaf = x.clone()
        if bad:
            leaf[4, 7] = float("nan")
        leaf.requires_grad_()
        grads.append(torch.autograd.grad(F_.gated_mlp(leaf, w1, w2, name), leaf, dy)[0])
    rest = torch.arange(T, device="cuda") != 4
    assert torch.isnan(grads[1][4].float()).all()   # dg = dh u slope with u NaN, whatever the slope
    assert torch.equal(grads[0][rest], grads[1][rest])


# ---- products whose first rows are done whole and whose last rows are split --------------------------------------------

MIXED = {False: [(4408, 3080, 2056), (4112, 1032, 8200), (9480, 264, 2056), (1448, 3080, 8200)],
         True: [(4112, 1032, 4104), (1448, 3080, 4104), (9736, 264, 4104), (4408, 1032, 4104)]}


@pytest.mark.parametrize("a_mn", [False, True])
@pytest.mark.parametrize("b_mn,M,N,K", [(b, *s) for b, shapes in MIXED.items() for s in shapes])
@pytest.mark.parametrize("fp32,accumulate,pad", [(False, False, 0), (True, True, 4), (False, True, 3), (True, False, 5)])
def test_gemm_split_after_whole_rows(a_mn, b_mn, M, N, K, fp32, accumulate, pad):
    """Both parts of a mixed plan, every row of the result, in rows of any pitch.  One rounding to the result's type; K products and their
    sums in fp32, in any order."""
    import ctypes
    from cppmega_b200.ops import cuda as cu
    L = cu.lib()
    plan = (ctypes.c_int * 4)()
    floats = L.cm_gemm_split_plan(torch.cuda.get_device_properties(0).multi_processor_count, M, N, K, int(b_mn), plan)
    assert 0 < plan[0] < M and plan[2] > 1 and floats > 0
    a, b = _randn(*((K, M) if a_mn else (M, K))), _randn(*((K, N) if b_mn else (N, K)), seed=1)
    c0 = _randn(M, N + pad, dtype=torch.float32 if fp32 else torch.bfloat16, seed=2)
    c, ws = c0.clone(), torch.full((floats + 64,), float("nan"), device="cuda")
    assert L.cm_gemm_split(a.data_ptr(), b.data_ptr(), c.data_ptr(), M, N, K, a.stride(0), b.stride(0), N + pad, int(a_mn), int(b_mn), int(fp32),
                           int(accumulate), ws.data_ptr(), cu.err_word().data_ptr(), cu.stream_ptr()) == 0
    torch.cuda.synchronize()
    cu.check_errors()
    x, y = (a.t() if a_mn else a).double(), (b if b_mn else b.t()).double()
    before = c0[:, :N].double()
    want = x @ y + (before if accumulate else 0)
    size = x.abs() @ y.abs() + (before.abs() if accumulate else 0)
    assert ((c[:, :N].double() - want).abs() <= (0 if fp32 else 2 ** -8) * want.abs() + (64 + K) * 2 ** -24 * size).all()
    assert torch.equal(c[:, N:], c0[:, N:]) and ws[floats:].isnan().all() and not ws[:floats].isnan().any()


# ---- many rows a block --------------------------------------------------------------------------------------------------

def _against_chunks(call, rows, grads, shared):
    """One call over all rows against calls over 100 rows each, where no block has a second one.  What belongs to a row has the same bits;
    the gradients of what the rows share are the same fp32 terms in another order: at most 64 + rows / 100 additions on either side."""
    def run(cut):
        outs, leaves = call(cut)
        return [t.detach() for t in outs], torch.autograd.grad(outs, leaves, [g[cut] for g in grads])

    outs, back = run(slice(None))
    parts = [run(slice(i, i + 100)) for i in range(0, rows, 100)]
    for k, t in enumerate(outs):
        assert torch.equal(t, torch.cat([p[0][k] for p in parts]))
    for k, t in enumerate(back):
        if k not in shared:
            assert torch.equal(t, torch.cat([p[1][k] for p in parts])), k
        elif t.dtype == torch.float32:
            total, size = sum(p[1][k].double() for p in parts), shared[k]
            assert ((t.double() - total).abs() <= 2 * (64 + rows / 100) * 2 ** -24 * size).all(), k
    return outs, back


MANY = [(12000, 816), (8000, 333), (40000, 64), (20001, 16), (3001, 4096), (2500, 8192), (6000, 2048)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("before", [True, False])
@pytest.mark.parametrize("rows,group,groups", [(r, w, 1) for r, w in MANY] + [(9000, 1024, 8), (5000, 333, 3)])
def test_gated_norm_with_many_rows_a_block(dtype, before, rows, group, groups):
    import test_gpu_block as tb
    D = group * groups
    x, w, z = _randn(rows, D, dtype=dtype), _randn(D, dtype=dtype, mean=1.0, std=0.1, seed=1).requires_grad_(), _randn(rows, D, dtype=dtype, std=2.0, seed=2)
    dy = _randn(rows, D, dtype=dtype, std=0.1, seed=3)

    def call(cut):
        ins = [x[cut].detach().requires_grad_(), w, z[cut].detach().requires_grad_()]
        return [F_.rmsnorm_gated(*ins, EPS, group, before)], ins

    xd, zd = x.double(), z.double()
    a = zd * torch.sigmoid(zd)
    v = (xd if before else xd * a).view(rows, groups, group)
    hat = (v * (v.square().mean(-1, keepdim=True) + EPS).rsqrt()).view(rows, D)
    terms = (dy.double() * hat * (a if before else 1)).abs().sum(0)
    (y,), (dx, dw, dz) = _against_chunks(call, rows, [dy], {1: 1.01 * terms})
    tb._check_gated(x, w, z, group, before, y, dict(x=dx, w=dw, z=dz), dy)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("post,gate,scale", [(False, "none", 1.0), (False, "none", 0.22), (True, "channel", 0.5), (True, "token", -0.5)])
@pytest.mark.parametrize("rows,width", MANY)
def test_residual_rmsnorm_with_many_rows_a_block(dtype, post, gate, scale, rows, width):
    import test_gpu_block as tb
    ins = tb._residual_inputs((rows,), width, dtype, post, gate)
    names = list(ins)
    dn, dh = (_randn(rows, width, dtype=dtype, std=0.1, seed=s) for s in (11, 12))

    def call(cut):
        leaves = {k: (t[cut] if t.dim() > 1 else t).detach().requires_grad_() for k, t in ins.items()}
        n, h = F_.residual_rmsnorm(leaves["y"], leaves["residual"], leaves["weight"], leaves.get("post_weight"), leaves.get("gate"), scale, EPS)
        return [n, h], list(leaves.values())

    d = {k: t.double() for k, t in ins.items()}
    y, one = d["y"], torch.ones(width, dtype=torch.float64, device="cuda")
    hat = y * (y.square().mean(-1, keepdim=True) + EPS).rsqrt() if post else y
    gs = scale * d.get("gate", one)
    h = d["residual"] + gs * hat * d.get("post_weight", one)
    rho = (h.square().mean(-1, keepdim=True) + EPS).rsqrt()
    g = dn.double() * d["weight"]
    full = rho * (g - h * rho * (g * h * rho).mean(-1, keepdim=True)) + dh.double()
    sizes = {"weight": dn.double() * h * rho, "post_weight": gs * full * hat, "gate": scale * full * hat * d.get("post_weight", one)}
    shared = {names.index(k): 1.01 * sizes[k].abs().sum(0) for k in sizes if k in ins and ins[k].dim() == 1}
    (n, h), back = _against_chunks(call, rows, [dn, dh], shared)
    tb._check_residual(ins, scale, n, h, dict(zip(names, back)), dn, dh)


@pytest.mark.parametrize("name", ["relu", "gelu_tanh"])
def test_gated_mlp_activations_against_differences(name):
    """The gradient along a random direction against the formula's own difference; relu's gates stay on their side of the kink (+-8 with
    a spread of one, moved by an eighth), where the block is a quadratic and a central difference exact."""
    import test_gpu_block as tb
    x, w1, w2 = (t.clone() for t in tb._mlp_inputs((64,), 64, 64, 64))
    x[:, 0] = 4.0
    if name == "relu":
        w1[:64, 0] = 2.0 * torch.where(torch.arange(64, device="cuda") % 3 == 0, -1.0, 1.0).bfloat16()
    v, dy = _randn(64, 64, seed=5), _randn(64, 64, seed=6)
    v[:, 0] = 0
    leaf = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(F_.gated_mlp(leaf, w1, w2, name), leaf, dy)
    xd, vd, w1d, w2d, dyd = (t.double() for t in (x, v, w1, w2, dy))

    def exact(t):
        gu = t @ w1d.t()
        return ((tb._act(name, gu[:, :64])[0] * gu[:, 64:]) @ w2d.t() * dyd).sum()

    def slope(e):
        return (exact(xd + e * vd) - exact(xd - e * vd)) / (2 * e)

    want, half = slope(2.0 ** -3), slope(2.0 ** -4)
    g, up = (xd @ w1d.t()).split(64, 1)
    a, s, _ = tb._act(name, g)
    dh = dyd @ w2d
    size = torch.cat([dh * up * s, dh * a], 1).abs() @ w1d.abs()
    # bf16: the two gradients and the result (2^-8 each of what they are or are summed from); g and u with 11 bits: another 2^-8 at most
    assert abs((dx.double() * vd).sum() - want) <= 2 * abs(want - half) + 4 * 2 ** -8 * (size * vd.abs()).sum()
