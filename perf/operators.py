"""The operators around a dense block, whose speed is followed: the gated feed-forward block, the residual step with its norms, and the
gated norm of the mixers.

A case is one call, the way a program of this framework makes it: with its gradients (training) or without (evaluation and
generation).  Sizes are those of the presets in ``config/model.py`` (full 4096 / 21504, quarter 3584 / 18944, slice 1024 / 2048), the
shared expert (1024), the Mamba inner width (8192 in 8 groups) and the M2RNN width (816).
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # dense MLP of the smallest production-shaped model on a short sequence: launches and host time
        _mlp("mlp_small", 512, 1024, 2048, train=True),
        # dense MLP of the quarter model on a batch that fills no tile
        _mlp("mlp_ragged", 4095, 3584, 18944, train=True),
        # shared expert of the full model at the benchmark's micro-batch, 4 x 4096 tokens
        _mlp("mlp_shared_expert", 16384, 4096, 1024, train=True),
        # dense MLP of the full model at the same micro-batch: the largest
        _mlp("mlp_full", 16384, 4096, 21504, train=True),
        # one token through the dense MLP of the full model: all of the time is the weights
        _mlp("mlp_one_token", 1, 4096, 21504, train=False),
        # a batch of generating sequences through the dense MLP of the quarter model
        _mlp("mlp_few_tokens", 24, 3584, 18944, train=False),
        # residual add and the norm after it, one generated token a sequence
        _residual("residual_one_token", 1, 4096, "bf16", post=False, gate="none", scale=1.0, train=False),
        # the residual step of the full model's stack at the benchmark's micro-batch
        _residual("residual_add", 16384, 4096, "bf16", post=False, gate="none", scale=1.0, train=True),
        # norms on both sides of the block, a learnt gate per channel and a residual scale, quarter model, ragged batch
        _residual("residual_post_gate", 4095, 3584, "bf16", post=True, gate="channel", scale=0.5, train=True),
        # the same with a gate per token and channel in 32 bits, at a width that no vector divides
        _residual("residual_fp32_odd", 1023, 1001, "fp32", post=True, gate="token", scale=0.25, train=True),
        # output norm of the M2RNN mixer: gate first, read in place from the projection
        _gated("gated_m2rnn", 8192, 816, 816, "bf16", before=False, train=True),
        # grouped output norm of the Mamba mixer at the benchmark's micro-batch
        _gated("gated_mamba", 16384, 8192, 1024, "bf16", before=True, train=True),
    ]


def _mlp(name, tokens, hidden, ffn, train, activation="silu"):
    return dict(name=name, kind="mlp", tokens=tokens, hidden=hidden, ffn=ffn, activation=activation, train=train)


def _residual(name, rows, width, dtype, post, gate, scale, train):
    return dict(name=name, kind="residual", rows=rows, width=width, dtype=dtype, post=post, gate=gate, scale=scale, train=train)


def _gated(name, rows, width, group, dtype, before, train):
    return dict(name=name, kind="gated", rows=rows, width=width, group=group, dtype=dtype, before=before, train=train)


def _log(rng, lo, hi, step=1):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def draw(rng):
    kind = rng.choice(["mlp", "mlp", "mlp", "residual", "residual", "gated", "gated"])
    train = rng.random() < 0.65
    if kind == "mlp":
        tokens = _log(rng, 1, 16384) if train else _log(rng, 1, 2048)
        case = _mlp("", tokens, _log(rng, 256, 4096, 8), _log(rng, 512, 21504, 8), train, rng.choice(["silu", "silu", "gelu_tanh", "relu"]))
    elif kind == "residual":
        case = _residual("", _log(rng, 1, 16384), _log(rng, 64, 8192, rng.choice([1, 8])), rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                         rng.random() < 0.5, rng.choice(["none", "channel", "token"]), rng.choice([1.0, 0.5, 0.22]), train)
    else:
        group, groups = _log(rng, 16, 2048, rng.choice([1, 8])), rng.choice([1, 1, 2, 5, 8])
        case = _gated("", _log(rng, 1, 16384), groups * group, group, rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.random() < 0.5, train)
    del case["name"]
    return case


# ---- inputs --------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    train, dtype = case["train"], DTYPES[case.get("dtype", "bf16")]

    def normal(*shape, std=1.0, mean=0.0, grad=True):
        t = torch.empty(shape, device="cuda").normal_(mean, std, generator=g).to(dtype)
        return t.requires_grad_() if grad and train else t

    s = dict(case)
    if case["kind"] == "mlp":
        T, H, F = case["tokens"], case["hidden"], case["ffn"]
        s["ins"] = dict(x=normal(T, H), w1=normal(2 * F, H, std=H ** -0.5), w2=normal(H, F, std=F ** -0.5))
        s["grads"] = dict(y=normal(T, H, std=0.1, grad=False))
    elif case["kind"] == "residual":
        R, W = case["rows"], case["width"]
        s["ins"] = dict(y=normal(R, W, std=0.7), residual=normal(R, W, std=2.0), weight=normal(W, mean=1.0, std=0.1))
        if case["post"]:
            s["ins"]["post_weight"] = normal(W, mean=1.0, std=0.1)
        if case["gate"] != "none":
            s["ins"]["gate"] = normal(*((W,) if case["gate"] == "channel" else (R, W)), mean=0.5, std=0.2)
        s["grads"] = dict(n=normal(R, W, std=0.1, grad=False), h=normal(R, W, std=0.1, grad=False))
    else:
        R, W = case["rows"], case["width"]
        x, weight = normal(R, W), normal(W, mean=1.0, std=0.1)
        z = normal(R, 2 * W, grad=False)[:, W:]            # the gate columns of a wider projection, read where they are
        s["ins"] = dict(x=x, weight=weight, z=z.requires_grad_() if train else z)
        s["grads"] = dict(y=normal(R, W, std=0.1, grad=False))
    if not train:
        del s["grads"]
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(s):
    if not s["train"]:
        with torch.no_grad():
            return _forward(s, s["ins"]) if own else {n: t.to(s["ins"][_like(s)].dtype) for n, t in _plain(s, _wide(s["ins"])).items()}
    if own:
        ins = s["ins"]
        out = _forward(s, ins)
    else:
        ins = {n: t.requires_grad_() for n, t in _wide(s["ins"]).items()}
        out = _plain(s, ins)
    back = torch.autograd.grad([out[n] for n in s["grads"]], list(ins.values()), [g.to(out[n].dtype) for n, g in s["grads"].items()])
    dtype = s["ins"][_like(s)].dtype
    res = {n: t.detach().to(dtype) for n, t in out.items()}
    res.update({"d" + n: g.to(dtype) for n, g in zip(ins, back)})
    return res


def _like(s):
    return "y" if s["kind"] == "residual" else "x"


def _forward(s, i):
    """The framework's operators."""
    from cppmega_b200.ops import functional as F_
    if s["kind"] == "mlp":
        return {"y": F_.gated_mlp(i["x"], i["w1"], i["w2"], activation=s["activation"])}
    if s["kind"] == "residual":
        n, h = F_.residual_rmsnorm(i["y"], i["residual"], i["weight"], post_weight=i.get("post_weight"), gate=i.get("gate"),
                                   scale=s["scale"], eps=EPS)
        return {"n": n, "h": h}
    return {"y": F_.rmsnorm_gated(i["x"], i["weight"], i["z"], EPS, s["group"], s["before"])}


def _wide(ins):
    return {n: t.detach().float().contiguous() for n, t in ins.items()}


def _act(name, t):
    if name == "silu":
        return t / (1 + torch.exp(-t))
    if name == "relu":
        return t * (t > 0)
    return 0.5 * t * (1 + torch.tanh(math.sqrt(2 / math.pi) * (t + 0.044715 * t * t * t)))


def _rms(t):
    return t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS)


def _plain(s, i):
    """The same in elementary operations, in 32 bits."""
    if s["kind"] == "mlp":
        F = s["ffn"]
        gate_up = i["x"] @ i["w1"].t()
        return {"y": (_act(s["activation"], gate_up[:, :F]) * gate_up[:, F:]) @ i["w2"].t()}
    if s["kind"] == "residual":
        p = _rms(i["y"]) * i["post_weight"] if s["post"] else i["y"]
        if s["gate"] != "none":
            p = p * i["gate"]
        h = i["residual"] + s["scale"] * p
        return {"n": _rms(h) * i["weight"], "h": h}
    x, gate = i["x"], _act("silu", i["z"])
    if not s["before"]:
        x = x * gate
    y = _rms(x.view(x.shape[0], -1, s["group"])).view(x.shape) * i["weight"]
    return {"y": y * gate if s["before"] else y}


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    size = DTYPES[case.get("dtype", "bf16")].itemsize
    train = case["train"]
    if case["kind"] == "mlp":
        T, H, F = case["tokens"], case["hidden"], case["ffn"]
        return dict(bytes=size * ((4 if train else 2) * T * H + (2 if train else 1) * 3 * F * H), flops=(18.0 if train else 6.0) * T * H * F)
    n = case["rows"] * case["width"]
    if case["kind"] == "residual":
        gate = {"none": 0, "channel": 0, "token": 1}[case["gate"]]
        return dict(bytes=size * n * (8 + 2 * gate if train else 4 + gate), flops=(30.0 if train else 10.0) * n)
    return dict(bytes=size * n * (6 if train else 3), flops=(30.0 if train else 12.0) * n)


# ---- the same in 64 bits ----------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    i = {n: t.detach().double() for n, t in s["ins"].items()}
    d = {n: t.double() for n, t in s.get("grads", {}).items()}
    return {"mlp": _exact_mlp, "residual": _exact_residual, "gated": _exact_gated}[case["kind"]](case, i, d)


def _act_and_slope(name, t):
    if name == "relu":
        return t.clamp_min(0), (t > 0).double()
    if name == "silu":
        q = torch.sigmoid(t)
        return t * q, q + t * q * (1 - q)
    c = math.sqrt(2 / math.pi)
    th = torch.tanh(c * (t + 0.044715 * t ** 3))
    return t * (1 + th) / 2, (1 + th) / 2 + t * (1 - th ** 2) * c * (1 + 3 * 0.044715 * t ** 2) / 2


def _exact_mlp(case, i, d):
    x, w1, w2 = i["x"], i["w1"], i["w2"]
    wg, wu = w1[:case["ffn"]], w1[case["ffn"]:]
    up = x @ wu.t()
    a, slope = _act_and_slope(case["activation"], x @ wg.t())
    out = {"y": (a * up) @ w2.t()}
    if d:
        out["dw2"] = d["y"].t() @ (a * up)
        dh = d["y"] @ w2
        dup = dh * a
        dgate = dh.mul_(up).mul_(slope)
        out["dx"] = dgate @ wg + dup @ wu
        out["dw1"] = torch.cat([dgate.t() @ x, dup.t() @ x])
    return out


def _norm_back(dhat, hat, inv):
    return inv * (dhat - hat * (dhat * hat).mean(-1, keepdim=True))


def _exact_residual(case, i, d):
    y, w = i["y"], i["weight"]
    gate = case["scale"] * i["gate"] if "gate" in i else torch.full_like(w, case["scale"])
    inv_y = (y.square().mean(-1, keepdim=True) + EPS) ** -0.5
    hat = y * inv_y
    p = hat * i["post_weight"] if case["post"] else y
    h = i["residual"] + gate * p
    inv_h = (h.square().mean(-1, keepdim=True) + EPS) ** -0.5
    out = {"n": h * inv_h * w, "h": h}
    if d:
        dh = _norm_back(d["n"] * w, h * inv_h, inv_h) + d["h"]
        dp = gate * dh
        out["dweight"] = (d["n"] * h * inv_h).sum(0)
        out["dresidual"] = dh
        out["dy"] = _norm_back(dp * i["post_weight"], hat, inv_y) if case["post"] else dp
        if case["post"]:
            out["dpost_weight"] = (dp * hat).sum(0)
        if "gate" in i:
            dg = case["scale"] * dh * p
            out["dgate"] = dg.sum(0) if i["gate"].dim() == 1 else dg
    return out


def _exact_gated(case, i, d):
    split = lambda t: t.reshape(t.shape[0], -1, case["group"])  # noqa: E731
    x, w, z = i["x"], i["weight"], i["z"]
    a, slope = _act_and_slope("silu", z)
    u = split(x if case["before"] else x * a)
    inv = (u.square().mean(-1, keepdim=True) + EPS) ** -0.5
    hat = (u * inv).reshape(x.shape)
    out = {"y": hat * w * a if case["before"] else hat * w}
    if d:
        dn = d["y"] * a if case["before"] else d["y"]
        du = _norm_back(split(dn * w), split(hat), inv).reshape(x.shape)
        out["dweight"] = (dn * hat).sum(0)
        out["dx"] = du if case["before"] else du * a
        out["dz"] = d["y"] * hat * w * slope if case["before"] else du * x * slope
    return out
