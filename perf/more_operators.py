"""Attention over packed sequences and over a paged key-value cache, whose speed is followed: whole prompts and documents of different
lengths in one buffer (with their gradients in training), the cache as it is written and read back, and one new token per sequence.

A case is one call, the way a program of this framework makes it.  Heads and widths are those of the presets in ``config/model.py`` (full: 32
heads of 64 + 64 with values of 64, quarter 28 heads, tiny 4 heads of 32 + 32), in their absorbed form (one key row of 64 + 64 for all heads), and
generic grouped heads of 64 and 128.  Lengths are drawn from the case's ``mix``, so that they belong to the case and not to the inputs.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}


def listed():
    return [
        # three short documents through the tiny model's attention: launches and host time
        _packed("packed_tiny", "129,64,7", 4, 4, 64, 64, "bf16", train=True),
        # documents packed into two rows of the full model's training batch: dense latent attention, 64 + 64 and 64
        _packed("packed_documents", "4096,1900,1031,640,300,128,64,32,1", 32, 32, 128, 64, "bf16", train=True),
        # a training batch of long and short documents with grouped heads: the largest
        _packed("packed_grouped", "6000,5000,3500,1883,1", 32, 8, 128, 128, "bf16", train=True),
        # prompts of a serving batch in fp16, 28 heads in groups of 7
        _packed("packed_prompts", "2047,1024,700,255,69", 28, 4, 128, 128, "fp16", train=False),
        # the next 512 tokens of four prompts whose beginnings lie in the cache already
        _packed("packed_continued", "512,512,512,512", 32, 8, 128, 128, "bf16", train=False, before="7680,3584,1001,0"),
        # one new token for each of 24 sequences: quantised, written, and their last page read back
        _cache("cache_step", tokens=24, sequences=24, kv_heads=8, dim=128, vdim=128, page=16, store="e4m3", dtype="bf16"),
        # a prompt batch quantised into the cache and read back for its continuation
        _cache("cache_prompt", tokens=16384, sequences=7, kv_heads=8, dim=128, vdim=128, page=64, store="e4m3", dtype="bf16"),
        # the same without quantisation, keys and values of the full model's dense attention, pages of an odd size
        _cache("cache_plain", tokens=4095, sequences=5, kv_heads=32, dim=128, vdim=64, page=48, store="bf16", dtype="bf16"),
        # one sequence of a chat: latency
        _decode("decode_one", 1, 1000, 1000, 32, 8, 128, 128, page=16, store="bf16", dtype="bf16"),
        # a serving batch, ragged lengths, quantised cache
        _decode("decode_batch", 64, 100, 16000, 32, 8, 128, 128, page=64, store="e4m3", dtype="bf16"),
        # the full model's latent attention in its absorbed form: 32 heads share one row of 64 + 64
        _decode("decode_latent", 48, 500, 8000, 32, 1, 128, 64, page=32, store="bf16", dtype="bf16"),
        # one very long sequence: all of the time is the cache, split over its length
        _decode("decode_long", 1, 131071, 131071, 64, 8, 128, 128, page=128, store="bf16", dtype="bf16"),
    ]


def _packed(name, lens, heads, kv_heads, dim, vdim, dtype, train, before=""):
    return dict(name=name, kind="packed", lens=lens, before=before, heads=heads, kv_heads=kv_heads, dim=dim, vdim=vdim, dtype=dtype, train=train)


def _cache(name, tokens, sequences, kv_heads, dim, vdim, page, store, dtype, mix=1):
    return dict(name=name, kind="cache", tokens=tokens, sequences=sequences, kv_heads=kv_heads, dim=dim, vdim=vdim, page=page, store=store,
                dtype=dtype, mix=mix)


def _decode(name, sequences, shortest, longest, heads, kv_heads, dim, vdim, page, store, dtype, mix=1):
    return dict(name=name, kind="decode", sequences=sequences, shortest=shortest, longest=longest, heads=heads, kv_heads=kv_heads, dim=dim,
                vdim=vdim, page=page, store=store, dtype=dtype, mix=mix)


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["packed", "packed", "packed", "cache", "decode", "decode"])
    dim, vdim = rng.choice([(128, 128), (128, 64), (64, 64), (128, 128), (96, 96), (80, 80)])
    if kind == "packed":
        train = rng.random() < 0.6
        lens = [_log(rng, 1, 4096) for _ in range(_log(rng, 1, 12))]
        before = "" if train or rng.random() < 0.5 else ",".join(str(rng.choice([0, _log(rng, 1, 6000)])) for _ in lens)
        kv_heads, group = rng.choice([(8, 4), (4, 7), (32, 1), (4, 4), (2, 8), (1, 16), (6, 3)])
        case = _packed("", ",".join(map(str, lens)), kv_heads * group, kv_heads, dim, vdim, rng.choice(["bf16", "bf16", "fp16"]), train, before)
    else:
        store, dtype = rng.choice([("e4m3", "bf16"), ("bf16", "bf16"), ("fp16", "fp16")])
        page, mix = rng.choice([16, 32, 48, 64, 128]), rng.randrange(1 << 20)
        if kind == "cache":
            sequences = _log(rng, 1, 64)
            tokens = max(sequences, _log(rng, 1, 16384))
            case = _cache("", tokens, sequences, rng.choice([1, 2, 4, 8]), dim, vdim, page, store, dtype, mix)
        else:
            longest = _log(rng, 1, 65536)
            sequences = _log(rng, 1, max(1, min(128, (1 << 19) // longest)))
            kv_heads, group = rng.choice([(8, 4), (8, 8), (4, 7), (8, 1), (2, 16), (1, 32)])
            case = _decode("", sequences, _log(rng, 1, longest), longest, kv_heads * group, kv_heads, dim, vdim, page, store, dtype, mix)
    del case["name"]
    return case


def _numbers(text):
    return [int(t) for t in text.split(",")] if text else []


def _lengths(case):
    """Tokens of each sequence of a cache or decode case."""
    rng = random.Random(case["mix"])
    if case["kind"] == "decode":
        return [_log(rng, case["shortest"], case["longest"]) for _ in range(case["sequences"] - 1)] + [case["longest"]]
    cuts = sorted(rng.sample(range(1, case["tokens"]), case["sequences"] - 1)) if case["sequences"] > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [case["tokens"]])]


def _ends(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


# ---- inputs --------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.empty(shape, device="cuda").normal_(0.0, std, generator=g).to(dtype)

    def ints(values, dtype=torch.int32):
        return torch.tensor(values, dtype=dtype, device="cuda")

    s = dict(case)
    K, D, V = case["kv_heads"], case["dim"], case["vdim"]
    s["scale"] = D ** -0.5
    if case["kind"] == "packed":
        lens, before = _numbers(case["lens"]), _numbers(case["before"])
        lens_k = [a + b for a, b in zip(lens, before)] if before else lens
        T, Tk = sum(lens), sum(lens_k)
        # a row of large keys now and then: attention that settles on few places
        s["q"], s["v"] = normal(T, case["heads"], D, std=1.5), normal(Tk, K, V)
        s["k"] = normal(Tk, K, D) * (1.0 + 2.0 * (torch.rand(Tk, 1, 1, device="cuda", generator=g) < 0.02)).to(dtype)
        s["ends"], s["ends_k"] = _ends(lens), _ends(lens_k)
        s["cu"], s["cu_k"] = ints(s["ends"]), ints(s["ends_k"]) if before else None
        if case["train"]:
            s["q"].requires_grad_(), s["k"].requires_grad_(), s["v"].requires_grad_()
            s["do"] = normal(T, case["heads"], V, std=0.1)
        return s
    lens, page = _lengths(case), case["page"]
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + 3                                    # some pages belong to nobody
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    at = ints(_ends(counts)[:-1])
    columns = torch.arange(max(counts), device="cuda")
    used = columns < ints(counts)[:, None]
    s["table"] = torch.where(used, order[(at[:, None] + columns).clamp(max=pages - 1).long()], torch.zeros_like(order[:1]))
    s["lens"] = ints(lens)
    stored = DTYPES[case["store"]]
    if case["store"] == "e4m3":
        if case["kind"] == "cache":
            s["kc"], s["vc"] = (torch.zeros(pages, page, K, n, dtype=torch.uint8, device="cuda").view(stored) for n in (D, V))
            s["ks"], s["vs"] = (torch.full((pages, page, K), 127, dtype=torch.uint8, device="cuda") for _ in range(2))
        else:
            # rows as a quantising writer leaves them: the largest magnitude between 224 and 448
            rows = [torch.empty(pages, page, K, n, device="cuda").normal_(0.0, 110.0, generator=g).clamp_(-448, 448) for n in (D, V)]
            s["kc"], s["vc"] = (t.to(stored) for t in rows)
            s["ks"], s["vs"] = (torch.randint(118, 122, (pages, page, K), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2))
    else:
        s["ks"] = s["vs"] = None
        if case["kind"] == "cache":
            s["kc"], s["vc"] = (torch.zeros(pages, page, K, n, dtype=stored, device="cuda") for n in (D, V))
        else:
            s["kc"], s["vc"] = normal(pages, page, K, D), normal(pages, page, K, V)
    if case["kind"] == "cache":
        T = case["tokens"]
        s["k"], s["v"] = normal(T, K, D), normal(T, K, V)
        s["ends"] = _ends(lens)
        s["cu"] = ints(s["ends"])
        seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), s["lens"].long())
        pos = torch.arange(T, device="cuda") - s["cu"].long()[seq]
        s["slots"] = s["table"][seq, pos // page].long() * page + pos % page
    else:
        s["q"] = normal(case["sequences"], case["heads"], D, std=1.5)
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(s):
    if own:
        return {"packed": _own_packed, "cache": _own_cache, "decode": _own_decode}[s["kind"]](s)
    return {"packed": _plain_packed, "cache": _plain_cache, "decode": _plain_decode}[s["kind"]](s)


def _own_packed(s):
    from cppmega_b200.ops import functional as F_
    if not s["train"]:
        with torch.no_grad():
            return {"o": F_.packed_attention(s["q"], s["k"], s["v"], s["cu"], s["scale"], s["cu_k"])}
    o = F_.packed_attention(s["q"], s["k"], s["v"], s["cu"], s["scale"])
    dq, dk, dv = torch.autograd.grad(o, [s["q"], s["k"], s["v"]], s["do"])
    return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}


def _own_cache(s):
    from cppmega_b200.ops import functional as F_
    F_.cache_write(s["k"], s["v"], s["kc"], s["vc"], s["slots"], s["ks"], s["vs"])
    k, v = F_.cache_read(s["kc"], s["vc"], s["table"], s["cu"], s["tokens"], s["ks"], s["vs"], dtype=s["k"].dtype)
    return {"k": k, "v": v}


def _own_decode(s):
    from cppmega_b200.ops import functional as F_
    return {"o": F_.paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["lens"], s["scale"], s["ks"], s["vs"])}


def _softmax(x):
    """Over the last axis; a row of nothing but -inf gives zeros."""
    m = x.detach().amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
    n = e.sum(-1, keepdim=True)
    return e / torch.where(n == 0, torch.ones_like(n), n)


def _plain_packed(s):
    dtype = s["q"].dtype
    q, k, v = (s[n].detach().float().requires_grad_(s["train"]) for n in "qkv")
    group = s["heads"] // s["kv_heads"]
    outs = []
    for a, b, c, d in zip(s["ends"], s["ends"][1:], s["ends_k"], s["ends_k"][1:]):
        heads = [t.transpose(0, 1) for t in (q[a:b], k[c:d].repeat_interleave(group, 1), v[c:d].repeat_interleave(group, 1))]
        scores = heads[0] @ heads[1].transpose(1, 2) * s["scale"]
        last = torch.arange(b - a, device="cuda")[:, None] + (d - c) - (b - a)
        seen = torch.arange(d - c, device="cuda")[None, :] <= last
        outs.append((_softmax(torch.where(seen, scores, -math.inf)) @ heads[2]).transpose(0, 1))
    o = torch.cat(outs)
    out = {"o": o.detach().to(dtype)}
    if s["train"]:
        for n, grad in zip("qkv", torch.autograd.grad(o, [q, k, v], s["do"].float())):
            out["d" + n] = grad.to(dtype)
    return out


def _power(e, bias=127, bits=23):
    """2^e of whole numbers in the range of normal values, without rounding."""
    return ((e.to(torch.int32 if bits == 23 else torch.int64) + bias) << bits).view(torch.float32 if bits == 23 else torch.float64)


def _plain_store(x, cache, scales, slots):
    rows = cache.view(-1, *cache.shape[2:])
    if scales is None:
        rows[slots] = x
        return
    x = x.float()
    m, e = torch.frexp(x.abs().amax(-1))
    e = torch.where(m == 0, torch.zeros_like(e), (e - 9 + (m > 0.875)).clamp(-126, 127))
    rows.view(torch.uint8)[slots] = (x * _power(-e)[..., None]).clamp(-448, 448).to(cache.dtype).view(torch.uint8)
    scales.view(-1, scales.shape[-1])[slots] = (e + 127).to(torch.uint8)


def _plain_load(cache, scales, pages):
    rows = cache.view(torch.uint8)[pages].view(cache.dtype).float()
    return rows if scales is None else rows * _power(scales[pages].int() - 127)[..., None]


def _plain_cache(s):
    _plain_store(s["k"], s["kc"], s["ks"], s["slots"])
    _plain_store(s["v"], s["vc"], s["vs"], s["slots"])
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(n.numel(), device="cuda"), n, output_size=s["tokens"])
    pos = torch.arange(s["tokens"], device="cuda") - s["cu"].long()[seq]
    page = s["kc"].shape[1]
    where = s["table"][seq, pos // page].long() * page + pos % page
    out = {}
    for name in "kv":
        cache, scales = s[name + "c"], s[name + "s"]
        flat = cache.view(torch.uint8).view(-1, cache.shape[2], cache.shape[3] * cache.element_size()).view(cache.dtype)
        out[name] = _plain_load(flat, None if scales is None else scales.view(-1, scales.shape[2]), where).to(s["k"].dtype)
    return out


def _plain_decode(s):
    B, K, page = s["sequences"], s["kv_heads"], s["page"]
    q = s["q"].float().view(B, K, -1, s["dim"])
    pages = s["table"].long()
    k, v = (_plain_load(s[n + "c"], s[n + "s"], pages).view(B, -1, K, s["vdim" if n == "v" else "dim"]).transpose(1, 2) for n in "kv")
    scores = q @ k.transpose(2, 3) * s["scale"]
    seen = torch.arange(pages.shape[1] * page, device="cuda") < s["lens"][:, None]
    o = _softmax(torch.where(seen[:, None, None], scores, -math.inf)) @ torch.where(seen[:, None, :, None], v, 0.0)
    return {"o": o.reshape(B, s["heads"], s["vdim"]).to(s["q"].dtype)}


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    H, K, D, V = case.get("heads", 0), case["kv_heads"], case["dim"], case["vdim"]
    if case["kind"] == "packed":
        lens, before = _numbers(case["lens"]), _numbers(case["before"])
        T, Tk = sum(lens), sum(lens) + sum(before)
        pairs = sum(n * (n + 1) // 2 + n * b for n, b in zip(lens, before or [0] * len(lens)))
        rows = T * H * (D + V) + Tk * K * (D + V)
        if case["train"]:        # q, k, v, do in; o, dq, dk, dv out; products q k', p v and do v', p' do, ds' q, ds k, q k' again
            return dict(bytes=2 * (2 * rows), flops=2.0 * pairs * H * (4 * D + 3 * V))
        return dict(bytes=2 * rows, flops=2.0 * pairs * H * (D + V))
    held = 1 if case["store"] == "e4m3" else 2
    row = K * (D + V)
    if case["kind"] == "cache":
        side = 4 * K if held == 1 else 0
        return dict(bytes=case["tokens"] * (2 * row + held * row + held * row + 2 * row + side + 8), flops=4.0 * case["tokens"] * row)
    n = sum(_lengths(case))
    return dict(bytes=n * (held * row + (2 * K if held == 1 else 0)) + 2 * case["sequences"] * H * (D + V), flops=2.0 * n * H * (D + V))


# ---- the same in 64 bits ----------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"packed": _exact_packed, "cache": _exact_cache, "decode": _exact_decode}[case["kind"]](s)


def _exact_packed(s):
    group, scale = s["heads"] // s["kv_heads"], s["scale"]
    q, k, v = (s[n].detach().double() for n in "qkv")
    o = torch.zeros(q.shape[0], s["heads"], s["vdim"], dtype=torch.float64, device="cuda")
    dq, dk, dv = (torch.zeros_like(t) for t in (q, k, v))
    for i in range(len(s["ends"]) - 1):
        rows, keys = slice(s["ends"][i], s["ends"][i + 1]), slice(s["ends_k"][i], s["ends_k"][i + 1])
        L, Lk = rows.stop - rows.start, keys.stop - keys.start
        hidden = torch.ones(L, Lk, dtype=torch.bool, device="cuda").triu(Lk - L + 1)
        for h in range(s["heads"]):
            qh, kh, vh = q[rows, h], k[keys, h // group], v[keys, h // group]
            p = torch.softmax((qh @ kh.T).mul_(scale).masked_fill_(hidden, -math.inf), dim=1)
            o[rows, h] = p @ vh
            if s["train"]:
                g = s["do"][rows, h].double()
                dp = g @ vh.T
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
                dq[rows, h] = ds @ kh
                dk[keys, h // group] += ds.T @ qh
                dv[keys, h // group] += p.T @ g
    return {"o": o, "dq": dq, "dk": dk, "dv": dv} if s["train"] else {"o": o}


def _exact_cache(s):
    if s["ks"] is None:
        return {"k": s["k"].double(), "v": s["v"].double()}
    out = {}
    for name in "kv":
        x = s[name].double()
        e = torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True) / 448))
        y = x * _power(-e, 1023, 52)
        step = _power(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3, 1023, 52)
        out[name] = torch.round(y / step) * step * _power(e, 1023, 52)
    return out


def _exact_decode(s):
    out = torch.zeros(s["sequences"], s["heads"], s["vdim"], dtype=torch.float64, device="cuda")
    group = s["heads"] // s["kv_heads"]
    for b, n in enumerate(s["lens"].tolist()):
        pages = s["table"][b, :-(-n // s["page"])].long()
        for h in range(s["kv_heads"]):
            k, v = (s[x + "c"].view(torch.uint8 if s["ks"] is not None else s["kc"].dtype)[pages, :, h].view(s["kc"].dtype).double() for x in "kv")
            if s["ks"] is not None:
                k, v = (t * _power(s[x + "s"][pages, :, h].long() - 127, 1023, 52)[..., None] for t, x in ((k, "k"), (v, "v")))
            k, v = k.reshape(-1, s["dim"])[:n], v.reshape(-1, s["vdim"])[:n]
            heads = slice(h * group, (h + 1) * group)
            out[b, heads] = torch.softmax(s["q"][b, heads].double() @ k.T * s["scale"], dim=1) @ v
    return {"o": out}
