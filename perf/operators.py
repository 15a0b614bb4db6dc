"""What the decode operators are measured on: one new token per request over a
paged key-value cache.  Four operators:

  plan  block tables, positions and cache slots from request lengths (b2q.kv_plan)
  rope  RMS norm of the query and key heads, rotation by position, keys and
        values to their cache slots (b2q.qk_norm_rope)
  attn  attention over the paged cache (b2q.attention_paged)
  vec   products with ggml Q4_0 / Q4_1 weights for few rows (b2q.mul_vec_q4)

`run` computes them in elementary torch operations in 32 bits where `own` is
false, and through the library where it is true.  `exact` is the definition in
64 bits, request by request and head by head.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = {"q4_0": 18, "q4_1": 20}      # bytes of a block of 32 weights
GOLDEN = 0.6180339887498949


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # a server's ordinary decode step: every request brings one token
        dict(name="plan-decode-33", op="plan", n=33, ctx_lo=0, ctx_hi=4099, new_lo=1, new_hi=1, page=16),
        # a large batch admitted at once: ragged prompts, some behind a cached prefix
        dict(name="plan-admit-509", op="plan", n=509, ctx_lo=0, ctx_hi=16384, new_lo=0, new_hi=1023, page=32),
        # five short prompts' tokens on the towers' head geometry (16 heads of 72), fp32 projections
        dict(name="rope-5x16x72", op="rope", T=5, hq=16, hk=16, d=72, rot=72, inter=False, dt="f32", cdt="f16",
             page=16, n_pos=4096, norm=True),
        # a decode step of a large batch, grouped heads
        dict(name="rope-256x32x128", op="rope", T=256, hq=32, hk=8, d=128, rot=128, inter=False, dt="bf16",
             cdt="bf16", page=16, n_pos=32768, norm=True),
        # a long prompt in one piece: half of each head rotated, neighbouring pairs, no norm
        dict(name="rope-20011x24x128", op="rope", T=20011, hq=24, hk=4, d=128, rot=64, inter=True, dt="f16",
             cdt="f16", page=64, n_pos=32768, norm=False),
        # one request on the towers' head geometry after an image's 729 patches and some text
        dict(name="attn-1x997x72", op="attn", n=1, lo=997, hi=997, hq=16, hk=16, d=72, dt="f16", out="f32", page=16,
             window=0, empty=0),
        # a decode batch of ragged lengths, a few rows of it idle
        dict(name="attn-61-ragged", op="attn", n=61, lo=17, hi=8191, hq=32, hk=8, d=128, dt="bf16", out="bf16",
             page=16, window=0, empty=3),
        # few requests with very long contexts: the split over the length carries it
        dict(name="attn-3x131071", op="attn", n=3, lo=131071, hi=131071, hq=40, hk=8, d=128, dt="f16", out="f32",
             page=64, window=0, empty=0),
        # one shared key head, wide heads, a sliding window
        dict(name="attn-256-window", op="attn", n=256, lo=1, hi=20000, hq=8, hk=1, d=256, dt="f16", out="f16",
             page=32, window=1024, empty=0),
        # the towers' second feed-forward projection for one token (4304 columns padded to 4320)
        dict(name="vec-1x1152x4320", op="vec", m=1, n=1152, k=4320, type="q4_0", dt="f32", bias=True, res=True),
        # logits of one token over the text tower's vocabulary
        dict(name="vec-1x256000x1152", op="vec", m=1, n=256000, k=1152, type="q4_1", dt="f32", bias=False, res=False),
        # a wide feed-forward projection for seven requests
        dict(name="vec-7x28672x8192", op="vec", m=7, n=28672, k=8192, type="q4_0", dt="bf16", bias=False, res=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "rope", "attn", "attn", "vec", "vec"])
    if op == "plan":
        new_hi = rng.choice([1, 1, _log(rng, 2, 2048)])
        return dict(op=op, n=_log(rng, 1, 1024 if new_hi == 1 else 400), ctx_lo=0, ctx_hi=_log(rng, 16, 32768),
                    new_lo=1 if new_hi == 1 else 0, new_hi=new_hi, page=rng.choice([8, 16, 32, 64, 128]))
    if op == "rope":
        d = rng.choice([64, 72, 80, 96, 128, 256])
        hk = rng.choice([1, 2, 4, 8, 16])
        hq = hk * rng.choice([1, 2, 3, 4, 5, 8])
        dt = rng.choice(["f32", "f16", "bf16"])
        rot = rng.choice([d, d, d // 2 // 8 * 8])
        T = _log(rng, 1, max(2, 60_000_000 // ((hq + 2 * hk) * d)))
        return dict(op=op, T=min(T, 30000), hq=hq, hk=hk, d=d, rot=rot, inter=rng.random() < 0.4, dt=dt,
                    cdt=dt if dt != "f32" else rng.choice(["f16", "bf16"]), page=rng.choice([16, 32, 64]),
                    n_pos=32768, norm=rng.random() < 0.7)
    if op == "attn":
        d = rng.choice([64, 72, 80, 96, 128, 128, 256])
        hk = rng.choice([1, 2, 4, 8, 16])
        hq = hk * rng.choice([1, 2, 3, 4, 5, 8, 16])
        n = _log(rng, 1, 512)
        hi = min(131072, _log(rng, 8, max(16, 250_000_000 // (n * hk * d))))
        dt = rng.choice(["f16", "bf16"])
        return dict(op=op, n=n, lo=rng.choice([1, (hi + 1) // 2, hi]), hi=hi, hq=hq, hk=hk, d=d, dt=dt,
                    out=rng.choice(["f32", dt]), page=rng.choice([8, 16, 32, 64, 128]),
                    window=rng.choice([0, 0, 0, _log(rng, 16, 8192)]), empty=rng.choice([0, 0, n // 8]))
    m = rng.choice([1, 1, 1, 2, 3, 4, 5, 8])
    k = 32 * _log(rng, 4, 448)
    return dict(op=op, m=m, n=_log(rng, 64, min(256000, 280_000_000 // k)), k=k, type=rng.choice(["q4_0", "q4_1"]),
                dt=rng.choice(["f32", "f32", "f16", "bf16"]), bias=rng.random() < 0.3, res=rng.random() < 0.3)


def _spread(n, lo, hi):
    """n lengths over [lo, hi], the same for every seed (the seed deals them
    to the requests); the first is hi."""
    return [hi] + [lo + int((hi - lo + 1) * ((i * GOLDEN) % 1.0)) for i in range(1, n)]


def _plan_lens(c):
    n = c["n"]
    ctx = _spread(n, c["ctx_lo"], c["ctx_hi"])
    new = _spread(n, c["new_lo"], c["new_hi"])
    # every fourth request of a ragged batch is a first prompt with nothing cached
    if c["new_hi"] > 1:
        ctx = [0 if i % 4 == 1 else x for i, x in enumerate(ctx)]
    return ctx, new[::-1]


def _attn_lens(c):
    lens = _spread(c["n"], c["lo"], c["hi"])
    return [0 if 0 < i <= c["empty"] else x for i, x in enumerate(lens)]


def _up(a, b):
    return -(-a // b)


def work(c):
    if c["op"] == "plan":
        ctx, new = _plan_lens(c)
        took = sum(_up(a + b, c["page"]) - _up(a, c["page"]) for a, b in zip(ctx, new))
        # lengths and taken pages read, table entries and four values a token written
        return {"bytes": 8 * c["n"] + 8 * took + 16 * sum(new), "flops": 0}
    if c["op"] == "rope":
        e = c["T"] * (c["hq"] + 2 * c["hk"]) * c["d"]
        return {"bytes": e * (SIZE[c["dt"]] + SIZE[c["cdt"]]) + c["T"] * (4 * c["rot"] + 8),
                "flops": 7 * c["T"] * (c["hq"] + c["hk"]) * c["d"]}
    if c["op"] == "attn":
        keys = sum(min(x, c["window"]) if c["window"] else x for x in _attn_lens(c))
        pages = sum(_up(min(x, c["window"]) if c["window"] else x, c["page"]) for x in _attn_lens(c))
        return {"bytes": keys * c["hk"] * c["d"] * 4 + 4 * pages + c["n"] * c["hq"] * c["d"] * (2 + SIZE[c["out"]]),
                "flops": 4 * keys * c["hq"] * c["d"]}
    n, k, m = c["n"], c["k"], c["m"]
    return {"bytes": n * k // 32 * BLOCK[c["type"]] + m * k * SIZE[c["dt"]] + m * n * SIZE[c["dt"]]
            + 4 * n * c["bias"] + 4 * m * n * c["res"], "flops": 2 * m * n * k}


# ---------------------------------------------------------------- the inputs
def _b2q():
    pkg = str(Path(__file__).resolve().parents[1] / "hbd-siglip2.cpp_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import b2q
    b2q.init(torch.cuda.current_device())
    return b2q


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + 17)

    def randn(*shape, dt=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dt)

    def perm(n):
        return torch.randperm(n, generator=g, device="cuda")

    s = {"c": c}
    if c["op"] == "plan":
        p = c["page"]
        deal = perm(c["n"])
        ctx, new = (_ints(v)[deal] for v in _plan_lens(c))
        need, have = (ctx + new + p - 1) // p, (ctx + p - 1) // p
        a, b = _plan_lens(c)
        owned = sum(_up(x, p) for x in a)
        took = sum(_up(x + y, p) - _up(x, p) for x, y in zip(a, b))
        width = max(_up(x + y, p) for x, y in zip(a, b)) + 2
        ids = perm(owned + took + 64).to(torch.int32)
        at = torch.arange(width, device="cuda")
        mine = at[None] < have[:, None]
        table = torch.full((c["n"], width), -1, dtype=torch.int32, device="cuda")
        first = torch.cumsum(have, 0) - have
        table = torch.where(mine, ids[(first[:, None] + at[None]).clamp(max=owned + took)], table)
        s.update(ctx=ctx, new=new, free=ids[owned:].contiguous(), table=table.contiguous(), T=sum(b))
    elif c["op"] == "rope":
        T, d, hk, p = c["T"], c["d"], c["hk"], c["page"]
        pages = _up(T, p) + 3
        s["qkv"] = (randn(T, (c["hq"] + 2 * hk) * d) * 1.5).to(DT[c["dt"]])
        s["qw"], s["kw"] = ((1 + 0.2 * randn(d)) if c["norm"] else None for _ in range(2))
        ang = torch.arange(c["n_pos"], device="cuda").double()[:, None] * \
            (10000.0 ** (-2.0 * torch.arange(c["rot"] // 2, device="cuda").double() / c["rot"]))[None]
        s["rope"] = torch.cat([ang.cos(), ang.sin()], 1).float()
        s["pos"] = torch.randint(0, c["n_pos"], (T,), generator=g, device="cuda", dtype=torch.int32)
        s["slot"] = perm(pages * p)[:T].to(torch.int32)
        s["k"], s["v"] = (randn(pages, hk, p, d, dt=DT[c["cdt"]]) for _ in range(2))
        s["q"] = torch.empty(T, c["hq"] * d, dtype=DT[c["cdt"]], device="cuda")
    elif c["op"] == "attn":
        d, hk, p, dt = c["d"], c["hk"], c["page"], DT[c["dt"]]
        host = _attn_lens(c)
        lens = _ints(host)[perm(c["n"])]
        blocks = (lens + p - 1) // p
        total = sum(_up(x, p) for x in host)
        ids = perm(total + 5).to(torch.int32)
        at = torch.arange(max(1, _up(c["hi"], p)), device="cuda")
        first = torch.cumsum(blocks, 0) - blocks
        s["table"] = torch.where(at[None] < blocks[:, None], ids[(first[:, None] + at[None]).clamp(max=total)],
                                 -1).to(torch.int32).contiguous()
        s["lens"] = lens
        s["scale"] = 1.0 / math.sqrt(d)
        # normed and rotated heads: scores with a spread of about two
        s["q"] = (2.0 * randn(c["n"], c["hq"] * d)).to(dt)
        s["k"], s["v"] = (randn(total + 5, hk, p, d, dt=dt) for _ in range(2))
        s["out"] = torch.empty(c["n"], c["hq"] * d, dtype=DT[c["out"]], device="cuda")
    else:
        n, k, m = c["n"], c["k"], c["m"]
        s["raw"] = torch.randint(0, 256, (n, k // 32, BLOCK[c["type"]]), generator=g, device="cuda", dtype=torch.uint8)
        step = (0.004 + 0.002 * torch.rand(n, k // 32, 1, generator=g, device="cuda")).half()
        s["raw"][:, :, 0:2] = step.view(torch.uint8)
        if c["type"] == "q4_1":
            s["raw"][:, :, 2:4] = (-7.5 * step.float() + 0.002 * randn(n, k // 32, 1)).half().view(torch.uint8)
        s["x"] = randn(m, k).to(DT[c["dt"]])
        s["bias"] = 0.1 * randn(n) if c["bias"] else None
        s["res"] = randn(m, n) if c["res"] else None
        s["y"] = torch.empty(m, n, dtype=DT[c["dt"]], device="cuda")
    return s


def prepare(c, seed):
    s = _inputs(c, seed)
    if c["op"] == "plan":
        n, T = c["n"], s["T"]
        s["out"] = {k: torch.empty(max(T, 1), dtype=torch.int32, device="cuda") for k in ("seq", "pos", "slot", "len")}
        s["counts"] = torch.zeros(2, dtype=torch.int32, device="cuda")
    if own:   # what a program keeps next to its buffers: the cache's description, scratch, the registered weight
        b = s["b2q"] = _b2q()
        if c["op"] in ("rope", "attn"):
            s["cache"] = b.KVCache(s["k"], s["v"])
        if c["op"] == "attn":
            s["scratch"] = b.attention_paged_scratch(c["hq"], s["cache"])
        if c["op"] == "vec":
            s["w"] = b.WeightQ4(s["raw"], c["n"], c["k"], b.GGML_Q4_1 if c["type"] == "q4_1" else b.GGML_Q4_0)
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    return (_own if own else _plain)[s["c"]["op"]](s)


def _own_plan(s):
    o = s["out"]
    s["b2q"].kv_plan(s["ctx"], s["new"], s["c"]["page"], s["free"], s["table"], o["seq"], o["pos"], o["slot"],
                     o["len"], s["counts"])
    return {"table": s["table"], "counts": s["counts"], **o}


def _own_rope(s):
    c = s["c"]
    s["b2q"].qk_norm_rope(s["qkv"], c["hq"], s["cache"], s["q"], s["pos"], s["slot"], q_weight=s["qw"],
                          k_weight=s["kw"], eps=1e-6, rope=s["rope"], interleaved=c["inter"])
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _own_attn(s):
    s["b2q"].attention_paged(s["q"], s["cache"], s["table"], s["lens"], s["out"], s["scratch"], scale=s["scale"],
                             window=s["c"]["window"])
    return s["out"]


def _own_vec(s):
    s["b2q"].mul_vec_q4(s["w"], s["x"], s["c"]["m"], s["y"], bias=s["bias"], residual=s["res"])
    return s["y"]


def _plain_plan(s):
    p, ctx, new, table, free, T = s["c"]["page"], s["ctx"], s["new"], s["table"], s["free"], s["T"]
    n, width = table.shape
    need, have = (ctx + new + p - 1) // p, (ctx + p - 1) // p
    add = need - have
    first = torch.cumsum(add, 0) - add
    j = torch.arange(width, device="cuda")[None] - have[:, None]
    mine = (j >= 0) & (j < add[:, None])
    table.copy_(torch.where(mine, free[(first[:, None] + j).clamp(0, free.numel() - 1)], table))
    end = torch.cumsum(new, 0)
    t = torch.arange(max(T, 1), device="cuda")
    seq = torch.searchsorted(end, t, right=True).clamp(max=n - 1)
    ok = t < end[-1]
    pos = ctx[seq] + t - (end[seq] - new[seq])
    slot = table[seq, (pos // p).clamp(0, width - 1)] * p + pos % p
    neg = torch.full_like(slot, -1)
    out = {"seq": torch.where(ok, seq, neg), "pos": torch.where(ok, pos, neg), "slot": torch.where(ok, slot, neg),
           "len": torch.where(ok, pos + 1, 0)}
    return {"table": table, "counts": torch.stack([end[-1], add.sum()]).to(torch.int32),
            **{k: v.to(torch.int32) for k, v in out.items()}}


def _plain_rope(s):
    c = s["c"]
    T, d, hq, hk, p, rot = c["T"], c["d"], c["hq"], c["hk"], c["page"], c["rot"]
    x = s["qkv"].float().view(T, hq + 2 * hk, d)
    cs = s["rope"][s["pos"].long()][:, None]
    cos, sin = cs[..., :rot // 2], cs[..., rot // 2:]

    def turn(h, w):
        if w is not None:
            h = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * w
        a, b = (h[..., 0:rot:2], h[..., 1:rot:2]) if c["inter"] else (h[..., :rot // 2], h[..., rot // 2:rot])
        u, v = a * cos - b * sin, b * cos + a * sin
        r = torch.stack([u, v], -1).flatten(-2) if c["inter"] else torch.cat([u, v], -1)
        return torch.cat([r, h[..., rot:]], -1)

    q, k = turn(x[:, :hq], s["qw"]), turn(x[:, hq:hq + hk], s["kw"])
    slot = s["slot"].long()
    s["k"][slot // p, :, slot % p] = k.to(s["k"].dtype)
    s["v"][slot // p, :, slot % p] = x[:, hq + hk:].to(s["v"].dtype)
    return {"q": q.reshape(T, hq * d).to(s["q"].dtype), "k": s["k"], "v": s["v"]}


def _plain_attn(s):
    c = s["c"]
    n, hq, hk, d, p = c["n"], c["hq"], c["hk"], c["d"], c["page"]
    lens, table = s["lens"], s["table"].clamp(min=0)
    span = table.shape[1] * p
    k = s["k"][table].transpose(1, 2).reshape(n, hk, span, d).float()
    v = s["v"][table].transpose(1, 2).reshape(n, hk, span, d).float()
    q = s["q"].float().view(n, hk, hq // hk, d)
    sc = (q @ k.transpose(-1, -2)) * s["scale"]
    at = torch.arange(span, device="cuda")[None]
    live = at < lens[:, None]
    if c["window"]:
        live = live & (at >= lens[:, None] - c["window"])
    sc = torch.where(live[:, None, None], sc, torch.full_like(sc, -1e30))
    e = torch.exp(sc - sc.amax(-1, keepdim=True)) * live[:, None, None]
    z = e.sum(-1, keepdim=True)
    o = (e @ v) / torch.where(z > 0, z, torch.ones_like(z))
    return o.reshape(n, hq * d).to(DT[c["out"]])


def _plain_vec(s):
    raw, c = s["raw"], s["c"]
    d = raw[:, :, 0:2].contiguous().view(torch.float16).float()
    q = raw[:, :, 4 if c["type"] == "q4_1" else 2:]
    q = torch.cat([q & 15, q >> 4], 2).float()
    if c["type"] == "q4_1":
        w = q * d + raw[:, :, 2:4].contiguous().view(torch.float16).float()
    else:
        w = (q - 8) * d
    y = s["x"].float() @ w.view(c["n"], c["k"]).t()
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["res"] is not None:
        y = y + s["res"]
    return y.to(s["y"].dtype)


_own = {"plan": _own_plan, "rope": _own_rope, "attn": _own_attn, "vec": _own_vec}
_plain = {"plan": _plain_plan, "rope": _plain_rope, "attn": _plain_attn, "vec": _plain_vec}


# ---------------------------------------------------------------- 64 bits
def exact(c, seed):
    if c["op"] == "plan":
        return None     # whole numbers: equality with the plain form decides
    s = _inputs(c, seed)
    return {"rope": _exact_rope, "attn": _exact_attn, "vec": _exact_vec}[c["op"]](c, s)


def _exact_rope(c, s):
    hq, hk, d, rot, p = c["hq"], c["hk"], c["d"], c["rot"], c["page"]
    x = s["qkv"].double()
    cos, sin = s["rope"].double()[s["pos"].long()].split(rot // 2, 1)
    lo = torch.arange(rot // 2, device="cuda")
    lo, hi = (2 * lo, 2 * lo + 1) if c["inter"] else (lo, lo + rot // 2)
    q = torch.empty_like(x[:, :hq * d])
    k, v = s["k"].double(), s["v"].double()
    page, row = s["slot"].long() // p, s["slot"].long() % p
    for h in range(hq + 2 * hk):
        y = x[:, h * d:(h + 1) * d].clone()
        w = s["qw"] if h < hq else s["kw"]
        if h < hq + hk:
            if w is not None:
                y *= w.double() * torch.rsqrt(y.pow(2).sum(1) / d + 1e-6)[:, None]
            a, b = y[:, lo], y[:, hi]
            y[:, lo], y[:, hi] = a * cos - b * sin, a * sin + b * cos
        if h < hq:
            q[:, h * d:(h + 1) * d] = y
        elif h < hq + hk:
            k[page, h - hq, row] = y
        else:
            v[page, h - hq - hk, row] = y
    return {"q": q, "k": k, "v": v}


def _exact_attn(c, s):
    n, hq, hk, d, p = c["n"], c["hq"], c["hk"], c["d"], c["page"]
    out = torch.zeros(n, hq, d, dtype=torch.float64, device="cuda")
    for i, L in enumerate(s["lens"].tolist()):
        if L == 0:
            continue
        a = max(0, L - c["window"]) if c["window"] else 0
        j = torch.arange(a, L, device="cuda")
        page = s["table"][i].long()[j // p]
        for h in range(hk):
            k, v = s["k"][page, h, j % p].double(), s["v"][page, h, j % p].double()
            g = slice(h * (hq // hk), (h + 1) * (hq // hk))
            q = s["q"][i].double().view(hq, d)[g]
            out[i, g] = torch.softmax(q @ k.t() / math.sqrt(d), 1) @ v
    return out.view(n, hq * d)


def _exact_vec(c, s):
    n, k, m, x = c["n"], c["k"], c["m"], s["x"].double()
    y = torch.empty(m, n, dtype=torch.float64, device="cuda")
    for r in range(0, n, 8192):
        b = s["raw"][r:r + 8192]
        d = b[..., :2].clone().view(torch.half).double()
        w = torch.empty(b.shape[0], k // 32, 32, dtype=torch.float64, device="cuda")
        if c["type"] == "q4_0":
            w[..., :16], w[..., 16:] = b[..., 2:].bitwise_and(15), b[..., 2:] // 16
            w = (w - 8) * d
        else:
            w[..., :16], w[..., 16:] = b[..., 4:].bitwise_and(15), b[..., 4:] // 16
            w = w * d + b[..., 2:4].clone().view(torch.half).double()
        y[:, r:r + 8192] = x @ w.view(-1, k).t()
    for more in (s["bias"], s["res"]):
        if more is not None:
            y += more.double()
    return y
