"""What the operators beside the sealed cache are measured on: the step from a projection to cache rows (norm of every
head, rotary positions, write into pages), attention of one new token over a paged 16-bit cache, and the ownership of
pages (fork, extend with copy on write, free, compact).

listed() and draw() give cases, prepare() what a program has in hand before the call, run() one pass: in plain torch
operations in 32 bits, or, where `own` is true, through kv16 (the framework's own calls). exact() states the computed
results in 64 bits.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def _kv16():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sj-kvarn-codec_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import kv16
    return kv16


# ---- the cases ------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one token of one chat through the norms, the rotation and the cache write: a launch's latency
        dict(name="qkv-1-token", op="qkv", n=1, D=128, H=8, grp=4, type="bf16", norm=True, n_rot=128, layout="half",
             scaling="none", factor=1.0, base=1e6, page=16, far=2000, to="pages"),
        # a pool's decode step: 64 sequences at up to 64K, rotation of half the head, scaled for long contexts, no norm
        dict(name="qkv-64-rotary", op="qkv", n=64, D=256, H=4, grp=4, type="f16", norm=False, n_rot=128, layout="half",
             scaling="yarn", factor=8.0, base=1e4, page=128, far=65536, to="pages"),
        # a long prompt's prefill at once: 32,768 positions written into the pages of one sequence
        dict(name="qkv-32768-prefill", op="qkv", n=32768, D=256, H=4, grp=4, type="bf16", norm=True, n_rot=256,
             layout="half", scaling="none", factor=1.0, base=1e6, page=128, far=32768, to="pages"),
        # rotary positions alone on 32-bit rows, as the sealed cache's store takes them: 8,320 positions near the end of
        # a context of a million tokens, neighbouring channels as pairs
        dict(name="rotary-8320-rows", op="qkv", n=8320, D=256, H=4, grp=4, type="f32", norm=False, n_rot=256,
             layout="pair", scaling="linear", factor=4.0, base=1e4, page=128, far=1048576, to="rows"),
        # the next token of one short chat
        dict(name="attend-1x611", op="attend", n=1, lo=611, hi=611, spread=0, D=128, H=8, grp=4, page=16, type="bf16",
             io="bf16", window=0),
        # one sequence of 100,000 tokens, 32-bit queries and outputs beside the sealed layers'
        dict(name="attend-1x100000", op="attend", n=1, lo=100000, hi=100000, spread=0, D=256, H=4, grp=4, page=128,
             type="f16", io="f32", window=0),
        # a pool of long contexts between 8K and 64K
        dict(name="attend-32x8k-64k", op="attend", n=32, lo=8192, hi=65536, spread=3, D=256, H=4, grp=4, page=128,
             type="bf16", io="bf16", window=0),
        # many short chats of very different lengths, a slot without a chat among them
        dict(name="attend-256-short", op="attend", n=256, lo=0, hi=2048, spread=5, D=128, H=8, grp=4, page=16,
             type="f16", io="f16", window=0),
        # sliding-window layers: every head has its own cache, 4,096 positions of up to 32K are live
        dict(name="attend-48-window", op="attend", n=48, lo=100, hi=32768, spread=7, D=64, H=24, grp=1, page=16,
             type="bf16", io="bf16", window=4096),
        # a beam step: 8 beams follow 4 of the old ones, which go; the shared last pages are split
        dict(name="pages-beams-8", op="pages", kind="beams", n=8, len=1003, page=16, H=8, D=128, layers=16, type="bf16",
             blocks=1024),
        # 64 samples of one prompt: the prompt forked 63 times, each copy's last page split, the copies dropped
        dict(name="pages-samples-64", op="pages", kind="samples", n=64, len=32700, page=128, H=4, D=256, layers=16,
             type="f16", blocks=384),
        # a server's turn: 4 of 32 sequences leave, the pool is compacted, new ones of the same lengths come in
        dict(name="pages-evict-compact", op="pages", kind="evict", n=32, len=2000, page=16, H=8, D=128, layers=8,
             type="bf16", blocks=4096),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["qkv", "attend", "attend", "pages"])
        D, H, grp = rng.choice([64, 96, 128, 256]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8])
        typ = rng.choice(["f16", "bf16"])
        if op == "qkv":
            n = _log(rng, 1, 16384)
            typ = rng.choice(["f16", "bf16", "f32"])
            c = dict(op=op, n=n, D=D, H=H, grp=grp, type=typ, norm=rng.random() < 0.6,
                     n_rot=rng.choice([D, D, D // 2, D // 4, 20]), layout=rng.choice(["half", "pair"]),
                     scaling=rng.choice(["none", "linear", "ntk", "yarn", "bands"]), factor=rng.choice([2.0, 4.0, 8.0]),
                     base=rng.choice([1e4, 5e5, 1e6]), page=rng.choice([16, 24, 64, 128]), far=max(n, _log(rng, 512, 1000000)),
                     to="rows" if typ == "f32" else rng.choice(["rows", "pages", "pages"]))
            if (H * grp + 2 * H) * D * n > 24 * 256 * 32768:
                continue
        elif op == "attend":
            n = _log(rng, 1, 256)
            hi = _log(rng, 1, 100000)
            lo = rng.choice([0, min(hi, _log(rng, 1, hi))])
            grp = rng.choice([1, 2, 4, 5, 8, 16, 20])
            c = dict(op=op, n=n, lo=lo, hi=hi, spread=rng.randrange(1, 1000), D=D, H=H, grp=grp,
                     page=rng.choice([16, 24, 32, 128, 1]), type=typ, io=rng.choice([typ, typ, "f32"]),
                     window=rng.choice([0, 0, _log(rng, 1, hi)]))
            if n * hi * H * D > 1.1e9 or 4 * sum(_lens(c)) * H * D > 4.0e9 or n * hi * H * grp > 3e8:
                continue
        else:
            kind = rng.choice(["beams", "samples", "evict"])
            n = {"beams": 2 * _log(rng, 1, 32), "samples": _log(rng, 2, 64), "evict": 8 * _log(rng, 1, 8)}[kind]
            page, length = rng.choice([16, 64, 128]), _log(rng, 20, 20000)
            D = rng.choice([64, 128, 256])
            layers = _log(rng, 1, 32)
            per = -(-length // page)
            blocks = {"beams": (n + n // 2) * (per + 1) + n, "samples": 2 * per + 2 * n, "evict": 2 * n * per}[kind] + rng.randrange(1, 50)
            c = dict(op=op, kind=kind, n=n, len=length, page=page, H=H, D=D, layers=layers, type=typ, blocks=blocks)
            if blocks * page * H * D * layers * 4 > 3.5e9:
                continue
        if 3072 not in _sizes(c):
            return c


def _sizes(c):
    H, D = c["H"], c["D"]
    s = [H * D, c["page"], c.get("len"), c.get("n"), c.get("lo"), c.get("hi"), c.get("blocks"), c.get("far"), c["page"] * H]
    if "grp" in c:
        s += [H * c["grp"] * D, (H * c["grp"] + 2 * H) * D, H * c["grp"]]
    if c["op"] == "attend":
        s += _lens(c)
    return s


def _lens(c):
    """The lengths of an attention case's sequences: between lo and hi, spread over their logarithm where that is wide."""
    if not c["spread"]:
        return [c["hi"]] * c["n"]
    r = random.Random(c["spread"])
    wide = c["hi"] > 10 * c["lo"]
    lens = [_log(r, max(c["lo"], 1), c["hi"]) if wide else r.randint(c["lo"], c["hi"]) for _ in range(c["n"])]
    lens[0], lens[-1] = c["lo"], c["hi"]
    return [n - 1 if n == 3072 else n for n in lens]


def _share(c):
    """Pages that one sequence of a page case holds, and whether its last page is only partly filled."""
    return -(-c["len"] // c["page"]), c["len"] % c["page"] != 0


# ---- what a program has in hand ------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(shape, dtype, g):
    return torch.randn(shape, dtype=dtype, device="cuda", generator=g)


def _inv_freq(c):
    """Angle per position of every pair (64 bits), and the amplitude of the rotation."""
    n, base, f, ctx = c["n_rot"], c["base"], c["factor"], 8192.0
    i = np.arange(n // 2, dtype=np.float64)
    amp = 1.0
    if c["scaling"] == "ntk" and n > 2:
        base = base * f ** (n / (n - 2.0))
    freq = base ** (-2.0 * i / n)
    if c["scaling"] == "linear":
        freq = freq / f
    if c["scaling"] == "yarn":
        at = [n * math.log(ctx / (b * 2 * math.pi)) / (2 * math.log(base)) for b in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), n - 1)
        ramp = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
        freq = freq / f * ramp + freq * (1 - ramp)
        amp = 0.1 * math.log(f) + 1.0
    if c["scaling"] == "bands":
        turns = ctx * freq / (2 * math.pi)              # turns over the original context
        s = np.clip((turns - 1.0) / (4.0 - 1.0), 0, 1)
        freq = freq / f * (1 - s) + freq * s
    return freq, amp


def _prepare_qkv(c, seed):
    g, T = _gen(seed), TYPES[c["type"]]
    n, D, H, HQ = c["n"], c["D"], c["H"], c["H"] * c["grp"]
    s = dict(case=c)
    s["qkv"] = _normal((n, (HQ + 2 * H) * D), T, g)                   # one projection's rows: q, k and v heads
    s["wq"] = (1 + 0.1 * _normal((D,), torch.float32, g)) if c["norm"] else None
    s["wk"] = (1 + 0.1 * _normal((D,), torch.float32, g)) if c["norm"] else None
    if c["n"] > 256:                                                  # a prompt: positions in a row, of one sequence
        first = c["far"] - n
        s["pos"] = torch.arange(first, first + n, dtype=torch.int32, device="cuda")
        s["rows"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        seqs = 1
    else:                                                             # a decode step: token i is sequence i's next
        s["pos"] = torch.randint(0, c["far"], (n,), generator=g, device="cuda").int()
        s["rows"] = torch.arange(n, dtype=torch.int32, device="cuda")
        seqs = n
    freq, amp = _inv_freq(c)
    s["amp"] = amp
    # turns per position in units of 2^-64: positions times these, modulo 2^64, are angles without a growing error
    step = [int(math.fmod(float(f) / (2 * math.pi), 1.0) * 2.0 ** 64) for f in freq]
    s["step"] = torch.tensor([x - 2 ** 64 if x >= 2 ** 63 else x for x in step], dtype=torch.int64, device="cuda")
    s["q_out"] = torch.empty((n, HQ, D), dtype=T, device="cuda")
    if c["to"] == "rows":
        s["k_out"] = torch.empty((n, H, D), dtype=T, device="cuda")
        s["v_out"] = torch.empty((n, H, D), dtype=T, device="cuda")
    else:
        # only pages that take a token exist: the others of a long context are behind the sequence's own
        P, stride = c["page"], -(-c["far"] // c["page"])
        slot = s["rows"].long() * stride + s["pos"].long() // P
        used, at = torch.unique(slot, return_inverse=True)
        pages = used.numel()
        perm = torch.randperm(pages, generator=g, device="cuda")
        s["tables"] = torch.full((seqs * stride,), -1, dtype=torch.int32, device="cuda")
        s["tables"][used] = perm.int()
        s["tables"] = s["tables"].view(seqs, stride)
        s["k"] = _normal((1, pages, P, H, D), T, g)
        s["v"] = _normal((1, pages, P, H, D), T, g)
    if own:
        kv16 = _kv16()
        rope = kv16.Rope(c["n_rot"], layout=c["layout"], base=c["base"], scaling=c["scaling"], factor=c["factor"], n_ctx=8192)
        s["cache"] = kv16.Cache(s["k"], s["v"], s["tables"]) if c["to"] == "pages" else None
        s["step_call"] = kv16.Qkv(D, rope=rope, q_norm=s["wq"], k_norm=s["wk"], eps=EPS, cache=s["cache"])
    return s


def _prepare_attend(c, seed):
    g, T = _gen(seed), TYPES[c["type"]]
    n, D, H, P = c["n"], c["D"], c["H"], c["page"]
    lens = _lens(c)
    per = [-(-x // P) for x in lens]
    stride, pages = max(per), sum(per)
    s = dict(case=c, scale=1.0 / math.sqrt(D))
    perm = torch.randperm(pages, generator=g, device="cuda").int()
    at = torch.tensor([0] + per[:-1], device="cuda").cumsum(0)
    idx = torch.arange(stride, device="cuda")
    have = idx[None, :] < torch.tensor(per, device="cuda")[:, None]
    s["tables"] = torch.where(have, perm[(at[:, None] + idx[None, :]).clamp(max=pages - 1)], torch.full((), -1, dtype=torch.int32, device="cuda"))
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["k"] = _normal((1, pages, P, H, D), T, g)
    s["k"] *= (0.5 * torch.randn((H, D), device="cuda", generator=g)).exp().to(T)     # channels of unlike size
    s["v"] = _normal((1, pages, P, H, D), T, g)
    s["q"] = _normal((n, H * c["grp"], D), torch.float32, g).to(TYPES[c["io"]])
    s["out"] = torch.empty_like(s["q"])
    if own:
        s["cache"] = _kv16().Cache(s["k"], s["v"], s["tables"])
    return s


def _prepare_pages(c, seed):
    g, T = _gen(seed), TYPES[c["type"]]
    n, P, blocks = c["n"], c["page"], c["blocks"]
    per, _ = _share(c)
    s = dict(case=c, turn=0)
    s["k"] = _normal((c["layers"], blocks, P, c["H"], c["D"]), T, g)
    s["v"] = _normal((c["layers"], blocks, P, c["H"], c["D"]), T, g)
    rows, live, stride = {"beams": (2 * n, n, per + 1), "samples": (n, 1, per + 1), "evict": (n, n, per + 1)}[c["kind"]]
    used = live * per
    ids = torch.randperm(used, generator=g, device="cuda").int()
    tables = torch.full((rows, stride), -1, dtype=torch.int32, device="cuda")
    tables[:live, :per] = ids.view(live, per)
    s["tables"] = tables
    # the pool: free ids as a stack (the lowest on top), how many are free, how many owners a page has beyond the first
    s["ids"] = torch.arange(blocks - 1, -1, -1, dtype=torch.int32, device="cuda")
    s["n_free"] = torch.tensor([blocks - used], dtype=torch.int32, device="cuda")
    s["shares"] = torch.zeros(blocks, dtype=torch.int32, device="cuda")
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    if c["kind"] == "beams":
        kids = torch.randperm(n, generator=g, device="cuda").int() % (n // 2)     # each survivor has two children
        keep = torch.randperm(n, generator=g, device="cuda").int()[: n // 2]
        par = keep[kids.long()]
        halves = (torch.arange(n, dtype=torch.int32, device="cuda"), torch.arange(n, 2 * n, dtype=torch.int32, device="cuda"))
        s["src"], s["dst"] = (par, par + n), (halves[1], halves[0])
        s["old"] = halves
        s["lens"] = dev([c["len"]] * n)
    elif c["kind"] == "samples":
        s["src"], s["dst"] = dev([0] * (n - 1)), dev(list(range(1, n)))
        s["all"] = dev(list(range(n)))
        s["lens"] = dev([c["len"]] * n)
    else:
        q = n // 8
        s["gone"] = [dev(list(range(i * q, (i + 1) * q))) for i in range(8)]
        s["none"], s["full"] = dev([0] * q), dev([c["len"]] * q)
    if own:
        kv16 = _kv16()
        s["pages"] = kv16.Pages(tables, c["page"], slabs=[s["k"], s["v"]], ids=s["ids"], n_free=blocks - used)
    return s


def prepare(case, seed):
    return {"qkv": _prepare_qkv, "attend": _prepare_attend, "pages": _prepare_pages}[case["op"]](case, seed)


# ---- one pass -------------------------------------------------------------------------------------------------------

def _heads(s):
    c = s["case"]
    n, D, H, HQ = c["n"], c["D"], c["H"], c["H"] * c["grp"]
    x = s["qkv"]
    return x[:, : HQ * D].view(n, HQ, D), x[:, HQ * D: (HQ + H) * D].view(n, H, D), x[:, (HQ + H) * D:].view(n, H, D)


def _norm_rotate(x, w, c, cos, sin):
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    n = c["n_rot"]
    r = x[..., :n]
    a, b = (r[..., : n // 2], r[..., n // 2:]) if c["layout"] == "half" else (r[..., 0::2], r[..., 1::2])
    ra, rb = a * cos - b * sin, a * sin + b * cos
    r = torch.cat((ra, rb), -1) if c["layout"] == "half" else torch.stack((ra, rb), -1).flatten(-2)
    return torch.cat((r, x[..., n:]), -1)


def _run_qkv(s):
    c = s["case"]
    q, k, v = _heads(s)
    if own:
        if c["to"] == "rows":
            s["step_call"](q, k, v, s["pos"], q_out=s["q_out"], k_out=s["k_out"], v_out=s["v_out"])
            return s["q_out"], s["k_out"], s["v_out"]
        s["step_call"](q, k, v, s["pos"], q_out=s["q_out"], rows=s["rows"])
        return s["q_out"], s["k"], s["v"]
    turns = ((s["pos"].long()[:, None] * s["step"][None, :]) >> 32).float() * 2.0 ** -32
    ang = turns * (2 * math.pi)
    cos, sin = (ang.cos() * s["amp"])[:, None], (ang.sin() * s["amp"])[:, None]
    T = TYPES[c["type"]]
    s["q_out"].copy_(_norm_rotate(q, s["wq"], c, cos, sin))
    kr = _norm_rotate(k, s["wk"], c, cos, sin).to(T)
    if c["to"] == "rows":
        s["k_out"].copy_(kr)
        s["v_out"].copy_(v)
        return s["q_out"], s["k_out"], s["v_out"]
    pos = s["pos"].long()
    page = s["tables"][s["rows"].long(), pos // c["page"]].long()
    s["k"][0][page, pos % c["page"]] = kr
    s["v"][0][page, pos % c["page"]] = v
    return s["q_out"], s["k"], s["v"]


def _run_attend(s):
    c = s["case"]
    if own:
        return s["cache"].attend(0, s["q"], s["lens"], s["scale"], window=c["window"], out=s["out"])
    n, H, grp, D, P = c["n"], c["H"], c["grp"], c["D"], c["page"]
    page = s["tables"].long().clamp(min=0)
    k = s["k"][0][page].view(n, -1, H, D)
    t = torch.arange(k.shape[1], device="cuda")
    dead = t[None, :] >= s["lens"][:, None]
    if c["window"]:
        dead = dead | (t[None, :] < s["lens"][:, None] - c["window"])
    q = s["q"].float().view(n, H, grp, D) * s["scale"]
    p = q @ k.float().permute(0, 2, 3, 1)
    p = p.masked_fill(dead[:, None, None, :], float("-inf"))
    p = (p - p.amax(-1, keepdim=True).clamp(min=-1e30)).exp()
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)                  # a sequence without a live position gives zeros
    del k
    v = s["v"][0][page].view(n, -1, H, D)
    out = p @ v.float().permute(0, 2, 1, 3)
    s["out"].copy_(out.view(n, H * grp, D))
    return s["out"]


# The pages' plain forms. A page is free (its id on the stack) or held by 1 + shares[id] table entries; -1 is no page.

def _fork(s, src, dst):
    t = s["tables"][src.long()]
    s["tables"][dst.long()] = t
    live = t[t >= 0].long()
    s["shares"].index_add_(0, live, torch.ones_like(live, dtype=torch.int32))


def _free(s, rows):
    """Entries of the rows give up their pages; the pages without an owner left go onto the stack, the lowest on top."""
    t = s["tables"][rows.long()]
    live = t[t >= 0].long()
    s["shares"].index_add_(0, live, torch.full_like(live, -1, dtype=torch.int32))
    gone = s["shares"] < 0
    s["shares"].clamp_(min=0)
    ids = gone.nonzero()[:, 0].int().flip(0)
    at = s["n_free"].long() + torch.arange(ids.numel(), device="cuda")
    s["ids"][at] = ids
    s["n_free"] += ids.numel()
    s["tables"][rows.long()] = -1


def _extend(s, rows, lens, add):
    """Pages for the positions [len, len + add) of the rows: missing ones are taken from the stack in (row, page) order;
    a page with other owners is replaced by an own copy, except for the last of its owners in the batch if all are in it."""
    P = s["case"]["page"]
    rows, first, end = rows.long(), lens.long() // P, (lens + add).long()
    g = first[:, None] + torch.arange(-(-s["case"]["len"] // P) + 1, device="cuda")[None, :]
    need = g * P < end[:, None]
    g = g.clamp(max=s["tables"].shape[1] - 1)
    at = rows[:, None].expand_as(g)
    e = s["tables"][at, g].long()
    hole = need & (e < 0)
    shared = need & (e >= 0) & (s["shares"][e.clamp(min=0)] > 0)
    order = torch.arange(e.numel(), device="cuda").view(e.shape)
    count = torch.zeros_like(s["shares"]).index_add_(0, e[shared], torch.ones_like(e[shared], dtype=torch.int32))
    last = torch.full((s["shares"].numel(),), -1, device="cuda").scatter_reduce_(0, e[shared], order[shared], "amax")
    keeps = shared & (count == s["shares"] + 1)[e.clamp(min=0)] & (last[e.clamp(min=0)] == order)
    take = hole | (shared & ~keeps)
    new = s["ids"][s["n_free"].long() - torch.arange(1, int(take.sum()) + 1, device="cuda")]
    s["n_free"] -= new.numel()
    old = e[take]
    kept = ((g * P < lens[:, None]) & shared)[take]                   # pages that hold tokens of the row
    lose = e[shared & ~keeps]
    s["shares"].index_add_(0, lose, torch.full_like(lose, -1, dtype=torch.int32))
    s["tables"][at[take], g[take]] = new
    a, b = old[kept], new[kept].long()
    s["k"][:, b] = s["k"][:, a]
    s["v"][:, b] = s["v"][:, a]


def _compact(s):
    """The used pages with the highest ids move, in order, into the free ids below the number of used pages."""
    blocks = s["shares"].numel()
    n_free = int(s["n_free"])
    used = torch.ones(blocks, dtype=torch.bool, device="cuda")
    used[s["ids"][:n_free].long()] = False
    top = blocks - n_free
    to = (~used[:top]).nonzero()[:, 0]
    frm = used[top:].nonzero()[:, 0] + top
    new = torch.arange(blocks, dtype=torch.int32, device="cuda")
    new[frm] = to.int()
    t = s["tables"]
    t.copy_(torch.where(t >= 0, new[t.long().clamp(min=0)], t))
    s["shares"][to] = s["shares"][frm]
    s["shares"][frm] = 0
    s["ids"][:n_free] = torch.arange(blocks - 1, top - 1, -1, dtype=torch.int32, device="cuda")
    s["k"][:, to] = s["k"][:, frm]
    s["v"][:, to] = s["v"][:, frm]


def _run_pages(s):
    c, turn = s["case"], s["turn"]
    kind = c["kind"]
    s["turn"] = (turn + 1) % (2 if kind == "beams" else 8)
    if own:
        p = s["pages"]
        if kind == "beams":
            p.fork(s["src"][turn], s["dst"][turn])
            p.free(s["old"][turn])
            p.extend(s["dst"][turn], s["lens"], 1)
        elif kind == "samples":
            p.fork(s["src"], s["dst"])
            p.extend(s["all"], s["lens"], 1)
            p.free(s["dst"])
        else:
            p.free(s["gone"][turn])
            p.compact()
            p.extend(s["gone"][turn], s["none"], s["full"])
        return s["k"], s["v"], s["tables"], p.shares, p.ids, p.n_free
    if kind == "beams":
        _fork(s, s["src"][turn], s["dst"][turn])
        _free(s, s["old"][turn])
        _extend(s, s["dst"][turn], s["lens"], 1)
    elif kind == "samples":
        _fork(s, s["src"], s["dst"])
        _extend(s, s["all"], s["lens"], 1)
        _free(s, s["dst"])
    else:
        _free(s, s["gone"][turn])
        _compact(s)
        _extend(s, s["gone"][turn], s["none"], s["full"])
    return s["k"], s["v"], s["tables"], s["shares"], s["ids"], s["n_free"]


def run(state):
    return {"qkv": _run_qkv, "attend": _run_attend, "pages": _run_pages}[state["case"]["op"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(case):
    c = case
    size = 4 if c["type"] == "f32" else 2
    if c["op"] == "qkv":
        heads = c["H"] * c["grp"] + 2 * c["H"]
        elems = c["n"] * heads * c["D"]
        return {"bytes": 2 * size * elems + 8 * c["n"], "flops": 8 * elems}
    if c["op"] == "attend":
        live = sum(min(x, c["window"]) if c["window"] else x for x in _lens(c))
        rows = c["n"] * c["H"] * c["grp"] * c["D"]
        io = 4 if c["io"] == "f32" else 2
        return {"bytes": 4 * live * c["H"] * c["D"] + 2 * io * rows + 4 * (live // c["page"] + c["n"]),
                "flops": 4 * live * c["H"] * c["grp"] * c["D"]}
    per, part = _share(c)
    block = 2 * c["layers"] * c["page"] * c["H"] * c["D"] * 2
    if c["kind"] == "beams":
        moved, entries = (c["n"] // 2 if part else 0), 6 * c["n"] * per
    elif c["kind"] == "samples":
        moved, entries = (c["n"] - 1 if part else 0), 6 * c["n"] * per
    else:
        gone = c["n"] // 8 * per
        moved = gone - gone * gone // (c["n"] * per)                  # of the freed ids, those below the used ones' number
        entries = 2 * c["n"] * per + 2 * c["blocks"]
    return {"bytes": 2 * moved * block + 4 * entries, "flops": entries}


# ---- the results in 64 bits -----------------------------------------------------------------------------------------

def exact(case, seed):
    c = case
    if c["op"] == "pages":
        return None
    s = prepare(c, seed)
    if c["op"] == "attend":
        outs = []
        for i, length in enumerate(_lens(c)):
            lo = max(0, length - c["window"]) if c["window"] else 0
            t = torch.arange(lo, length, device="cuda")
            page = s["tables"][i, t // c["page"]].long()
            k, v = (s[x][0][page, t % c["page"]].double() for x in ("k", "v"))
            q = s["q"][i].double().view(c["H"], c["grp"], c["D"])
            w = torch.softmax(torch.einsum("hgd,thd->hgt", q, k) * s["scale"], -1)
            outs.append(torch.einsum("hgt,thd->hgd", w, v).reshape(-1, c["D"]))
        return torch.stack(outs)
    freq, amp = _inv_freq(c)
    ang = s["pos"].double()[:, None] * torch.tensor(freq, device="cuda")[None, :]
    turn = torch.polar(torch.full_like(ang, amp), ang)[:, None]
    res = []
    for x, w in zip(_heads(s)[:2], (s["wq"], s["wk"])):
        x = x.double()
        if w is not None:
            x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
        n = c["n_rot"]
        a, b = (x[..., : n // 2], x[..., n // 2: n]) if c["layout"] == "half" else (x[..., 0:n:2], x[..., 1:n:2])
        z = torch.complex(a.contiguous(), b.contiguous()) * turn
        y = x.clone()
        if c["layout"] == "half":
            y[..., : n // 2], y[..., n // 2: n] = z.real, z.imag
        else:
            y[..., 0:n:2], y[..., 1:n:2] = z.real, z.imag
        res.append(y)
    v = _heads(s)[2].double()
    if c["to"] == "rows":
        return res[0], res[1], v
    k_all, v_all = s["k"].double(), s["v"].double()
    pos = s["pos"].long()
    page = s["tables"][s["rows"].long(), pos // c["page"]].long()
    k_all[0, page, pos % c["page"]] = res[1]
    v_all[0, page, pos % c["page"]] = v
    return res[0], k_all, v_all
