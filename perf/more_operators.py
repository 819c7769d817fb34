"""What the operators of a step with several new tokens a sequence, and of attention to a part of a long context, are
measured on: the maps that such a step needs (which token is whose, where it goes), attention of a tree of drafted tokens
over the paged 16-bit cache, the move of the accepted ones to their places, bounds of every page's keys, and attention to
the pages that these bounds choose for a query.

listed() and draw() give cases, prepare() what a program has in hand before the call, run() one pass: in plain torch
operations in 32 bits (64 where a choice hangs on a border), or, where `own` is true, through kv16 (the framework's own
calls). exact() states the computed results in 64 bits.
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _kv16():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sj-kvarn-codec_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import kv16
    return kv16


# ---- the cases ------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one chat whose next tokens are drafted as a tree of 8: a call's latency
        dict(name="tree-1x611-8", op="tree", n=1, lo=611, hi=611, spread=1, nodes=8, ragged=False, tree="tree", D=128, H=8,
             grp=4, page=16, type="bf16", window=0),
        # a pool of long contexts between 8K and 64K, 16 drafted tokens each
        dict(name="tree-32x8k-64k-16", op="tree", n=32, lo=8192, hi=65536, spread=3, nodes=16, ragged=False, tree="tree",
             D=256, H=4, grp=4, page=128, type="bf16", window=0),
        # one sequence of 100,000 tokens, a wide tree: 256 query rows for every key
        dict(name="tree-1x100000-64", op="tree", n=1, lo=100000, hi=100000, spread=2, nodes=64, ragged=False, tree="tree",
             D=128, H=8, grp=4, page=128, type="f16", window=0),
        # many short chats on a sliding-window layer with a cache per head, pieces of prompts (0 to 33 tokens) in a row
        dict(name="tree-64-pieces", op="tree", n=64, lo=0, hi=2048, spread=5, nodes=33, ragged=True, tree="chain", D=64,
             H=24, grp=1, page=24, type="bf16", window=512),
        # one chat's accepted path of up to 5 tokens to its place in 16 layers: a launch
        dict(name="keep-1x5", op="keep", n=1, len=1003, nodes=8, width=5, spread=1, layers=16, page=16, H=8, D=128, type="bf16"),
        # the accepted paths of 64 sequences, up to 9 of 64 drafted tokens, 32 layers
        dict(name="keep-64x9", op="keep", n=64, len=2000, nodes=64, width=9, spread=2, layers=32, page=128, H=4, D=256, type="f16"),
        # maps of one chat's tree
        dict(name="maps-1x8", op="maps", n=1, far=2000, add=8, spread=1, tree="tree", page=16),
        # maps of 512 requests that bring between 1 and 60 tokens each
        dict(name="maps-512x60", op="maps", n=512, far=65536, add=60, spread=2, tree="chain", page=16),
        # a decode step of 64 sequences: the newest page's bounds in 4 layers
        dict(name="bounds-64-step", op="bounds", n=64, far=16384, add=1, spread=1, layers=4, page=16, H=8, D=128, type="bf16"),
        # bounds of all pages of a prompt of 32,700 tokens
        dict(name="bounds-32700-prompt", op="bounds", n=1, far=0, add=32700, spread=2, layers=2, page=64, H=4, D=256, type="f16"),
        # one sequence of 100,000 tokens: 128 of its 6,250 pages chosen for every KV head
        dict(name="sparse-1x100000-128", op="sparse", n=1, lo=100000, hi=100000, spread=1, D=128, H=8, grp=4, page=16,
             budget=128, type="bf16", io="bf16"),
        # a pool of long contexts between 8K and 64K: 16 of up to 512 pages for every KV head
        dict(name="sparse-32x8k-64k-16", op="sparse", n=32, lo=8192, hi=65536, spread=3, D=256, H=4, grp=4, page=128,
             budget=16, type="bf16", io="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["tree", "tree", "keep", "maps", "bounds", "sparse", "sparse"])
        D, H, typ = rng.choice([64, 96, 128, 256]), rng.choice([1, 2, 4, 8]), rng.choice(["f16", "bf16"])
        page, spread = rng.choice([16, 24, 32, 64, 128]), rng.randrange(1, 1000)
        if op == "tree":
            n, hi = _log(rng, 1, 128), _log(rng, 1, 100000)
            lo, grp, nodes = rng.choice([0, min(hi, _log(rng, 1, hi))]), rng.choice([1, 2, 3, 4, 7, 8, 16]), _log(rng, 1, 64)
            c = dict(op=op, n=n, lo=lo, hi=hi, spread=spread, nodes=nodes, ragged=rng.random() < 0.5,
                     tree=rng.choice(["tree", "tree", "chain"]), D=D, H=H, grp=grp, page=rng.choice([page, 1, 5]), type=typ,
                     window=rng.choice([0, 0, 0, _log(rng, 1, hi)]))
            w = work(c)
            if n * hi * H * D > 1.1e9 or w["bytes"] > 3.5e9 or w["flops"] > 1.0e11 or n * hi * H * grp * nodes > 6e8:
                continue
        elif op == "keep":
            nodes = _log(rng, 1, 64)
            c = dict(op=op, n=_log(rng, 1, 128), len=_log(rng, 1, 4000), nodes=nodes, width=_log(rng, 1, min(nodes, 12)),
                     spread=spread, layers=_log(rng, 1, 32), page=page, H=H, D=D, type=typ)
            if work(c)["bytes"] > 6.0e7:
                continue
        elif op == "maps":
            c = dict(op=op, n=_log(rng, 1, 512), far=_log(rng, 64, 100000), add=_log(rng, 1, 60), spread=spread,
                     tree=rng.choice(["tree", "chain"]), page=page)
        elif op == "bounds":
            add = rng.choice([1, 1, _log(rng, 1, 30000)])
            c = dict(op=op, n=_log(rng, 1, 64) if add == 1 else _log(rng, 1, 8), far=rng.choice([0, _log(rng, 1, 16384)]), add=add,
                     spread=spread, layers=_log(rng, 1, 4), page=page, H=H, D=D, type=typ)
            if work(c)["bytes"] > 1.4e8 or c["n"] * (c["far"] + add) * H * D * c["layers"] > 1e9:
                continue
        else:
            n, hi = _log(rng, 1, 64), _log(rng, 1, 100000)
            c = dict(op=op, n=n, lo=rng.choice([0, min(hi, _log(rng, 1, hi))]), hi=hi, spread=spread, D=D, H=H,
                     grp=rng.choice([1, 2, 3, 4, 7, 8, 16]), page=page, budget=_log(rng, 3, 160), type=typ, io=rng.choice([typ, typ, "f32"]))
            if n * hi * H * D > 1.1e9 or work(c)["bytes"] > 3.0e8:
                continue
        return c


def _lens(c):
    """The lengths of a case's sequences: between lo and hi, spread over their logarithm where that is wide."""
    if c["n"] == 1:
        return [c["hi"]]
    r = random.Random(c["spread"])
    wide = c["hi"] > 10 * c["lo"]
    lens = [_log(r, max(c["lo"], 1), c["hi"]) if wide else r.randint(c["lo"], c["hi"]) for _ in range(c["n"])]
    lens[0], lens[-1] = c["lo"], c["hi"]
    return lens


def _counts(c):
    """Drafted tokens of each sequence of a tree case."""
    if not c["ragged"] or c["n"] == 1:
        return [c["nodes"]] * c["n"]
    r = random.Random(c["spread"] + 1)
    n = [r.randint(0, c["nodes"]) for _ in range(c["n"])]
    n[-1] = c["nodes"]
    return n


def _tree(r, n):
    """Masks of a random tree of n drafted tokens: token j sees itself and what its parent, an earlier one, sees."""
    masks = []
    for j in range(n):
        masks.append((masks[r.randrange(j)] if j else 0) | 1 << j)
    return masks


def _signed(masks):
    return [m - (1 << 64) if m >= 1 << 63 else m for m in masks]


def _paths(c):
    """Accepted tokens of each sequence of a keep case: ascending ones of the drafted, from 0 to width many."""
    r = random.Random(c["spread"])
    paths = [sorted(r.sample(range(c["nodes"]), r.randint(0, c["width"]))) for _ in range(c["n"])]
    paths[-1] = sorted(r.sample(range(c["nodes"]), c["width"]))
    return paths


def _spans(c):
    """(length, new tokens) of each sequence of a maps or bounds case."""
    r = random.Random(c["spread"])
    if c["n"] == 1:
        return [(c["far"], c["add"])]
    if c["op"] == "bounds":
        return [(r.randint(0, c["far"]), c["add"]) for _ in range(c["n"])]
    return [(r.randint(0, c["far"]), r.randint(1, c["add"])) for _ in range(c["n"])]


# ---- what a program has in hand ------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(shape, dtype, g):
    return torch.randn(shape, dtype=dtype, device="cuda", generator=g)


def _ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def _tables(lens, P, g, spare=0):
    """Table rows for sequences of these lengths over pages in random order, and the number of pages."""
    per = [-(-x // P) for x in lens]
    stride, pages = max(max(per), 1), max(sum(per), 1) + spare
    perm = torch.randperm(pages, generator=g, device="cuda").int()
    at = _ints([0] + per[:-1], torch.int64).cumsum(0)
    idx = torch.arange(stride, device="cuda")
    have = idx[None, :] < _ints(per)[:, None]
    return torch.where(have, perm[(at[:, None] + idx[None, :]).clamp(max=pages - 1)], torch.full((), -1, dtype=torch.int32, device="cuda")), pages


def _cache(s, c, lens, g, layers=1):
    """K and V pages: channels of unlike size, and pages whose keys lean somewhere, as neighbouring tokens' do."""
    T, P, H, D = TYPES[c["type"]], c["page"], c["H"], c["D"]
    s["tables"], pages = _tables(lens, P, g)
    s["k"] = _normal((layers, pages, P, H, D), T, g)
    s["k"] += 0.7 * _normal((layers, pages, 1, H, D), T, g)
    s["k"] *= (0.5 * torch.randn((H, D), device="cuda", generator=g)).exp().to(T)
    s["v"] = _normal((layers, pages, P, H, D), T, g)


def _prepare_tree(c, seed):
    g = _gen(seed)
    lens, counts, D = _lens(c), _counts(c), c["D"]
    s = dict(case=c, scale=1.0 / math.sqrt(D))
    _cache(s, c, [a + b for a, b in zip(lens, counts)], g)
    s["lens"] = _ints(lens)
    s["first"] = _ints([0] + counts, torch.int64).cumsum(0).int()
    n = sum(counts)
    r = random.Random(c["spread"] + 2 + seed)
    s["masks"] = _ints([m for x in counts for m in _signed(_tree(r, x))], torch.int64) if c["tree"] == "tree" else None
    s["q"] = _normal((n, c["H"] * c["grp"], D), TYPES[c["type"]], g)
    s["out"] = torch.empty_like(s["q"])
    if own:
        s["cache"] = _kv16().Cache(s["k"], s["v"], s["tables"])
    return s


def _prepare_keep(c, seed):
    g = _gen(seed)
    s = dict(case=c)
    _cache(s, c, [c["len"] + c["nodes"]] * c["n"], g, c["layers"])
    paths = _paths(c)
    s["lens"] = _ints([c["len"]] * c["n"])
    s["path"] = _ints([p + [0] * (c["width"] - len(p)) for p in paths])
    s["count"] = _ints([len(p) for p in paths])
    s["new"] = torch.empty_like(s["lens"])
    if own:
        s["cache"] = _kv16().Cache(s["k"], s["v"], s["tables"])
    return s


def _prepare_maps(c, seed):
    g = _gen(seed)
    spans = _spans(c)
    s = dict(case=c)
    s["tables"], pages = _tables([a + b for a, b in spans], c["page"], g)
    s["lens"], s["add"] = _ints([a for a, _ in spans]), _ints([b for _, b in spans])
    s["n_tok"] = sum(b for _, b in spans) + 5                         # a step's room is rounded up: the rest is padding
    r = random.Random(c["spread"] + 2 + seed)
    s["masks"] = None
    if c["tree"] == "tree":
        s["masks"] = _ints([m for _, b in spans for m in _signed(_tree(r, b))] + [0] * 5, torch.int64)
    if own:
        kv16 = _kv16()
        k = torch.zeros((1, pages, c["page"], 1, 64), dtype=torch.bfloat16, device="cuda")
        s["call"] = kv16.Maps(kv16.Cache(k, torch.zeros_like(k), s["tables"]), c["n"], s["n_tok"])
    return s


def _prepare_bounds(c, seed):
    g = _gen(seed)
    spans = _spans(c)
    s = dict(case=c)
    _cache(s, c, [a + b for a, b in spans], g, c["layers"])
    s["from"], s["to"] = _ints([a for a, _ in spans]), _ints([a + b for a, b in spans])
    s["pages"] = (max(a for a, _ in spans) % c["page"] + c["add"]) // c["page"] + 2    # of a sequence, at most
    s["bounds"] = torch.zeros((c["layers"], s["k"].shape[1], 2, c["H"], c["D"]), dtype=s["k"].dtype, device="cuda")
    if own:
        kv16 = _kv16()
        s["call"] = kv16.Blocks(kv16.Cache(s["k"], s["v"], s["tables"]), bounds=s["bounds"])
    return s


def _prepare_sparse(c, seed):
    g = _gen(seed)
    lens, D = _lens(c), c["D"]
    s = dict(case=c, scale=1.0 / math.sqrt(D))
    _cache(s, c, lens, g)
    s["lens"] = _ints(lens)
    s["bounds"] = torch.stack((s["k"].amin(2), s["k"].amax(2)), 2).contiguous()
    s["q"] = _normal((c["n"], c["H"] * c["grp"], D), torch.float32, g).to(TYPES[c["io"]])
    s["out"] = torch.empty_like(s["q"])
    if own:
        kv16 = _kv16()
        s["call"] = kv16.Blocks(kv16.Cache(s["k"], s["v"], s["tables"]), bounds=s["bounds"])
    return s


def prepare(case, seed):
    return {"tree": _prepare_tree, "keep": _prepare_keep, "maps": _prepare_maps, "bounds": _prepare_bounds,
            "sparse": _prepare_sparse}[case["op"]](case, seed)


# ---- one pass -------------------------------------------------------------------------------------------------------

def _owner(first, n_tok):
    """Of every token its sequence (len(first) - 1: padding) and its number there."""
    t = torch.arange(n_tok, device="cuda")
    i = torch.searchsorted(first, t.int(), right=True) - 1
    return i, t - first[i].long()


def _bits(masks, n):
    return (masks[:, None] >> torch.arange(n, device="cuda")[None, :]) & 1


def _run_tree(s):
    """A token sees the committed positions [0, len) and those drafted ones (at len + k) whose bit k its mask has (without
    masks: itself and those before it); with a window only the last `window` of all these."""
    c = s["case"]
    if own:
        return s["cache"].attend_tree(0, s["q"], s["lens"], s["masks"], s["scale"], first=s["first"], nodes=c["nodes"],
                                      window=c["window"], out=s["out"])
    H, grp, D, N, P, W = c["H"], c["grp"], c["D"], c["nodes"], c["page"], c["window"]
    n_tok = s["q"].shape[0]
    i, j = _owner(s["first"], n_tok)
    k = torch.arange(N, device="cuda")[None, :]
    sees = _bits(s["masks"], N) == 1 if s["masks"] is not None else k <= j[:, None]
    tree = torch.zeros((c["n"], N, N), dtype=torch.bool, device="cuda")        # by sequence and number
    tree[i, j] = sees
    q = torch.zeros((c["n"], N, H * grp, D), device="cuda")
    q[i, j] = s["q"].float() * s["scale"]
    q = q.view(c["n"], N, H, grp, D).permute(0, 2, 1, 3, 4).reshape(c["n"], H, N * grp, D)
    page = s["tables"].long().clamp(min=0)
    keys = s["k"][0][page].view(c["n"], -1, H, D)
    t = torch.arange(keys.shape[1], device="cuda")
    lens = s["lens"].long()
    node = t[None, :] - lens[:, None]                                          # which drafted token a position is
    live = torch.gather(tree, 2, node.clamp(0, N - 1)[:, None, :].expand(-1, N, -1)) & ((node >= 0) & (node < N))[:, None, :]
    live |= (node < 0)[:, None, :]
    if W:
        left = live.long().flip(-1).cumsum(-1).flip(-1)                        # live positions from here on
        live &= left <= W
    p = q @ keys.float().permute(0, 2, 3, 1)
    del keys
    dead = (~live)[:, None, :, None, :].expand(-1, 1, -1, grp, -1).reshape(c["n"], 1, N * grp, -1)
    p = p.masked_fill_(dead, float("-inf"))
    p = p.sub_(p.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp(min=1e-30))
    v = s["v"][0][page].view(c["n"], -1, H, D)
    out = p @ v.float().permute(0, 2, 1, 3)
    out = out.view(c["n"], H, N, grp, D).permute(0, 2, 1, 3, 4).reshape(c["n"], N, H * grp, D)
    s["out"].copy_(out[i, j])
    return s["out"]


def _run_keep(s):
    """Rows of the accepted tokens, path[i][0], path[i][1], ... of sequence i, to the positions len, len + 1, ..."""
    c = s["case"]
    if own:
        s["cache"].keep(s["lens"], s["path"], s["count"], new_lens=s["new"])
        return s["k"], s["v"], s["new"]
    P, w = c["page"], c["width"]
    lens = s["lens"].long()[:, None]
    j = torch.arange(w, device="cuda")[None, :]
    on = j < s["count"][:, None]
    frm = (lens + s["path"].long()).clamp(max=s["tables"].shape[1] * P - 1)
    frm = torch.where(on, frm, lens + j)                                       # (a row to itself where nothing moves)
    row = torch.arange(c["n"], device="cuda")[:, None]
    a, b = s["tables"][row, frm // P].long(), s["tables"][row, (lens + j) // P].long()
    for x in (s["k"], s["v"]):
        x[:, b, (lens + j) % P] = x[:, a, frm % P]
    s["new"].copy_(s["lens"] + s["count"])
    return s["k"], s["v"], s["new"]


def _run_maps(s):
    """first: where each sequence's tokens begin; of every token: its table row, rotary position (length and the number of
    other drafted tokens it sees), cache position (-1: padding) and slot (page * page tokens + place, -1: none)."""
    c = s["case"]
    if own:
        m = s["call"](s["lens"], s["add"], masks=s["masks"])
        return m.first, m.rows, m.pos, m.at, m.slots
    first = torch.cat((torch.zeros(1, dtype=torch.int64, device="cuda"), s["add"].long().cumsum(0))).int()
    i, j = _owner(first, s["n_tok"])
    on = i < c["n"]
    i = i.clamp(max=c["n"] - 1)
    lens = s["lens"].long()[i]
    at = lens + j
    pos = at
    if s["masks"] is not None:
        pos = lens + _bits(s["masks"], 64).sum(-1) - (s["masks"] >> j.clamp(max=63) & 1)
    at = torch.where(on, at, -1)
    slot = s["tables"][i, at.clamp(min=0) // c["page"]].long() * c["page"] + at % c["page"]
    return (first, torch.where(on, i, 0).int(), torch.where(on, pos, -1).int(), at.int(), torch.where(on, slot, -1))


def _run_bounds(s):
    """Smallest and largest key of every channel, over the tokens that pages with positions in [from, to) hold before
    `to`."""
    c = s["case"]
    if own:
        s["call"].update(s["from"], s["to"])
        return s["bounds"]
    P = c["page"]
    g = (s["from"].long() // P)[:, None] + torch.arange(s["pages"], device="cuda")[None, :]
    end = s["to"].long()[:, None]
    on = g * P < end
    i, at = on.nonzero(as_tuple=True)
    g = g[i, at]
    ids = s["tables"][i, g].long()
    live = (g[:, None] * P + torch.arange(P, device="cuda")[None, :] < s["to"].long()[i][:, None])[None, :, :, None, None]
    k = s["k"][:, ids].float()
    s["bounds"][:, ids, 0] = k.masked_fill(~live, float("inf")).amin(2).to(s["bounds"].dtype)
    s["bounds"][:, ids, 1] = k.masked_fill(~live, float("-inf")).amax(2).to(s["bounds"].dtype)
    return s["bounds"]


def _run_sparse(s):
    """For every KV head the first page, the newest one and those pages whose bound on the sum of its query heads' scores
    is largest (ties to the lower number), `budget` in all, in ascending order; attention over their tokens."""
    c = s["case"]
    if own:
        blocks, _ = s["call"].select(0, s["q"], s["lens"], c["budget"])
        s["call"].attend(0, s["q"], s["lens"], blocks, s["scale"], out=s["out"])
        return blocks, s["out"]
    n, H, grp, D, P, B = c["n"], c["H"], c["grp"], c["D"], c["page"], c["budget"]
    page = s["tables"].long().clamp(min=0)
    stride = page.shape[1]
    q = s["q"].view(n, H, grp, D)
    up, down = q.double().clamp(min=0).sum(2), q.double().clamp(max=0).sum(2)  # [n][H][D]
    score = torch.empty((n, H, stride), dtype=torch.float64, device="cuda")
    for i in range(n):
        b = s["bounds"][0][page[i]].double()                                   # [stride][2][H][D]
        score[i] = (torch.einsum("shd,hd->hs", b[:, 0], down[i]) + torch.einsum("shd,hd->hs", b[:, 1], up[i]))
    g = torch.arange(stride, device="cuda")[None, :]
    blocks = (s["lens"].long()[:, None] + P - 1) // P
    score = score.masked_fill(((g == 0) | (g == blocks - 1))[:, None, :], float("inf"))
    score = score.masked_fill((g >= blocks)[:, None, :], float("-inf"))
    order = score.argsort(dim=-1, descending=True, stable=True)[:, :, :B]
    order = torch.where(order < blocks[:, :, None], order, stride).sort(-1).values      # ascending, missing ones last
    pick = torch.full((n, H, B), -1, dtype=torch.int32, device="cuda")
    pick[:, :, : order.shape[2]] = torch.where(order < stride, order, -1).int()
    ids = page[torch.arange(n, device="cuda")[:, None, None], pick.long().clamp(min=0)]
    head = torch.arange(H, device="cuda")[None, :, None]
    k = s["k"][0][ids, :, head].reshape(n, H, B * P, D)
    t = (pick.long()[..., None] * P + torch.arange(P, device="cuda")).view(n, H, B * P)
    dead = (pick < 0)[..., None].expand(-1, -1, -1, P).reshape(n, H, B * P) | (t >= s["lens"].long()[:, None, None])
    p = (q.float() * s["scale"]) @ k.float().transpose(2, 3)
    p = p.masked_fill(dead[:, :, None, :], float("-inf"))
    p = (p - p.amax(-1, keepdim=True).clamp(min=-1e30)).exp()
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    v = s["v"][0][ids, :, head].reshape(n, H, B * P, D)
    s["out"].copy_((p @ v.float()).view(n, H * grp, D))
    return pick, s["out"]


def run(state):
    return {"tree": _run_tree, "keep": _run_keep, "maps": _run_maps, "bounds": _run_bounds,
            "sparse": _run_sparse}[state["case"]["op"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "tree":
        lens, counts, W = _lens(c), _counts(c), c["window"]
        pos = sum((min(a, W + b) if W else a) + b for a, b in zip(lens, counts) if b)       # positions that some token sees
        seen = sum(b * (min(a + b // 2 + 1, W) if W else a + b // 2 + 1) for a, b in zip(lens, counts))
        rows = sum(counts) * c["H"] * c["grp"] * c["D"]
        return {"bytes": 4 * pos * c["H"] * c["D"] + 4 * rows + 4 * (pos // c["page"] + 3 * c["n"]) + 8 * sum(counts),
                "flops": 4 * seen * c["H"] * c["grp"] * c["D"]}
    if c["op"] == "keep":
        moved = sum(p != j for path in _paths(c) for j, p in enumerate(path))
        return {"bytes": 8 * moved * c["layers"] * c["H"] * c["D"] + 4 * c["n"] * (c["width"] + 3), "flops": c["n"]}
    if c["op"] == "maps":
        t = sum(b for _, b in _spans(c))
        return {"bytes": (20 + (8 if c["tree"] == "tree" else 0)) * t + 4 * (t // c["page"] + 4 * c["n"]), "flops": 4 * t}
    if c["op"] == "bounds":
        toks = sum(a + b - a // c["page"] * c["page"] for a, b in _spans(c))
        pages = sum((a + b - 1) // c["page"] - a // c["page"] + 1 for a, b in _spans(c))
        width = 2 * c["layers"] * c["H"] * c["D"]
        return {"bytes": width * (toks + 2 * pages) + 4 * (pages + 2 * c["n"]), "flops": width * toks}
    pages = [-(-x // c["page"]) for x in _lens(c)]
    scored = sum(x for x in pages if x > c["budget"])
    kept = sum(min(x, min(b, c["budget"]) * c["page"]) for x, b in zip(_lens(c), pages))
    rows = c["n"] * c["H"] * c["grp"] * c["D"]
    return {"bytes": 4 * scored * c["H"] * c["D"] + 4 * kept * c["H"] * c["D"] + 2 * rows * (4 if c["io"] == "f32" else 2) +
            4 * (scored + c["n"] * (1 + c["H"] * c["budget"])),
            "flops": 4 * scored * c["H"] * c["D"] + 4 * kept * c["H"] * c["grp"] * c["D"]}


# ---- the results in 64 bits -----------------------------------------------------------------------------------------

def _visible(c, length, masks, j):
    """Positions that drafted token j of a sequence sees, in order."""
    node = [k for k in range(len(masks)) if masks[j] >> k & 1]
    drop = max(0, length + len(node) - c["window"]) if c["window"] else 0
    return min(drop, length), [length + k for k in node[max(0, drop - length):]]


def _exact_tree(c, s):
    outs, at = [], 0
    for i, (length, n) in enumerate(zip(_lens(c), _counts(c))):
        if n == 0:
            continue
        masks = [(1 << (j + 1)) - 1 for j in range(n)] if s["masks"] is None else s["masks"][at:at + n].tolist()
        t = torch.arange(length + n, device="cuda")
        live = torch.zeros((n, length + n), dtype=torch.bool, device="cuda")
        for j in range(n):
            lo, nodes = _visible(c, length, masks, j)
            live[j, lo:length] = True
            live[j, nodes] = True
        page = s["tables"][i, t // c["page"]].long()
        q = s["q"][at:at + n].double().view(n, c["H"], c["grp"], c["D"])
        out = torch.empty_like(q)
        for h in range(c["H"]):                                                # a head at a time: 64-bit scores are large
            k, v = (s[x][0][page, t % c["page"], h].double() for x in ("k", "v"))
            w = torch.einsum("jgd,td->jgt", q[:, h], k) * s["scale"]
            w = torch.softmax(w.masked_fill(~live[:, None, :], -math.inf), -1)
            out[:, h] = torch.einsum("jgt,td->jgd", w, v)
        outs.append(out.reshape(n, -1, c["D"]))
        at += n
    return torch.cat(outs)


def _exact_sparse(c, s):
    P, H, B = c["page"], c["H"], c["budget"]
    picks, outs = [], []
    for i, length in enumerate(_lens(c)):
        blocks = -(-length // P)
        ids = s["tables"][i, :blocks].long()
        q = s["q"][i].double().view(H, c["grp"], -1)
        out = torch.zeros_like(q)
        for h in range(H):
            lo, hi = s["bounds"][0, ids, 0, h].double(), s["bounds"][0, ids, 1, h].double()
            bound = sum(torch.maximum(lo * x, hi * x).sum(-1) for x in q[h])
            mid = range(1, blocks - 1)
            score = bound.tolist()
            best = sorted(mid, key=lambda b: (-score[b], b))[: max(0, B - min(blocks, 2))]
            pick = sorted(set(best) | ({0, blocks - 1} if blocks else set()))
            picks.append(pick + [-1] * (B - len(pick)))
            t = torch.cat([torch.arange(b * P, min((b + 1) * P, length)) for b in pick]).cuda() if pick else None
            if t is not None:
                k, v = (s[x][0][s["tables"][i, t // P].long(), t % P, h].double() for x in ("k", "v"))
                out[h] = torch.softmax(q[h] @ k.T * s["scale"], -1) @ v
        outs.append(out.reshape(-1, c["D"]))
    return _ints(picks).view(c["n"], H, B), torch.stack(outs)


def exact(case, seed):
    c = case
    if c["op"] in ("keep", "maps", "bounds"):                                  # copies, whole numbers and inputs' own values
        return None
    s = prepare(c, seed)
    return _exact_tree(c, s) if c["op"] == "tree" else _exact_sparse(c, s)
