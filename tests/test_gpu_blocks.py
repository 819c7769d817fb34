"""Attention to chosen pages: sjk_kv16_bounds (exact), sjk_kv16_select against a plain choice in 64 bits (exact: the products
are exact in both, and sums of 512 in 64 bits are off by 2^-43 of their terms, where random scores lie 2^-30 of them apart), and
sjk_kv16_attend_blocks against the definition in 64 bits.

Error bound of an output element y, with A the same attention over |V|: u |y| for the rounding to the output type, (p + 2 e) A
for the rounded weights and the scores behind them: p = 2^-16 (bf16 cache) or 2^-21 (f16), e = 2^-20 (1 + max_t scale sum_d
|q_d k_td|) in units of ln 2, as for the attention over all positions, whose kernel this is."""
import math
import random

import pytest

import kv16
import sjk

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    import build
    build.build()
    import torch
    assert torch.cuda.is_available()
    return torch


def _dt(T, name):
    return {"f32": T.float32, "f16": T.float16, "bf16": T.bfloat16}[name]


def _ints(T, x):
    return T.tensor(x, dtype=T.int32, device="cuda")


def _cache(T, lens, page, H, D, dtype, seed=0, layers=1, junk=math.nan):
    """Live positions are normal values that lean to one side page by page; other slots are junk."""
    g = T.Generator(device="cuda")
    g.manual_seed(seed)
    n, stride = len(lens), max(1, max(-(-x // page) for x in lens)) + 1
    pages = sum(-(-x // page) for x in lens) + 3
    cache = kv16.Cache.alloc(layers, pages, page, H, D, dtype, n, stride)
    cache.k.fill_(junk)
    cache.v.fill_(junk)
    perm = T.randperm(pages, generator=g, device="cuda")
    at = 0
    for i, x in enumerate(lens):
        per = -(-x // page)
        ids = perm[at:at + per]
        at += per
        cache.tables[i, :per] = ids.int()
        t = T.arange(x, device="cuda")
        lean = T.randn((layers, per, H, D), device="cuda", generator=g)
        cache.k[:, ids[t // page], t % page] = (T.randn((layers, x, H, D), device="cuda", generator=g) + lean[:, t // page]).to(dtype)
        cache.v[:, ids[t // page], t % page] = T.randn((layers, x, H, D), device="cuda", generator=g).to(dtype)
    return cache, g


def _bounds(T, cache, row, end, layer=0):
    """[pages][2][H][D] of a row's pages, over its positions before `end`."""
    P = cache.page_tokens
    out = []
    for b in range(-(-end // P)):
        k = cache.k[layer, int(cache.tables[row, b]), : min(P, end - b * P)]
        out.append(T.stack((k.amin(0), k.amax(0))))
    return T.stack(out) if out else T.zeros((0, 2, *cache.k.shape[3:]), dtype=cache.k.dtype, device="cuda")


def _choose(T, bounds, q, have, budget, sink, recent):
    """bounds [pages][2][H][D], q [heads][D]; have: which pages exist. A list per KV head."""
    n, H = bounds.shape[0], bounds.shape[2]
    q = q.double().view(H, -1, q.shape[-1])
    lo, hi = bounds[:, 0].double(), bounds[:, 1].double()
    score = sum(T.maximum(lo * q[None, :, g], hi * q[None, :, g]).sum(-1) for g in range(q.shape[1])).T.tolist()
    out = []
    for h in range(H):
        must = [b for b in range(n) if have[b] and (n <= budget or b < sink or b >= n - recent)]
        rest = sorted((b for b in range(n) if have[b] and b not in must), key=lambda b: (-score[h][b], b))
        pick = sorted(must + rest[: max(0, budget - len(must))])
        out.append(pick + [-1] * (budget - len(pick)))
    return out


def _check(T, cache, got, q, lens, blocks, scale, rows=None, layer=0):
    P, H, D = cache.page_tokens, cache.n_head_kv, cache.head_dim
    bf = cache.k.dtype == T.bfloat16
    p = 2.0 ** -16 if bf else 2.0 ** -21
    u = {T.float32: 2.0 ** -24, T.float16: 2.0 ** -11, T.bfloat16: 2.0 ** -8}[got.dtype]
    tiny = 2.0 ** -25 if got.dtype == T.float16 else 1e-37
    lists = blocks if isinstance(blocks, list) else blocks.tolist()
    for i, length in enumerate(lens):
        x = q[i].double().view(H, -1, D)
        y = got[i].double().view(H, -1, D)
        row = i if rows is None else rows[i]
        for h in range(H):
            t = [b * P + j for b in lists[i][h] if b >= 0 for j in range(min(P, length - b * P))]
            t = T.tensor(t, dtype=T.long, device="cuda")
            ids = cache.tables[row, t // P].long()
            t, ids = t[ids >= 0], ids[ids >= 0]
            if t.numel() == 0:
                assert bool((y[h] == 0).all())
                continue
            k, v = (c[layer][ids, t % P, h].double() for c in (cache.k, cache.v))
            s = x[h] @ k.T * scale
            e = 2.0 ** -20 * (1 + float((x[h].abs() @ k.abs().T * abs(scale)).max()))
            w = T.softmax(s, -1)
            want, mag = w @ v, w @ v.abs()
            err = (y[h] - want).abs()
            bound = u * want.abs() * (1 + 2.0 ** -7) + (p + 2 * e) * mag + tiny
            assert bool((err <= bound).all()), f"sequence {i}, head {h}: worst {float((err / bound).max()):.3g} of the bound"


LENS = [0, 1, 15, 16, 17, 100, 300, 1000, 2500]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,H", [(64, 1), (64, 3), (96, 1), (96, 5), (128, 8), (256, 2)])
@pytest.mark.parametrize("page", [1, 5, 16, 100])
def test_bounds(T, dtype, D, H, page):
    """Whole sequences, then the pages of new positions alone, in every layer; other pages keep theirs."""
    r = random.Random(page)
    cache, g = _cache(T, LENS, page, H, D, _dt(T, dtype), seed=D, layers=2)
    blocks = kv16.Blocks(cache)
    blocks.bounds.fill_(7.0)
    n = len(LENS)
    order = r.sample(range(n), n)
    blocks.update(_ints(T, [0] * n), _ints(T, [LENS[i] for i in order]), rows=_ints(T, order))
    want = T.full_like(blocks.bounds, 7.0)
    for i, x in enumerate(LENS):
        for layer in range(2):
            want[layer, cache.tables[i, : -(-x // page)].long()] = _bounds(T, cache, i, x, layer)
    assert T.equal(blocks.bounds, want)
    blocks.bounds.fill_(7.0)
    first = [r.randint(0, x) for x in LENS]
    end = [r.randint(a, x) for a, x in zip(first, LENS)]
    blocks.update(_ints(T, first), _ints(T, end))
    want.fill_(7.0)
    for i, (a, b) in enumerate(zip(first, end)):
        if a < b:
            for layer in range(2):
                s = slice(a // page, -(-b // page))
                want[layer, cache.tables[i, s].long()] = _bounds(T, cache, i, b, layer)[s]
    assert T.equal(blocks.bounds, want) and sjk.lib().sjk_device_status() == 0


@pytest.mark.parametrize("dtype,io", [("bf16", "bf16"), ("f16", "f16"), ("f16", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("D,H,grp", [(64, 2, 1), (64, 1, 16), (96, 3, 4), (128, 8, 7), (256, 2, 20)])
@pytest.mark.parametrize("page,budget,sink,recent", [(16, 8, 1, 1), (5, 40, 0, 0), (1, 200, 3, 5), (24, 1, 0, 1), (16, 500, 1, 1), (16, 6, 2, 4)])
def test_chosen_pages(T, dtype, io, D, H, grp, page, budget, sink, recent):
    cache, g = _cache(T, LENS, page, H, D, _dt(T, dtype), seed=D + budget)
    blocks = kv16.Blocks(cache)
    n = len(LENS)
    blocks.update(_ints(T, [0] * n), _ints(T, LENS))
    q = T.randn((n, H * grp, D), device="cuda", generator=g).to(_dt(T, io))
    lists, count = blocks.select(0, q, _ints(T, LENS), budget, sink=sink, recent=recent)
    want = [_choose(T, _bounds(T, cache, i, x), q[i], [True] * -(-x // page), budget, sink, recent) for i, x in enumerate(LENS)]
    assert lists.tolist() == want
    assert count.tolist() == [[sum(b >= 0 for b in h) for h in w] for w in want]
    out = blocks.attend(0, q, _ints(T, LENS), lists, 1 / math.sqrt(D))
    _check(T, cache, out, q, LENS, lists, 1 / math.sqrt(D))
    again, _ = blocks.select(0, q, _ints(T, LENS), budget, sink=sink, recent=recent)
    assert T.equal(again, lists) and T.equal(out, blocks.attend(0, q, _ints(T, LENS), again, 1 / math.sqrt(D)))
    assert sjk.lib().sjk_device_status() == 0


def test_all_pages_is_the_whole_attention(T):
    """With room for all pages the result is that of the attention over all positions, within both bounds."""
    lens = [3000, 77, 0, 512]
    cache, g = _cache(T, lens, 16, 4, 128, T.bfloat16)
    blocks = kv16.Blocks(cache)
    q = T.randn((4, 16, 128), device="cuda", generator=g).bfloat16()
    lists, _ = blocks.select(0, q, _ints(T, lens), 300)
    a = blocks.attend(0, q, _ints(T, lens), lists, 0.1).float()
    b = cache.attend(0, q, _ints(T, lens), 0.1).float()
    assert bool(((a - b).abs() <= 2 * 2.0 ** -8 * b.abs() + 1e-3).all())


def test_long_lists(T):
    """More pages than the choice holds in registers (8,192), and a chosen list over more than one window of the look-ups."""
    page, D = 1, 64
    lens = [20000, 8192, 8193, 100]
    cache, g = _cache(T, lens, page, 1, D, T.float16)
    blocks = kv16.Blocks(cache)
    blocks.update(_ints(T, [0] * 4), _ints(T, lens))
    q = T.randn((4, 2, D), device="cuda", generator=g).half()
    lists, _ = blocks.select(0, q, _ints(T, lens), 3000)
    for i, x in enumerate(lens):
        assert lists[i].tolist() == _choose(T, _bounds(T, cache, i, x), q[i], [True] * x, 3000, 1, 1)
    out = blocks.attend(0, q, _ints(T, lens), lists, 0.2)
    _check(T, cache, out, q, lens, lists, 0.2)


def test_ties_and_infinities(T):
    """Equal scores go to the lower pages; pages with a NaN among their keys come first, ones with infinities by their sign;
    NaN queries choose the first pages."""
    lens, page, D, n = [400], 8, 64, 50
    cache, g = _cache(T, lens, page, 1, D, T.bfloat16)
    cache.k[0] = 1.0
    blocks = kv16.Blocks(cache)
    pick = lambda q, b: blocks.select(0, q, _ints(T, lens), b, sink=0, recent=0)[0][0, 0].tolist()  # noqa: E731
    q = T.ones((1, 1, D), dtype=T.bfloat16, device="cuda")
    ids = cache.tables[0, :n].long()
    blocks.update(_ints(T, [0]), _ints(T, lens))
    assert pick(q, 5) == [0, 1, 2, 3, 4]
    cache.k[0, ids[30], 3, 0, 7] = 2.0
    cache.k[0, ids[40], 3, 0, 7] = math.nan
    cache.k[0, ids[41], 3, 0, 7] = math.inf
    cache.k[0, ids[0], :, 0, 7] = -math.inf
    cache.k[0, ids[1], :, 0, 7] = 2.0 ** -130                 # (subnormal in bf16)
    blocks.update(_ints(T, [0]), _ints(T, lens))
    assert bool(T.isnan(blocks.bounds[0, ids[40], :, 0, 7]).all())
    assert pick(q, 5) == [2, 3, 30, 40, 41]
    assert 0 not in pick(q, 49) and 1 in pick(q, 49) and 1 not in pick(q, 48)
    assert pick(q * math.nan, 3) == [0, 1, 2]
    assert pick(q * 0, 3)[0] == 0
    # 16-bit subnormals against each other: what differs in the last bit alone
    cache.k[0] = 0
    for b in range(n):
        cache.k[0, ids[b], :, 0, 0] = T.tensor((b * 7 % n + 1) * 2.0 ** -133, dtype=T.float64).to(T.bfloat16)
    blocks.update(_ints(T, [0]), _ints(T, lens))
    best = sorted(sorted(range(n), key=lambda b: -(b * 7 % n))[:6])
    assert pick(q, 6) == best and pick(q * 2.0 ** -60, 6) == best


def test_holes_and_bad_entries(T):
    """Missing pages are never chosen; ids, rows and lengths out of range set SJK_DEVICE_PAGE; lists end at what is no entry."""
    lens, page, D = [200, 200, 200], 16, 64
    cache, g = _cache(T, lens, page, 2, D, T.bfloat16)
    blocks = kv16.Blocks(cache)
    blocks.update(_ints(T, [0] * 3), _ints(T, lens))
    have = [b not in (0, 4, 12) for b in range(13)]
    b0 = _bounds(T, cache, 0, 200)
    cache.tables[0, [0, 4, 12]] = -1
    cache.tables[2] = -1
    q = T.randn((3, 4, D), device="cuda", generator=g).bfloat16()
    lists, count = blocks.select(0, q, _ints(T, lens), 5)
    assert lists[0].tolist() == _choose(T, b0, q[0], have, 5, 1, 1)
    assert lists[2].tolist() == [[-1] * 5] * 2 and count[2].tolist() == [0, 0] and sjk.lib().sjk_device_status() == 0
    out = blocks.attend(0, q, _ints(T, lens), lists, 0.1)
    _check(T, cache, out, q, lens, lists, 0.1)
    assert bool((out[2] == 0).all())
    cache.tables[1, 3] = cache.k.shape[1]
    lists, _ = blocks.select(0, q, _ints(T, lens), 20)
    assert 3 not in lists[1, 0].tolist() and sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE
    cache.tables[1, 3] = -1
    lists, _ = blocks.select(0, q, _ints(T, lens), 4, rows=_ints(T, [1, 9, -1]))
    assert lists[1:].tolist() == [[[-1] * 4] * 2] * 2 and sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE
    # lists of a caller: a later page's entry after one that does not ascend, is none, or lies behind the sequence
    mine = [[[1, 2, 2, 5], [5, 1, -1, -1]], [[0, 12, 13, -1], [-1, 3, 4, 5]], [[0, 1, 2, 3]] * 2]
    out = blocks.attend(0, q, _ints(T, lens), _ints(T, mine), 0.1)
    assert sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE
    _check(T, cache, out, q, lens, [[[1, 2], [5]], [[0, 12], []], [[], []]], 0.1)
    far = cache.tables.shape[1] * page + 50
    blocks.select(0, q, _ints(T, [far] * 3), 4)
    assert sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE
    out = blocks.attend(0, q, _ints(T, [-3, 0, 1]), _ints(T, [[[0, -1, -1, -1]] * 2] * 3), 0.1)
    assert bool((out == 0).all()) or bool((out[:2] == 0).all())
    blocks.update(_ints(T, [0, 0, 0]), _ints(T, [far, 5, 5]), rows=_ints(T, [1, 7, -2]))
    assert sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE


def test_layouts_strides_and_layers(T):
    """Heads before slots, interleaved K and V, wide query rows, any layer."""
    lens, page, H, D = [500, 90], 16, 4, 128
    cache, g = _cache(T, lens, page, H, D, T.float16, layers=3)
    blocks = kv16.Blocks(cache)
    blocks.update(_ints(T, [0, 0]), _ints(T, lens))
    q = T.randn((2, 8, D), device="cuda", generator=g).half()
    wide = T.zeros((2, 9 * D + 8), dtype=T.float16, device="cuda")
    qs = wide[:, : 8 * D].view(2, 8, D)
    qs.copy_(q)
    for layer in range(3):
        lists, _ = blocks.select(layer, q, _ints(T, lens), 7)
        assert lists.tolist() == [_choose(T, _bounds(T, cache, i, x, layer), q[i], [True] * 40, 7, 1, 1) for i, x in enumerate(lens)]
        out = blocks.attend(layer, q, _ints(T, lens), lists, 0.1)
        _check(T, cache, out, q, lens, lists, 0.1, layer=layer)
        n = cache.k.shape[1]
        hk, hv = (T.empty((3, n, H, page, D), dtype=T.float16, device="cuda").transpose(2, 3) for _ in range(2))
        both = T.empty((3, n, page, H, 2, D), dtype=T.float16, device="cuda")
        for k, v in ((hk, hv), (both[..., 0, :], both[..., 1, :])):
            k.copy_(cache.k)
            v.copy_(cache.v)
            other = kv16.Blocks(kv16.Cache(k, v, cache.tables))
            other.update(_ints(T, [0, 0]), _ints(T, lens))
            same, _ = other.select(layer, qs, _ints(T, lens), 7)
            to = T.zeros((8, 2, D), dtype=T.float16, device="cuda").transpose(0, 1)
            assert T.equal(other.bounds.nan_to_num(), blocks.bounds.nan_to_num()) and T.equal(same, lists)
            assert T.equal(other.attend(layer, qs, _ints(T, lens), same, 0.1, out=to), out)


def test_pages_carry_their_bounds(T):
    """A ledger over K, V and the bounds: a fork's split page and compacted pages bring theirs along."""
    page, H, D = 16, 2, 64
    cache = kv16.Cache.alloc(2, 40, page, H, D, T.bfloat16, 3, 8)
    blocks = kv16.Blocks(cache)
    pages = cache.pages(slabs=[blocks.bounds])
    g = T.Generator(device="cuda")
    g.manual_seed(1)
    cache.k.normal_(generator=g)
    cache.v.normal_(generator=g)
    pages.extend(_ints(T, [2, 0]), _ints(T, [0, 0]), 70)
    pages.free(_ints(T, [2]))
    blocks.update(_ints(T, [0]), _ints(T, [70]))
    before = [_bounds(T, cache, 0, 70, layer) for layer in range(2)]
    pages.fork(_ints(T, [0]), _ints(T, [1]))
    pages.extend(_ints(T, [1, 0]), _ints(T, [70, 70]), 1)
    assert int(cache.tables[1, 4]) != int(cache.tables[0, 4])
    pages.compact()
    for row in (0, 1):
        for layer in range(2):
            ids = cache.tables[row, :5].long()
            assert int(ids.max()) < 6 and T.equal(blocks.bounds[layer, ids], before[layer])
    assert sjk.lib().sjk_device_status() == 0


def test_graph_replays_with_new_lengths(T):
    """A captured step (page, cache write, choice, attention, bounds of the new position) replays as the context grows; two
    graphs captured on one stream, replayed on two, do not share scratch."""
    n, H, grp, D, page, budget = 2, 2, 4, 64, 16, 4
    cache = kv16.Cache.alloc(1, 60, page, H, D, T.float16, n, 24)
    blocks = kv16.Blocks(cache)
    pages = cache.pages(slabs=[blocks.bounds])
    rows, lens = _ints(T, [0, 1]), _ints(T, [0, 0])
    k, v, q = (T.empty((n, h, D), dtype=T.float16, device="cuda") for h in (H, H, H * grp))
    write = kv16.Qkv(D, cache=cache)
    out, lists, count = T.empty_like(q), T.empty((n, H, budget), dtype=T.int32, device="cuda"), T.empty((n, H), dtype=T.int32, device="cuda")

    def one():
        pages.extend(rows, lens, 1)
        write(k=k, v=v, pos=lens, rows=rows)
        now = lens + 1
        blocks.select(0, q, now, budget, blocks=lists, count=count)
        blocks.attend(0, q, now, lists, 0.125, out=out)
        blocks.update(lens, now)
        lens.copy_(now)

    g = T.Generator(device="cuda")
    g.manual_seed(9)
    for x in (k, v, q):
        x.normal_(generator=g)
    one()
    graph = T.cuda.CUDAGraph()
    with T.cuda.graph(graph):
        one()
    for i in range(150):
        for x in (k, v, q):
            x.normal_(generator=g)
        graph.replay()
        if i % 37 == 0 or i == 149:
            length = 2 + i
            assert lens.tolist() == [length] * n
            for s in range(n):
                assert lists[s].tolist() == _choose(T, _bounds(T, cache, s, length), q[s], [True] * 24, budget, 1, 1)
            _check(T, cache, out, q, [length] * n, lists, 0.125)
    # two graphs of choices, at once
    qs = [T.randn((n, H * grp, D), device="cuda", generator=g).half() for _ in range(2)]
    want = [blocks.select(0, x, lens, budget)[0].clone() for x in qs]
    outs = [blocks.attend(0, x, lens, w, 0.125) for x, w in zip(qs, want)]
    graphs, got = [], []
    for x in qs:
        gr = T.cuda.CUDAGraph()
        with T.cuda.graph(gr):
            ls, _ = blocks.select(0, x, lens, budget)
            got.append((ls, blocks.attend(0, x, lens, ls, 0.125)))
        graphs.append(gr)
    streams = [T.cuda.Stream() for _ in range(2)]
    T.cuda.synchronize()
    for _ in range(10):
        for gr, s in zip(graphs, streams):
            with T.cuda.stream(s):
                gr.replay()
    T.cuda.synchronize()
    for j in range(2):
        assert T.equal(got[j][0], want[j]) and T.equal(got[j][1], outs[j])
    assert sjk.lib().sjk_device_status() == 0
