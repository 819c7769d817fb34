"""sjk_kv16_attend_tree over V with infinities and NaNs: an output element is the sum of those that its token sees (an infinity where
they have one sign, NaN otherwise) and, where it sees none, what it is without them. Long pairs beside short ones (the bad values
of one sequence cost no other its results, and no wait runs out), pairs cut into many runs, more pairs a CTA than are gone through
at once, outputs over the queries. Finite elements are held to the bound of test_gpu_cache_draft."""
import math
import random

import pytest

import sjk
from test_gpu_cache_draft import _cache, _first, _ints, _signed, _tree

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan


@pytest.fixture(scope="module")
def T():
    import build
    build.build()
    import torch
    assert torch.cuda.is_available()
    return torch


def _sees(length, mask, t, window):
    """Whether a token that sees the drafted ones of `mask` sees position t (numbers, or a tensor of positions)."""
    drafts = [k for k in range(64) if mask >> k & 1]
    if window:
        drafts = drafts[-window:]
    low = max(0, length - (window - len(drafts))) if window else 0
    on = (t >= low) & (t < length)
    for k in drafts:
        on = on | (t == length + k)
    return on


def _check(T, cache, got, q, lens, counts, chains, scale, window):
    """As test_gpu_cache_draft's, for long sequences."""
    P, H = cache.page_tokens, cache.n_head_kv
    u, p, tiny = (2.0 ** -8, 2.0 ** -16, 1e-37) if cache.k.dtype == T.bfloat16 else (2.0 ** -11, 2.0 ** -21, 2.0 ** -25)
    at = 0
    for i, (length, n) in enumerate(zip(lens, counts)):
        t = T.arange(length + n, device="cuda")
        sees = T.stack([_sees(length, m & ((1 << n) - 1), t, window) for m in chains[i]])
        ids = cache.tables[i, t // P].long()
        k, v = (c[0][ids, t % P].double() for c in (cache.k, cache.v))
        x = q[at:at + n].double().view(n, H, -1, q.shape[-1])
        s = T.einsum("jhgd,thd->jhgt", x, k) * scale
        mag = float((T.einsum("jhgd,thd->jhgt", x.abs(), k.abs()) * abs(scale)).max())
        w = T.nan_to_num(T.softmax(s.masked_fill(~sees[:, None, None, :], -math.inf), -1))
        want, mag_v = T.einsum("jhgt,thd->jhgd", w, v), T.einsum("jhgt,thd->jhgd", w, v.abs())
        bound = u * want.abs() * (1 + 2.0 ** -7) + (p + 2.0 ** -17 * (1 + mag) + 2.0 ** -26 * (length + n + 1600)) * mag_v + tiny
        err = (got[at:at + n].double().view(want.shape) - want).abs()
        assert bool((err <= bound).all()), f"sequence {i} of {length} + {n}: worst {float((err / bound).max()):.3g} of the bound"
        at += n


def _odd(T, cache, q, lens, counts, masks, scale, window, bad):
    """bad: (sequence, position, head, channel, value). The call with them, and without them the call's check."""
    flat = None if masks is None else _ints(T, [m for x in masks for m in _signed(x)], T.int64)
    first = _ints(T, _first(counts))
    call = lambda **kw: cache.attend_tree(0, q, _ints(T, lens), flat, scale, first=first, window=window, **kw)  # noqa: E731
    P, H = cache.page_tokens, cache.n_head_kv
    chains = [[(2 << j) - 1 for j in range(n)] for n in counts] if masks is None else masks
    place = lambda i, t: (0, int(cache.tables[i, t // P]), t % P)  # noqa: E731
    was = []
    for i, t, h, d, x in bad:
        was.append(cache.v[place(i, t)][h, d].clone())
        cache.v[place(i, t)][h, d] = x
    out = call()
    assert T.equal(out.view(T.int16), call().view(T.int16))
    over = q.clone()
    assert cache.attend_tree(0, over, _ints(T, lens), flat, scale, first=first, window=window, out=over) is over
    assert T.equal(out.view(T.int16), over.view(T.int16))
    assert sjk.lib().sjk_device_status() == 0
    # the values are zeros from here on, of which no sum takes notice
    for i, t, h, d, x in bad:
        cache.v[place(i, t)][h, d] = 0
    clean = call()
    grp = q.shape[1] // H
    want = T.zeros(q.shape, dtype=T.float64)
    at = 0
    for i, (length, n) in enumerate(zip(lens, counts)):
        for j in range(n):
            for b, t, h, d, x in bad:
                if b == i and _sees(length, chains[i][j] & ((1 << n) - 1), t, window):
                    want[at + j, h * grp:(h + 1) * grp, d] += x
        at += n
    want = want.cuda()
    odd = want != 0
    assert bool(odd.any()) and bool((~odd).any())
    assert T.equal(out[odd].double().nan_to_num(7.0), want[odd].nan_to_num(7.0)), "infinities and NaNs"
    assert bool(T.isfinite(out[~odd]).all())
    _check(T, cache, T.where(odd, clean, out), q, lens, counts, chains, scale, window)
    for b, x in zip(bad, was):
        cache.v[place(b[0], b[1])][b[2], b[3]] = x


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("D,H,grp,nodes", [(64, 1, 4, 64), (128, 1, 2, 33), (256, 1, 4, 16), (96, 2, 8, 9)])
@pytest.mark.parametrize("page,window", [(16, 0), (5, 0), (128, 3000), (24, 3000)])
def test_long_pairs_beside_short_ones(T, dtype, D, H, grp, nodes, page, window):
    """Three long sequences, of which the second has the bad values, between short ones: a CTA's run goes over both."""
    r = random.Random(D + page)
    lens = [40, 60000, 7, 90000, 300, 50000, 12, 0]
    counts = [3, nodes, 1, nodes, nodes, nodes, 2, 5]
    cache, g = _cache(T, [a + b for a, b in zip(lens, counts)], page, H, D, getattr(T, dtype), seed=page)
    masks = [_tree(r, n) for n in counts]
    q = T.randn((sum(counts), H * grp, D), device="cuda", generator=g).to(cache.k.dtype)
    h = H - 1
    some = [(3, 90000 + 2, h, d, NAN) for d in range(D)]
    _odd(T, cache, q, lens, counts, masks, 0.1, window, some + [(3, 90000 + nodes - 1, 0, 1, INF), (3, 90000 + nodes // 2, 0, D - 1, -INF)])
    # positions that all tokens see (without a window): the first, one in the middle, the last, one at the window's edge
    low = 90000 - window if window else 0
    for t in {low, low + 5, low + (90000 - low) // 2, 90000 - 1}:
        _odd(T, cache, q, lens, counts, masks, 0.1, window, [(3, t, h, 3, INF), (3, t, h, 4, -INF), (3, t, 0, D // 2, NAN), (3, 90000 + 1, h, 3, -INF)])
    # short sequences' and a long one's at once
    _odd(T, cache, q, lens, counts, masks, 0.1, window, [(0, 41, 0, 0, INF), (4, 299, h, 7, INF), (4, 301, h, 7, -INF), (5, 50000, h, 9, NAN), (6, 0, 0, 33, -INF)])


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("D,grp", [(64, 2), (128, 4), (256, 4)])
@pytest.mark.parametrize("n,length", [(1, 70000), (40, 900), (300, 200)])
def test_the_same_however_the_list_is_cut(T, dtype, D, grp, n, length):
    """An infinity in a place that every token sees is one in the output, in pairs that one CTA has whole and in ones cut into many runs, and
    where a later run's scores are far above its own."""
    cache, g = _cache(T, [length + 4] * n, 16, 2, D, getattr(T, dtype), seed=n)
    q = T.randn((4 * n, 2 * grp, D), device="cuda", generator=g).to(cache.k.dtype)
    i = n // 2
    bad = [(i, t, 1, d, x) for t, d, x in ((length // 3, 0, INF), (length // 2, 1, -INF), (length - 1, 2, NAN), (length, 3, INF), (length + 3, 4, -INF), (5, 5, INF), (length // 2, 5, -INF))]
    _odd(T, cache, q, [length] * n, [4] * n, None, 0.1, 0, bad)
    t = _ints(T, [length - 2]).long()
    cache.k[0, cache.tables[i, t // 16].long(), t % 16, 1] = 3.0 * q[4 * i + 3, 2 * grp - 1]
    _odd(T, cache, q, [length] * n, [4] * n, None, 1.0, 0, bad)


@pytest.mark.parametrize("page", [16, 12])
def test_more_pairs_than_are_gone_through_at_once(T, page):
    """1,100 and more pairs a CTA, some of them with infinities, before and behind the thousandth."""
    n, H, D, length, nodes = 21000, 8, 64, 9, 2
    g = T.Generator(device="cuda")
    g.manual_seed(page)
    import kv16
    cache = kv16.Cache.alloc(1, n, page, H, D, T.bfloat16, n, 1)
    cache.tables[:, 0] = T.randperm(n, generator=g, device="cuda").int()
    cache.k.normal_(generator=g)
    cache.v.normal_(generator=g)
    ids = cache.tables[:, 0].long()
    q = T.randn((n * nodes, H, D), device="cuda", generator=g).bfloat16()
    lens = T.full((n,), length, dtype=T.int32, device="cuda")
    i, h, d = (T.randint(0, top, (700,), generator=g, device="cuda") for top in (n, H, D))
    i[:20] = T.arange(20, device="cuda")
    i[20:40] = n - 1 - T.arange(20, device="cuda")
    t = T.randint(0, length + nodes, (700,), generator=g, device="cuda")
    t[:400] = length + 1                                     # (which the first of the two tokens does not see)
    cache.v[0, ids[i], t, h, d] = INF
    out = cache.attend_tree(0, q, lens, None, 0.2).view(n, nodes, H, D)
    assert sjk.lib().sjk_device_status() == 0
    odd = T.zeros((n, nodes, H, D), dtype=T.bool, device="cuda")
    for j in range(nodes):
        on = t <= length + j
        odd[i[on], j, h[on], d[on]] = True
    assert T.equal(out == INF, odd) and bool(T.isfinite(out[~odd]).all())
    cache.v[0, ids[i], t, h, d] = 0
    for a in range(0, n, 3000):
        b = slice(a, a + 3000)
        k, v = (c[0, ids[b], : length + nodes].double() for c in (cache.k, cache.v))
        x = q.view(n, nodes, H, D)[b].double()
        s = T.einsum("njhd,nthd->njht", x, k) * 0.2
        last = length + T.arange(nodes, device="cuda")
        s = s.masked_fill((T.arange(length + nodes, device="cuda")[None] > last[:, None])[None, :, None, :], -INF)
        w = T.softmax(s, -1)
        want, mag = T.einsum("njht,nthd->njhd", w, v), T.einsum("njht,nthd->njhd", w, v.abs())
        e = 2.0 ** -18 * (1 + float((T.einsum("njhd,nthd->njht", x.abs(), k.abs()) * 0.2).max()))
        bound = 2.0 ** -8 * want.abs() * (1 + 2.0 ** -7) + (2.0 ** -16 + 2 * e + 2.0 ** -26 * 1700) * mag + 1e-37
        assert bool(((out[b].double() - want).abs() <= bound)[~odd[b]].all())


@pytest.mark.parametrize("page", [16, 5])
def test_replays_with_and_without(T, page):
    """A captured call replays over values that come and go, on two streams at once; a page is missing, and slots of nobody are NaN."""
    lens, counts, H, D = [700, 30, 20000], [5, 9, 16], 2, 128
    cache, g = _cache(T, [a + b for a, b in zip(lens, counts)], page, H, D, T.float16, seed=page)
    cache.tables[2, 3] = -1
    masks = [_tree(random.Random(i), n) for i, n in enumerate(counts)]
    flat, first, dl = _ints(T, [m for x in masks for m in _signed(x)], T.int64), _ints(T, _first(counts)), _ints(T, lens)
    qs = [T.randn((sum(counts), 3 * H, D), device="cuda", generator=g).half() for _ in range(2)]
    call = lambda q: cache.attend_tree(0, q, dl, flat, 0.1, first=first)  # noqa: E731
    clean = [call(q) for q in qs]
    graphs, outs = [], []
    for q in qs:
        gr = T.cuda.CUDAGraph()
        with T.cuda.graph(gr):
            outs.append(call(q))
        graphs.append(gr)
    streams = [T.cuda.Stream() for _ in range(2)]
    place = (0, int(cache.tables[2, 20003 // page]), 20003 % page)
    was = cache.v[place][1, 7].clone()
    for x in (None, INF, None, NAN, -INF, None):
        cache.v[place][1, 7] = was if x is None else x
        T.cuda.synchronize()
        for gr, s in zip(graphs, streams):
            with T.cuda.stream(s):
                gr.replay()
                gr.replay()
        T.cuda.synchronize()
        for o, c in zip(outs, clean):
            if x is None:
                assert T.equal(o, c)
                continue
            hit = T.zeros(o.shape, dtype=T.bool, device="cuda")
            for j in range(counts[2]):
                hit[14 + j, 3:, 7] = bool(masks[2][j] >> 3 & 1)
            assert T.equal(o[hit].nan_to_num(7.0), T.full_like(o[hit], x).nan_to_num(7.0)) and bool(T.isfinite(o[~hit]).all())
            # what does not see it is as without it: a sum of the same terms, of which one is now left out where its weight was 0
            assert T.equal(o[~hit], c[~hit])
    assert sjk.lib().sjk_device_status() == 0
