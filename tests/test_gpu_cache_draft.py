"""Steps with several new tokens of every sequence: sjk_kv16_maps, sjk_qkv_at, sjk_kv16_attend_tree and sjk_kv16_keep, each
against its definition (64 bits for what is computed), and together as a decode loop with drafted trees.

Error bound of an output element y of the attention, with A the same attention over |V|: u |y| for the rounding to the output
type (half a step: 2^-8 bf16, 2^-11 f16), and (p + 2 e + s) A for the weights and the sums. p is what two 16-bit terms leave of
a weight, 2^-16 (bf16) or 2^-21 (f16). e bounds the error of a score in units of ln 2: sums of at most 256 exact products in
16 + 16 additions, each off by at most 2^-23 of the sum of magnitudes, and what turns it into a weight, 2^-18 (1 + max_t scale
sum_d |q_d k_td|) in all. s: a sum over T positions is made of at most T / 8 + 200 additions (groups of 16, two terms each, and
the joins), each off by 2^-23 of A: 2^-26 (T + 1600)."""
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


def _cache(T, ends, page, H, D, dtype, seed=0, layers=1, junk=math.nan):
    """A cache whose positions below `ends` are normal values and whose other slots are junk."""
    g = T.Generator(device="cuda")
    g.manual_seed(seed)
    n, stride = len(ends), max(1, max(-(-x // page) for x in ends)) + 1
    pages = sum(-(-x // page) for x in ends) + 3
    cache = kv16.Cache.alloc(layers, pages, page, H, D, dtype, n, stride)
    cache.k.fill_(junk)
    cache.v.fill_(junk)
    perm = T.randperm(pages, generator=g, device="cuda")
    at = 0
    for i, x in enumerate(ends):
        per = -(-x // page)
        ids = perm[at:at + per]
        at += per
        cache.tables[i, :per] = ids.int()
        t = T.arange(x, device="cuda")
        for c in (cache.k, cache.v):
            c[:, ids[t // page], t % page] = T.randn((layers, x, H, D), device="cuda", generator=g).to(dtype)
    return cache, g


def _tree(r, n):
    masks = []
    for j in range(n):
        masks.append((masks[r.randrange(j)] if j else 0) | 1 << j)
    return masks


def _visible(length, masks, j, window, ends=None):
    """Positions that drafted token j sees: the last `window` of the committed and its drafted ones."""
    seen = list(range(length)) + [length + k for k in range(len(masks)) if masks[j] >> k & 1]
    return seen[-window:] if window else seen


def _signed(masks):
    return [m - (1 << 64) if m >> 63 else m for m in masks]


def _check(T, cache, got, q, lens, counts, masks, scale, window=0, rows=None, layer=0, live=lambda i, t: True):
    """masks: a list per sequence; None: positions in a row."""
    P, H, D = cache.page_tokens, cache.n_head_kv, cache.head_dim
    bf = cache.k.dtype == T.bfloat16
    u, p, tiny = (2.0 ** -8, 2.0 ** -16, 1e-37) if bf else (2.0 ** -11, 2.0 ** -21, 2.0 ** -25)
    at = 0
    for i, (length, n) in enumerate(zip(lens, counts)):
        row = i if rows is None else rows[i]
        m = [(2 << j) - 1 for j in range(n)] if masks is None else [x & ((1 << n) - 1) for x in masks[i]]
        if n == 0:
            continue
        t = T.arange(length + n, device="cuda")
        ids = cache.tables[row, (t // P).clamp(max=cache.tables.shape[1] - 1)].long()
        have = (ids >= 0) & (t // P < cache.tables.shape[1]) & T.tensor([live(i, x) for x in range(length + n)], device="cuda")
        sees = T.zeros((n, length + n), dtype=T.bool)
        for j in range(n):
            sees[j, _visible(length, m, j, window)] = True
        sees = sees.cuda() & have
        k, v = (T.where(have[:, None, None], c[layer][ids.clamp(min=0), t % P].double(), 0.0) for c in (cache.k, cache.v))
        x = q[at:at + n].double().view(n, H, -1, D)
        s = T.einsum("jhgd,thd->jhgt", x, k) * scale
        mag = float((T.einsum("jhgd,thd->jhgt", x.abs(), k.abs()) * abs(scale)).max())
        s = s.masked_fill(~sees[:, None, None, :], -math.inf)
        w = T.nan_to_num(T.softmax(s, -1))                     # a token that sees nothing gets zeros
        want, mag_v = T.einsum("jhgt,thd->jhgd", w, v), T.einsum("jhgt,thd->jhgd", w, v.abs())
        e = 2.0 ** -18 * (1 + mag)
        bound = u * want.abs() * (1 + 2.0 ** -7) + (p + 2 * e + 2.0 ** -26 * (length + n + 1600)) * mag_v + tiny
        err = (got[at:at + n].double().view(want.shape) - want).abs()
        assert bool((err <= bound).all()), f"sequence {i} of {length} + {n}: worst {float((err / bound).max()):.3g} of the bound"
        at += n


def _ints(T, x, dtype=None):
    return T.tensor(x, dtype=dtype or T.int32, device="cuda")


def _first(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


# ---- attention ------------------------------------------------------------------------------------------------------

LENS = [0, 1, 7, 127, 128, 129, 255, 300, 1000, 0]
COUNTS = [1, 64, 3, 0, 5, 2, 33, 17, 64, 0]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("grp", [1, 3, 4, 16])
@pytest.mark.parametrize("page", [5, 16, 24, 128])
def test_trees(T, dtype, D, grp, page):
    """Ragged trees, pages that are and are no multiple of 8 tokens, one to sixteen tiles of rows; slots that nobody sees are NaN."""
    r = random.Random(D + grp + page)
    cache, g = _cache(T, [a + b for a, b in zip(LENS, COUNTS)], page, 2, D, getattr(T, dtype), seed=grp)
    masks = [_tree(r, n) for n in COUNTS]
    q = (1.5 * T.randn((sum(COUNTS), 2 * grp, D), device="cuda", generator=g)).to(cache.k.dtype)
    flat = _ints(T, [m for x in masks for m in _signed(x)], T.int64)
    out = cache.attend_tree(0, q, _ints(T, LENS), flat, 1 / math.sqrt(D), first=_ints(T, _first(COUNTS)))
    _check(T, cache, out, q, LENS, COUNTS, masks, 1 / math.sqrt(D))
    again = cache.attend_tree(0, q, _ints(T, LENS), flat, 1 / math.sqrt(D), first=_ints(T, _first(COUNTS)))
    assert T.equal(out, again) and sjk.lib().sjk_device_status() == 0


@pytest.mark.parametrize("window", [1, 5, 40, 64, 200, 100000])
@pytest.mark.parametrize("page", [1, 16, 24])
@pytest.mark.parametrize("kind", ["tree", "chain", "any"])
def test_windows_and_masks(T, window, page, kind):
    """Windows that end among the drafted ones and before them; masks of any kind, empty ones and ones with bits behind the
    sequence's tokens among them. Pages that the window has passed are gone."""
    r = random.Random(window)
    cache, g = _cache(T, [a + b for a, b in zip(LENS, COUNTS)], page, 1, 64, T.bfloat16, seed=page)
    for i, x in enumerate(LENS):
        cache.tables[i, : max(0, x - window) // page] = -1
    masks = None
    if kind == "tree":
        masks = [_tree(r, n) for n in COUNTS]
    if kind == "any":
        masks = [[r.choice([0, r.getrandbits(64), 1 << r.randrange(64)]) for _ in range(n)] for n in COUNTS]
    q = T.randn((sum(COUNTS), 5, 64), device="cuda", generator=g).bfloat16()
    flat = None if masks is None else _ints(T, [m for x in masks for m in _signed(x)], T.int64)
    out = cache.attend_tree(0, q, _ints(T, LENS), flat, 0.2, first=_ints(T, _first(COUNTS)), window=window)
    _check(T, cache, out, q, LENS, COUNTS, masks, 0.2, window)
    assert sjk.lib().sjk_device_status() == 0


@pytest.mark.parametrize("n,top,nodes", [(1, 20000, 8), (3, 100000, 64), (40, 900, 16), (300, 90, 3), (1100, 5, 2)])
@pytest.mark.parametrize("H,grp,D", [(1, 4, 128), (4, 4, 256), (8, 1, 64)])
def test_batches(T, n, top, nodes, H, grp, D):
    """From one sequence that all CTAs share to more than there are CTAs, rows in any order, and the tokens of each the same
    number (no `first`)."""
    r = random.Random(n)
    lens = [r.randint(0, top) for _ in range(n)]
    lens[-1] = top
    cache, g = _cache(T, [x + nodes for x in lens], 16, H, D, T.bfloat16, seed=n, junk=math.inf)
    order = list(range(n))
    r.shuffle(order)
    mine = [lens[i] for i in order]
    q = T.randn((n * nodes, H * grp, D), device="cuda", generator=g).bfloat16()
    masks = [_tree(r, nodes) for _ in range(n)]
    flat = _ints(T, [m for x in masks for m in _signed(x)], T.int64)
    out = cache.attend_tree(0, q, _ints(T, mine), flat, 0.1, rows=_ints(T, order))
    _check(T, cache, out, q, mine, [nodes] * n, masks, 0.1, rows=order)
    assert T.equal(out, cache.attend_tree(0, q, _ints(T, mine), flat, 0.1, rows=_ints(T, order)))
    assert sjk.lib().sjk_device_status() == 0


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("page", [5, 16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 150])
def test_infinities_in_masked_places(T, dtype, page, D, window):
    """Infinities and NaNs in K and V of drafted tokens (and at a window's edge) reach the tokens that see them alone."""
    length, n = 300, 12
    cache, g = _cache(T, [length + n], page, 2, D, getattr(T, dtype), seed=1)
    masks = [_tree(random.Random(4), n)]
    place = lambda t: (0, cache.tables[0, t // page].long(), t % page)  # noqa: E731
    bad = {length + 5: ("v", math.nan), length + 7: ("v", math.inf), length + 9: ("k", math.nan), length + 11: ("v", -math.inf)}
    if window:
        bad[length - window + 3] = ("v", math.inf)           # tokens that see four or more others do not see it
    for t, (which, x) in bad.items():
        (cache.v if which == "v" else cache.k)[place(t)][:, D // 3] = x
    q = T.randn((n, 6, D), device="cuda", generator=g).to(cache.k.dtype)
    out = cache.attend_tree(0, q, _ints(T, [length]), _ints(T, _signed(masks[0]), T.int64), 0.1, window=window)
    sees = [set(_visible(length, masks[0], j, window)) for j in range(n)]
    # what sees no such place is what it would be without them, within the bound of each (the sums may go another way)
    for t, (which, x) in bad.items():
        (cache.v if which == "v" else cache.k)[place(t)][:, D // 3] = 0
    clean = cache.attend_tree(0, q, _ints(T, [length]), _ints(T, _signed(masks[0]), T.int64), 0.1, window=window)
    _check(T, cache, clean, q, [length], [n], masks, 0.1, window)
    hit, mended = 0, out.clone()
    for j in range(n):
        mine = [bad[t] for t in bad if t in sees[j]]
        if not mine:
            continue
        hit += 1
        mended[j] = clean[j]
        if any(w == "k" for w, _ in mine):
            assert bool(T.isnan(out[j]).all())
            continue
        assert not bool(T.isfinite(out[j][:, D // 3]).any())
        rest = [d for d in range(D) if d != D // 3]
        mended[j][:, rest] = out[j][:, rest]
        xs = {x for _, x in mine}
        if len(xs) == 1 and not math.isnan(next(iter(xs))):
            assert bool((out[j][:, D // 3] == next(iter(xs))).all())
    _check(T, cache, mended, q, [length], [n], masks, 0.1, window)
    assert 0 < hit < n and sjk.lib().sjk_device_status() == 0


def test_layouts_and_strides(T):
    """Heads before slots, K and V interleaved, queries and outputs of other strides and of a wider row give the same bits."""
    lens, counts, page, H, D = [3, 200, 77], [4, 4, 4], 16, 2, 128
    cache, g = _cache(T, [a + b for a, b in zip(lens, counts)], page, H, D, T.float16)
    q = T.randn((12, 8, D), device="cuda", generator=g).half()
    dl = _ints(T, lens)
    want = cache.attend_tree(0, q, dl, None, 0.1)
    _check(T, cache, want, q, lens, counts, None, 0.1)
    n = cache.k.shape[1]
    hk, hv = (T.empty((1, n, H, page, D), dtype=T.float16, device="cuda").transpose(2, 3) for _ in range(2))
    both = T.empty((1, n, page, H, 2, D), dtype=T.float16, device="cuda")
    for k, v in ((hk, hv), (both[..., 0, :], both[..., 1, :])):
        k.copy_(cache.k)
        v.copy_(cache.v)
        assert T.equal(kv16.Cache(k, v, cache.tables).attend_tree(0, q, dl, None, 0.1), want)
    wide = T.full((12, 8 * D + 64), 7.0, dtype=T.float16, device="cuda")
    qs = wide[:, : 8 * D].view(12, 8, D)
    qs.copy_(q)
    out = T.full((8, 12, D + 1), 7.0, dtype=T.float16, device="cuda")
    to = out[:, :, :D].transpose(0, 1)
    assert T.equal(cache.attend_tree(0, qs, dl, None, 0.1, out=to), want)
    assert bool((out[:, :, D] == 7).all()) and bool((wide[:, 8 * D:] == 7).all())


def test_rows_of_nobody(T):
    """Rows before the first sequence's and behind the last one's, and those of a sequence with too many tokens, stay as they
    were; the latter is reported."""
    cache, g = _cache(T, [40, 50], 16, 1, 64, T.bfloat16)
    q = T.randn((20, 2, 64), device="cuda", generator=g).bfloat16()
    out = T.full_like(q, 3.0)
    cache.attend_tree(0, q, _ints(T, [35, 44]), None, 0.1, first=_ints(T, [2, 7, 13]), out=out)
    assert bool((out[:2] == 3).all()) and bool((out[13:] == 3).all())
    _check(T, cache, out[2:13], q[2:13], [35, 44], [5, 6], None, 0.1)
    assert sjk.lib().sjk_device_status() == 0
    out.fill_(3.0)
    cache.attend_tree(0, q, _ints(T, [35, 44]), None, 0.1, first=_ints(T, [2, 7, 13]), nodes=5, out=out)
    assert bool((out[7:] == 3).all()) and sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE
    _check(T, cache, out[2:7], q[2:7], [35], [5], None, 0.1)
    for first in ([0, 9, 4], [0, 5, 21], [-1, 5, 9]):
        out.fill_(3.0)
        cache.attend_tree(0, q, _ints(T, [35, 44]), None, 0.1, first=_ints(T, first), out=out)
        assert sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE


def test_holes_and_bad_entries(T):
    """Positions on a missing page are left out, silently for SJKVARN_NO_BLOCK and with SJK_DEVICE_PAGE for ids, rows and
    lengths out of range; tokens that see nothing get zeros."""
    for page in (16, 5):
        lens, counts = [100, 100, 60], [4, 4, 4]
        cache, g = _cache(T, [a + b for a, b in zip(lens, counts)], page, 2, 64, T.bfloat16)
        cache.tables[0, 2] = -1
        cache.tables[2] = -1
        q = T.randn((12, 4, 64), device="cuda", generator=g).bfloat16()
        out = cache.attend_tree(0, q, _ints(T, lens), None, 0.1)
        _check(T, cache, out, q, lens, counts, None, 0.1)
        assert bool((out[8:] == 0).all()) and sjk.lib().sjk_device_status() == 0
        cache.tables[1, 3] = cache.k.shape[1]
        out = cache.attend_tree(0, q, _ints(T, lens), None, 0.1)
        cache.tables[1, 3] = -1
        _check(T, cache, out, q, lens, counts, None, 0.1)
        assert sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE
        out = cache.attend_tree(0, q[:8], _ints(T, lens[:2]), None, 0.1, rows=_ints(T, [7, 1]))
        assert bool((out[:4] == 0).all()) and sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE
        _check(T, cache, out[4:], q[4:8], [100], [4], None, 0.1, rows=[1])
        far = cache.tables.shape[1] * page
        for window in (0, 8):
            out = cache.attend_tree(0, q[:4], _ints(T, [far + 1000]), None, 0.1, rows=_ints(T, [1]), window=window)
            assert sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE
            if window:
                assert bool((out == 0).all())
        out = cache.attend_tree(0, q[:4], _ints(T, [-5]), None, 0.1, rows=_ints(T, [1]))
        _check(T, cache, out, q[:4], [0], [4], None, 0.1, rows=[1])


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_extreme_scores(T, dtype):
    """Large scores of both signs, scale 0 and negative ones; one token that takes all, late in a long sequence (the maximum
    in use has to change then), and small ones that keep their share."""
    lens, D = [700, 64], 128
    cache, g = _cache(T, [710, 74], 16, 1, D, getattr(T, dtype))
    q = (30 * T.randn((20, 4, D), device="cuda", generator=g)).to(cache.k.dtype)
    for scale in (1.0, -1.0, 0.0, 1e-3, -0.05):
        out = cache.attend_tree(0, q, _ints(T, lens), None, scale)
        _check(T, cache, out, q, lens, [10, 10], None, scale)
    assert bool(T.isfinite(cache.attend_tree(0, q, _ints(T, lens), None, 1e4)).all())
    # scores that rise along the sequence: 0, 30, 60, ... nats
    cache.k.zero_()
    t = T.arange(710, device="cuda")
    cache.k[0, cache.tables[0, t // 16].long(), t % 16, 0, 0] = (t // 100).to(cache.k.dtype)
    q.zero_()
    q[:, :, 0] = 30.0
    out = cache.attend_tree(0, q, _ints(T, lens), None, 1.0)
    _check(T, cache, out, q, lens, [10, 10], None, 1.0)
    # 16 nats below the largest one, 700 of them: their sum counts 2^-14
    cache.k.zero_()
    cache.k[0, cache.tables[0, 0].long(), 0, 0, 0] = 16.0
    q.zero_()
    q[:, :, 0] = 1.0
    cache.v.fill_(0.0)
    cache.v[0, cache.tables[0, t // 16].long(), t % 16, 0] = 1.0
    cache.v[0, cache.tables[0, 0].long(), 0, 0] = 0.0
    out = cache.attend_tree(0, q, _ints(T, lens), None, 1.0)
    _check(T, cache, out, q, lens, [10, 10], None, 1.0)
    assert float(out[0].min()) > 0


def test_offsets_past_32_bits(T):
    """A cache of more than 2^32 elements: pages at its far end are read and moved where they are."""
    page, H, D = 128, 4, 256
    n_pages = 2 ** 32 // (page * H * D) + 8
    k, v = (T.empty((1, n_pages, page, H, D), dtype=T.bfloat16, device="cuda") for _ in range(2))
    tables = _ints(T, [[n_pages - 1, 0, n_pages - 3]])
    g = T.Generator(device="cuda")
    g.manual_seed(2)
    for i in (0, n_pages - 3, n_pages - 1):
        k[0, i].normal_(generator=g)
        v[0, i].normal_(generator=g)
    cache = kv16.Cache(k, v, tables)
    q = T.randn((9, 16, D), device="cuda", generator=g).bfloat16()
    out = cache.attend_tree(0, q, _ints(T, [300]), None, 1 / 16)
    _check(T, cache, out, q, [300], [9], None, 1 / 16)
    row = k[0, n_pages - 3, 304 - 256].clone()
    assert cache.keep(_ints(T, [300]), _ints(T, [[0, 4]]), _ints(T, [2])).tolist() == [302]
    assert T.equal(k[0, n_pages - 3, 301 - 256], row)


@pytest.mark.parametrize("page", [2 ** 20 + 8, 2 ** 20])
def test_longest_sequence(T, page):
    """The last positions below 2^31 - 1."""
    n, D = 7, 64
    length = 2 ** 31 - 1 - n
    cache = kv16.Cache.alloc(1, 2, page, 1, D, T.bfloat16, 1, 2048)
    g = T.Generator(device="cuda")
    g.manual_seed(page)
    cache.k.normal_(generator=g)
    cache.v.normal_(generator=g)
    cache.tables.fill_(-1)
    cache.tables[0, 2046:] = _ints(T, [1, 0])
    q = T.randn((n, 2, D), device="cuda", generator=g).bfloat16()
    window = 5000
    out = cache.attend_tree(0, q, _ints(T, [length]), None, 0.5, window=window)
    assert sjk.lib().sjk_device_status() == 0
    t = T.arange(length - window, length + n, device="cuda")
    ids = cache.tables[0, t // page].long()
    kk, vv = (c[0][ids, t % page, 0].double() for c in (cache.k, cache.v))
    s = q.double() @ kk.T * 0.5
    last = length + T.arange(n, device="cuda")[:, None]
    s = s.masked_fill(((t > last) | (t <= last - window))[:, None, :], -math.inf)
    w = T.softmax(s, -1)
    want, mag = w @ vv, w @ vv.abs()
    e = 2.0 ** -18 * (1 + float((q.double().abs() @ kk.abs().T * 0.5).max()))
    assert bool(((out.double() - want).abs() <= 2.0 ** -8 * 1.01 * want.abs() + (2.0 ** -16 + 2 * e + 2.0 ** -26 * 7000) * mag).all())
    m = kv16.Maps(cache, 1, 8)(_ints(T, [length]), _ints(T, [n]))
    assert m.at.tolist() == list(range(length, length + n)) + [-1] and sjk.lib().sjk_device_status() == 0


def test_two_streams(T):
    """Calls of one cache on two streams at once keep their own scratch."""
    lens, D = [9000, 4000], 128
    cache, g = _cache(T, [x + 8 for x in lens], 16, 4, D, T.bfloat16)
    qs = [T.randn((16, 16, D), device="cuda", generator=g).bfloat16() for _ in range(2)]
    dl = _ints(T, lens)
    want = [cache.attend_tree(0, q, dl, None, 0.1) for q in qs]
    T.cuda.synchronize()
    streams, outs = [T.cuda.Stream() for _ in range(2)], [[], []]
    for i in range(20):
        for j, s in enumerate(streams):
            with T.cuda.stream(s):
                outs[j].append(cache.attend_tree(0, qs[j], dl, None, 0.1))
    T.cuda.synchronize()
    assert all(T.equal(o, want[j]) for j in range(2) for o in outs[j]) and sjk.lib().sjk_device_status() == 0


# ---- maps, cache positions, keep ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("n,page,top", [(1, 16, 8), (5, 24, 40), (300, 16, 7), (1000, 1, 64), (8192, 128, 3)])
@pytest.mark.parametrize("trees", [False, True])
def test_maps(T, n, page, top, trees):
    r = random.Random(n)
    lens = [r.randint(0, 500) for _ in range(n)]
    adds = [r.randint(0, top) for _ in range(n)]
    rows = r.sample(range(n + 3), n)
    stride = (500 + top) // page + 1
    tables = T.randperm((n + 3) * stride, device="cuda").int().view(n + 3, stride)
    tables[rows[0], 0] = -1
    k = T.zeros((1, (n + 3) * stride, 1, 1, 64), dtype=T.bfloat16, device="cuda").expand(-1, -1, page, -1, -1)
    cache = kv16.Cache(k, k, tables)
    n_tok = sum(adds) + 9
    masks = [_tree(r, a) for a in adds]
    flat = _ints(T, [m for x in masks for m in _signed(x)] + [-1] * 9, T.int64) if trees else None
    m = kv16.Maps(cache, n, n_tok)
    assert m(_ints(T, lens), _ints(T, adds), rows=_ints(T, rows), masks=flat) is m
    host = tables.tolist()
    first, row, at, pos, slot = [0], [], [], [], []
    for i in range(n):
        first.append(first[-1] + adds[i])
        for j in range(adds[i]):
            t = lens[i] + j
            row.append(rows[i])
            at.append(t)
            pos.append(lens[i] + bin(masks[i][j]).count("1") - 1 if trees else t)
            p = host[rows[i]][t // page]
            slot.append(-1 if p < 0 else p * page + t % page)
    assert m.first.tolist() == first and m.rows.tolist() == row + [0] * 9 and m.at.tolist() == at + [-1] * 9
    assert m.pos.tolist() == pos + [-1] * 9 and m.slots.tolist() == slot + [-1] * 9
    assert sjk.lib().sjk_device_status() == 0


def test_maps_refusals_on_the_device(T):
    """Tokens beyond the room, negative counts and lengths, rows and positions outside the tables."""
    cache = kv16.Cache.alloc(1, 8, 16, 1, 64, T.bfloat16, 4, 2)
    cache.tables.copy_(T.arange(8, device="cuda").int().view(4, 2))
    m = kv16.Maps(cache, 3, 6)
    m(_ints(T, [3, 4, 5]), _ints(T, [2, 3, 4]))
    assert m.first.tolist() == [0, 2, 5, 6] and m.at.tolist() == [3, 4, 4, 5, 6, 5]
    assert sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE
    m(_ints(T, [3, -4, 31]), _ints(T, [-2, 3, 2]), rows=_ints(T, [0, 1, 9]))
    assert m.first.tolist() == [0, 0, 3, 5] and m.at.tolist() == [-1, -1, -1, 31, 32, -1] and m.slots.tolist() == [-1] * 6
    assert m.pos.tolist() == [-1, -1, -1, 31, 32, -1] and sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE
    m(_ints(T, [0, 30, 0]), _ints(T, [1, 3, 0]))
    assert m.slots.tolist() == [0, 3 * 16 + 14, 3 * 16 + 15, -1, -1, -1] and sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE


@pytest.mark.parametrize("D,norm", [(64, True), (96, False), (20, True)])
def test_cache_positions(T, D, norm):
    """K and V go to `at`, turned by `pos`: the rows that pos alone would put elsewhere; a negative one is not written."""
    n, H, page = 7, 2, 16
    caches = [kv16.Cache.alloc(1, 8, page, H, D, T.bfloat16, 2, 4) for _ in range(2)]
    g = T.Generator(device="cuda")
    g.manual_seed(1)
    q, k, v = (T.randn((n, h, D), device="cuda", generator=g).bfloat16() for h in (4, H, H))
    rows, pos, at = _ints(T, [0, 0, 0, 1, 1, 0, 1]), _ints(T, [40, 41, 41, 3, 9, 42, -1]), _ints(T, [40, 41, 42, 50, -1, 43, 60])
    w = T.rand(D, device="cuda", generator=g) if norm else None
    outs = []
    for c in caches:
        c.tables.copy_(T.arange(8, device="cuda").int().view(2, 4))
        step = kv16.Qkv(D, rope=kv16.Rope(D), q_norm=w, k_norm=w, cache=c)
        q2 = T.zeros_like(q)
        if c is caches[0]:
            step(q, k, v, pos, q_out=q2, rows=rows, at=at)
        else:
            kr, vr = T.zeros_like(k), T.zeros_like(v)
            step(q, k, v, pos, q_out=q2, k_out=kr, v_out=vr, rows=rows, to_cache=False)
            for t in range(n):
                if pos[t] >= 0 and at[t] >= 0:
                    page_id, place = int(c.tables[int(rows[t]), int(at[t]) // page]), int(at[t]) % page
                    c.k[0, page_id, place], c.v[0, page_id, place] = kr[t], vr[t]
        outs.append(q2)
    assert T.equal(outs[0], outs[1]) and T.equal(caches[0].k, caches[1].k) and T.equal(caches[0].v, caches[1].v)
    assert sjk.lib().sjk_device_status() == 0


@pytest.mark.parametrize("D,H,page", [(64, 1, 1), (96, 3, 5), (128, 8, 16), (256, 4, 128), (20, 2, 24)])
@pytest.mark.parametrize("width", [1, 9, 200])
def test_keep(T, D, H, page, width):
    """Every path of the batch in every layer, row by row."""
    r = random.Random(width)
    n, layers = 6, 3
    lens = [r.randint(0, 300) for _ in range(n)]
    cache, g = _cache(T, [x + 2 * width + 5 for x in lens], page, H, D, T.float16, layers=layers, junk=1.0)
    paths = [sorted(r.sample(range(2 * width + 5), r.randint(0, width))) for _ in range(n)]
    paths[0], paths[1] = list(range(width)), list(range(width + 5, 2 * width + 5))
    order = r.sample(range(n), n)
    want = []
    for c in (cache.k, cache.v):
        x = c.clone()
        for i, p in zip(order, paths):
            for j, t in enumerate(p):
                a, b = lens[i] + t, lens[i] + j
                x[:, int(cache.tables[i, b // page]), b % page] = c[:, int(cache.tables[i, a // page]), a % page]
        want.append(x)
    new = cache.keep(_ints(T, [lens[i] for i in order]), _ints(T, [p + [0] * (width - len(p)) for p in paths]),
                     _ints(T, [len(p) for p in paths]), rows=_ints(T, order))
    assert T.equal(cache.k, want[0]) and T.equal(cache.v, want[1])
    assert new.tolist() == [lens[i] + len(p) for i, p in zip(order, paths)] and sjk.lib().sjk_device_status() == 0


def test_keep_refusals_on_the_device(T):
    """Paths that do not ascend, places without a page, rows twice or out of range: that sequence stays as it is."""
    lens = [10, 10, 10, 10, 10, 10, 30, 10]
    cache, g = _cache(T, [x + 8 for x in lens], 16, 2, 64, T.bfloat16, junk=1.0)
    cache.tables[5, 1] = -1
    paths = [[1, 1], [2, 1], [-1, 3], [0, 1], [3, 5], [4, 7], [200, 201], [1, 2]]
    rows = [0, 1, 2, 3, 4, 5, 6, 4]
    k, v = cache.k.clone(), cache.v.clone()
    count = [2, 2, 2, 3, 2, 2, 2, 2]
    new = cache.keep(_ints(T, lens), _ints(T, paths), _ints(T, count), rows=_ints(T, rows))
    assert new.tolist() == [10, 10, 10, 10, 12, 10, 30, 10] and sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE
    for x, was in ((cache.k, k), (cache.v, v)):
        p = int(cache.tables[4, 0])
        was[0, p, 10], was[0, p, 11] = was[0, p, 13].clone(), was[0, p, 15].clone()
        assert T.equal(x, was)
    lens_d = _ints(T, lens)
    with pytest.raises(sjk.SjkError):
        cache.keep(lens_d, _ints(T, paths), _ints(T, count), rows=_ints(T, rows), new_lens=lens_d)


# ---- together ---------------------------------------------------------------------------------------------------------

def _rows(T, x, w, pos, D):
    """Norm and rotary positions of heads x [n][h][D] in 64 bits."""
    x = x.double()
    x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    ang = T.tensor(pos, dtype=T.float64, device="cuda")[:, None] * 1e4 ** (-2 * T.arange(D // 2, device="cuda").double() / D)
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = x[..., : D // 2], x[..., D // 2:]
    return T.cat((a * c - b * s, a * s + b * c), -1)


@pytest.mark.parametrize("captured", [False, True])
def test_decode_loop_with_trees(T, captured):
    """Steps of a draft-and-verify loop: pages for the drafts (shared prompts split), maps, norm, rotation and cache write at
    other places than the positions, attention of the tree, the accepted path kept, the others' pages given back. Each token's
    output is what the same token gives in a plain history of accepted ones; captured, the step replays with other lengths.
    Bound: K rows are rounded to bf16 once (2^-8 of a row's elements, half of it on average, in the scores) beside the kernel's own; 3 of
    the output's own roundings of the largest output element cover both (scores here are sums of at most |q| |k| 2^-8 <= 2^-8 sqrt(D) scale sqrt(D) = 2^-8 ... 0.05 of a weight)."""
    n, H, grp, D, page, N = 3, 2, 4, 64, 16, 8
    r = random.Random(5)
    cache = kv16.Cache.alloc(1, 64, page, H, D, T.bfloat16, n, 12)
    pages = cache.pages()
    g = T.Generator(device="cuda")
    g.manual_seed(3)
    wq, wk = (1 + 0.1 * T.randn(D, device="cuda", generator=g) for _ in range(2))
    step = kv16.Qkv(D, rope=kv16.Rope(D), q_norm=wq, k_norm=wk, cache=cache)
    rows, lens = _ints(T, list(range(n))), _ints(T, [0] * n)
    maps = kv16.Maps(cache, n, n * N)
    x = T.empty((n * N, (H * grp + 2 * H) * D), dtype=T.bfloat16, device="cuda")
    heads = [x[:, a * D: b * D].view(n * N, b - a, D) for a, b in ((0, H * grp), (H * grp, H * grp + H), (H * grp + H, H * grp + 2 * H))]
    q2, out = T.empty((n * N, H * grp, D), dtype=T.bfloat16, device="cuda"), T.empty((n * N, H * grp, D), dtype=T.bfloat16, device="cuda")
    add, masks = _ints(T, [N] * n), T.zeros(n * N, dtype=T.int64, device="cuda")
    path, count, new = T.zeros((n, N), dtype=T.int32, device="cuda"), T.zeros(n, dtype=T.int32, device="cuda"), T.zeros_like(lens)
    # a shared prompt of 21 tokens
    prompt = T.randn((21, (H * grp + 2 * H) * D), device="cuda", generator=g).bfloat16()
    ph = [prompt[:, a * D: b * D].view(21, b - a, D) for a, b in ((0, H * grp), (H * grp, H * grp + H), (H * grp + H, H * grp + 2 * H))]
    pages.extend(rows[:1], lens[:1], 21)
    step(k=ph[1], v=ph[2], pos=T.arange(21, dtype=T.int32, device="cuda"), rows=T.zeros(21, dtype=T.int32, device="cuda"))
    pages.fork(_ints(T, [0] * (n - 1)), rows[1:])
    lens.fill_(21)
    hist = [(_rows(T, ph[1], wk, list(range(21)), D), ph[2].double()) for _ in range(n)]

    def one():
        pages.extend(rows, lens, add)
        m = maps(lens, add, masks=masks)
        step(*heads, m.pos, q_out=q2, rows=m.rows, at=m.at)
        cache.attend_tree(0, q2, lens, masks, 1 / math.sqrt(D), first=m.first, nodes=N, out=out)
        cache.keep(lens, path, count, new_lens=new)
        lens.copy_(new)
        pages.free(rows, first=(new + page - 1) // page)

    graph = None
    for turn in range(12):
        trees = [_tree(r, N) for _ in range(n)]
        paths = []
        for t in trees:
            leaf = r.randrange(N)
            paths.append([k for k in range(N) if t[leaf] >> k & 1][: r.randint(1, N)])
        x.normal_(generator=g)
        masks.copy_(_ints(T, [m for t in trees for m in _signed(t)], T.int64))
        path.copy_(_ints(T, [p + [0] * (N - len(p)) for p in paths]))
        count.copy_(_ints(T, [len(p) for p in paths]))
        before = lens.tolist()
        if captured and turn == 1:
            graph = T.cuda.CUDAGraph()
            with T.cuda.graph(graph):
                one()
        if graph is not None:
            graph.replay()
        else:
            one()
        for i in range(n):
            sl = slice(i * N, (i + 1) * N)
            pos = [before[i] + bin(t).count("1") - 1 for t in trees[i]]
            k, v, q = _rows(T, heads[1][sl], wk, pos, D), heads[2][sl].double(), _rows(T, heads[0][sl], wq, pos, D)
            for j in range(N):
                on = [c for c in range(N) if trees[i][j] >> c & 1]
                K, V = T.cat((hist[i][0], k[on])), T.cat((hist[i][1], v[on]))
                w = T.softmax(T.einsum("hgd,thd->hgt", q[j].view(H, grp, D), K) / math.sqrt(D), -1)
                want = T.einsum("hgt,thd->hgd", w, V).reshape(-1, D)
                got = out[i * N + j].double()
                assert float((got - want).abs().max()) <= 3 * 2.0 ** -8 * float(V.abs().max()), f"turn {turn}, sequence {i}, token {j}"
            hist[i] = T.cat((hist[i][0], k[paths[i]])), T.cat((hist[i][1], v[paths[i]]))
        assert lens.tolist() == [b + len(p) for b, p in zip(before, paths)]
    used = 64 - pages.n_free.item()
    assert used == sum(-(-x // page) for x in lens.tolist()) - (n - 1) * (21 // page)
    assert sjk.lib().sjk_device_status() == 0
