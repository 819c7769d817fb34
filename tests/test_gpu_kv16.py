"""sjk_kv16_attend (one new token per sequence over paged 16-bit caches) against the definition in 64 bits.

Error bound of an output element y, with A the same attention over |V|: u |y| for the rounding to the output type,
(p + 2 e) A for the rounded weights and the scores behind them. p is the relative rounding of a weight: 2^-8 (bf16) or
2^-11 (f16) where queries and outputs are of the cache's type, else 2^-16 and 2^-21 (two terms). e bounds the error of a
score in units of ln 2: 2^-20 (1 + max_t scale sum_d |q_d k_td|), from 32-bit sums of exact 16-bit products (at most 256
terms in chains of 16), the scale's product, the difference to the maximum and ex2 (2^-22)."""
import math

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


def _build(T, lens, page, H, D, dtype, seed=0, layers=1, junk=math.nan):
    """A cache whose live positions are normal values and whose other slots (tails of pages, pages of nobody) are junk."""
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
        for c in (cache.k, cache.v):
            c[:, ids[t // page], t % page] = T.randn((layers, x, H, D), device="cuda", generator=g).to(dtype)
    return cache, g


def _expect(T, cache, layer, row, length, q, scale, window):
    """(out, out over |V|, score bound) of one sequence in 64 bits: [heads][D]; positions without a page left out."""
    P, H, D = cache.page_tokens, cache.n_head_kv, cache.head_dim
    lo = max(0, length - window) if window else 0
    t = T.arange(lo, max(length, lo), device="cuda")
    ids = cache.tables[row, t // P].long()
    t, ids = t[ids >= 0], ids[ids >= 0]
    q = q.double().view(H, -1, D)
    if t.numel() == 0:
        z = T.zeros((q.shape[0] * q.shape[1], D), dtype=T.float64)
        return z, z, 0.0
    k, v = (c[layer][ids, t % P].double() for c in (cache.k, cache.v))
    s = T.einsum("hgd,thd->hgt", q, k) * scale
    mag = float((T.einsum("hgd,thd->hgt", q.abs(), k.abs()) * abs(scale)).max())
    w = T.softmax(s, -1)
    return T.einsum("hgt,thd->hgd", w, v).reshape(-1, D).cpu(), T.einsum("hgt,thd->hgd", w, v.abs()).reshape(-1, D).cpu(), mag


def _check(T, cache, got, q, lens, scale, window=0, rows=None, layer=0):
    split = q.dtype != cache.k.dtype or got.dtype == T.float32
    bf = cache.k.dtype == T.bfloat16
    p = (2.0 ** -16 if bf else 2.0 ** -21) if split else (2.0 ** -8 if bf else 2.0 ** -11)
    u = {T.float32: 2.0 ** -23, T.float16: 2.0 ** -11, T.bfloat16: 2.0 ** -8}[got.dtype]
    tiny = 2.0 ** -25 if got.dtype == T.float16 else 1e-37
    for i, x in enumerate(lens):
        want, mag_v, mag = _expect(T, cache, layer, i if rows is None else rows[i], x, q[i], scale, window)
        e = 2.0 ** -20 * (1 + mag)
        bound = u * want.abs() * (1 + 2.0 ** -7) + (p + 2 * e) * mag_v + tiny
        err = (got[i].double().cpu() - want).abs()
        assert bool((err <= bound).all()), f"sequence {i} of length {x}: worst {float((err / bound).max()):.3g} of the bound"


LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 100, 257, 1000]


@pytest.mark.parametrize("dtype,io,out", [("bf16", "bf16", "bf16"), ("f16", "f16", "f16"), ("f16", "f32", "f32"), ("bf16", "f32", "f32"),
                                          ("bf16", "f16", "bf16"), ("f16", "f16", "f32"), ("bf16", "bf16", "f16")])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("grp", [1, 4, 7, 8, 9, 16, 17, 40])
def test_types_heads_lengths(T, dtype, io, out, D, grp):
    H, page = 2, 16
    cache, g = _build(T, LENS, page, H, D, _dt(T, dtype), seed=D + grp)
    q = (1.5 * T.randn((len(LENS), H * grp, D), device="cuda", generator=g)).to(_dt(T, io))
    got = T.full(q.shape, 9.0, dtype=_dt(T, out), device="cuda")
    lens = T.tensor(LENS, dtype=T.int32, device="cuda")
    cache.attend(0, q, lens, 1 / math.sqrt(D), out=got)
    _check(T, cache, got, q, LENS, 1 / math.sqrt(D))
    assert sjk.lib().sjk_device_status() == 0


@pytest.mark.parametrize("page", [1, 5, 16, 24, 32, 100, 128])
@pytest.mark.parametrize("window", [0, 1, 16, 17, 40, 5000])
@pytest.mark.parametrize("D", [64, 128])
def test_pages_and_windows(T, page, window, D):
    """Pages that end inside a step, and windows that begin inside one; a window's passed pages may be gone."""
    cache, g = _build(T, LENS, page, 2, D, T.float16, seed=page + window)
    if window:
        for i, x in enumerate(LENS):
            cache.tables[i, : max(0, x - window) // page] = -1
    q = T.randn((len(LENS), 4, D), device="cuda", generator=g).half()
    got = cache.attend(0, q, T.tensor(LENS, dtype=T.int32, device="cuda"), 0.11, window=window)
    _check(T, cache, got, q, LENS, 0.11, window)
    assert sjk.lib().sjk_device_status() == 0


@pytest.mark.parametrize("n,top", [(1, 1), (1, 5000), (3, 100000), (40, 700), (300, 90), (1100, 5)])
@pytest.mark.parametrize("H,grp,D", [(1, 4, 128), (4, 4, 256), (8, 1, 64)])
def test_batches(T, n, top, H, grp, D):
    """From one sequence that every worker shares to more sequences than workers, ragged, rows in any order."""
    import random
    r = random.Random(n)
    lens = [r.randint(0, top) for _ in range(n)]
    lens[-1] = top
    cache, g = _build(T, lens, 16, H, D, T.bfloat16, seed=n, junk=math.inf)
    order = list(range(n))
    r.shuffle(order)
    q = T.randn((n, H * grp, D), device="cuda", generator=g).bfloat16()
    rows = T.tensor(order, dtype=T.int32, device="cuda")
    lens2 = [lens[i] for i in order]
    dl = T.tensor(lens2, dtype=T.int32, device="cuda")
    got = cache.attend(0, q, dl, 0.1, rows=rows)
    _check(T, cache, got, q, lens2, 0.1, rows=order)
    assert T.equal(got, cache.attend(0, q, dl, 0.1, rows=rows))            # the same bits again


def test_no_sequences(T):
    cache, g = _build(T, [5], 16, 2, 64, T.bfloat16)
    q = T.empty((0, 4, 64), dtype=T.bfloat16, device="cuda")
    assert cache.attend(0, q, T.empty(0, dtype=T.int32, device="cuda"), 0.1).shape == q.shape


def test_layouts(T):
    """Heads before slots, and K and V interleaved in one buffer, give the bits of the plain layout."""
    lens, page, H, D = [3, 200, 77], 16, 2, 128
    cache, g = _build(T, lens, page, H, D, T.float16)
    q = T.randn((3, 8, D), device="cuda", generator=g).half()
    dl = T.tensor(lens, dtype=T.int32, device="cuda")
    want = cache.attend(0, q, dl, 0.1)
    n = cache.k.shape[1]
    hk, hv = (T.empty((1, n, H, page, D), dtype=T.float16, device="cuda").transpose(2, 3) for _ in range(2))
    both = T.empty((1, n, page, H, 2, D), dtype=T.float16, device="cuda")
    for k, v in ((hk, hv), (both[..., 0, :], both[..., 1, :])):
        k.copy_(cache.k)
        v.copy_(cache.v)
        assert T.equal(kv16.Cache(k, v, cache.tables).attend(0, q, dl, 0.1), want)
    # queries and outputs of other strides
    qt = T.empty((8, 3, D), dtype=T.float16, device="cuda").transpose(0, 1)
    qt.copy_(q)
    out = T.empty((8, 3, D), dtype=T.float16, device="cuda").transpose(0, 1)
    assert T.equal(cache.attend(0, qt, dl, 0.1, out=out), want)


def test_holes_and_bad_entries(T):
    """Positions on a missing page are left out, silently for SJKVARN_NO_BLOCK and with SJK_DEVICE_PAGE for ids, rows and
    lengths out of range; a sequence with no page left gives zeros."""
    lens, page, D = [100, 100, 60, 64], 16, 64
    cache, g = _build(T, lens, page, 2, D, T.bfloat16)
    cache.tables[0, 2] = -1
    cache.tables[2] = -1
    q = T.randn((4, 4, D), device="cuda", generator=g).bfloat16()
    dl = T.tensor(lens, dtype=T.int32, device="cuda")
    got = cache.attend(0, q, dl, 0.1)
    _check(T, cache, got, q, lens, 0.1)
    assert bool((got[2] == 0).all()) and sjk.lib().sjk_device_status() == 0
    cache.tables[1, 3] = cache.k.shape[1]
    got = cache.attend(0, q, dl, 0.1)
    cache.tables[1, 3] = -1
    _check(T, cache, got, q, lens, 0.1)
    assert sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE
    stride = cache.tables.shape[1]
    cache.tables[3, 4:] = -1
    got = cache.attend(0, q[3:], T.tensor([stride * page + 1000], dtype=T.int32, device="cuda"), 0.1, rows=T.tensor([3], dtype=T.int32, device="cuda"))
    _check(T, cache, got, q[3:], [64], 0.1, rows=[3])
    assert sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE
    got = cache.attend(0, q[:2], T.tensor([64, -5], dtype=T.int32, device="cuda"), 0.1, rows=T.tensor([9, 0], dtype=T.int32, device="cuda"))
    assert bool((got == 0).all()) and sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE


@pytest.mark.parametrize("io", ["bf16", "f32"])
def test_extreme_scores(T, io):
    """Large scores of both signs, one token that takes all, scale 0 and a negative scale."""
    lens, D = [70, 70], 128
    cache, g = _build(T, lens, 16, 1, D, T.bfloat16)
    q = (30 * T.randn((2, 4, D), device="cuda", generator=g)).to(_dt(T, io))
    dl = T.tensor(lens, dtype=T.int32, device="cuda")
    for scale in (1.0, -1.0, 0.0, 1e-3, 1e4):
        out = cache.attend(0, q, dl, scale)
        if abs(scale) < 100:
            _check(T, cache, out, q, lens, scale)
        else:
            assert bool(T.isfinite(out).all())
    # a query far below or above the 16-bit range as a 32-bit row
    if io == "f32":
        for big in (1e-12, 1e12):
            out = cache.attend(0, q * big, dl, 0.1 / big)
            _check(T, cache, out, q * big, lens, 0.1 / big)


def test_offsets_past_32_bits(T):
    """A cache of more than 2^32 elements: pages at its far end are read and written where they are."""
    page, H, D = 128, 4, 256
    n_pages = 2 ** 32 // (page * H * D) + 8
    k, v = (T.empty((1, n_pages, page, H, D), dtype=T.bfloat16, device="cuda") for _ in range(2))
    tables = T.tensor([[n_pages - 1, 0, n_pages - 3]], dtype=T.int32, device="cuda")
    g = T.Generator(device="cuda")
    g.manual_seed(2)
    for i in (0, n_pages - 3, n_pages - 1):
        k[0, i].normal_(generator=g)
        v[0, i].normal_(generator=g)
    cache = kv16.Cache(k, v, tables)
    q = T.randn((1, 16, D), device="cuda", generator=g).bfloat16()
    new = T.randn((1, H, D), device="cuda", generator=g).bfloat16()
    kv16.Qkv(D, cache=cache)(k=new, v=new, pos=T.tensor([300], dtype=T.int32, device="cuda"))
    assert T.equal(k[0, n_pages - 3, 300 - 256], new[0]) and T.equal(v[0, n_pages - 3, 300 - 256], new[0])
    got = cache.attend(0, q, T.tensor([301], dtype=T.int32, device="cuda"), 1 / 16)
    _check(T, cache, got, q, [301], 1 / 16)


def test_graph_replays_with_new_lengths(T):
    """A captured step (pages, projection to cache, attention) replays: positions, tables and lengths are device memory."""
    n, H, grp, D, page = 3, 2, 4, 64, 16
    cache = kv16.Cache.alloc(1, 40, page, H, D, T.float16, n, 8)
    pages = cache.pages()
    rows = T.arange(n, dtype=T.int32, device="cuda")
    lens = T.zeros(n, dtype=T.int32, device="cuda")
    x = T.empty((n, (H * grp + 2 * H) * D), dtype=T.float16, device="cuda")
    q, k, v = x[:, : H * grp * D].view(n, -1, D), x[:, H * grp * D: (H * grp + H) * D].view(n, H, D), x[:, (H * grp + H) * D:].view(n, H, D)
    q2, out = T.empty((n, H * grp, D), dtype=T.float16, device="cuda"), T.empty((n, H * grp, D), dtype=T.float16, device="cuda")
    step = kv16.Qkv(D, rope=kv16.Rope(D), cache=cache)

    def one():
        pages.extend(rows, lens, 1)
        step(q, k, v, lens, q_out=q2, rows=rows)
        lens.add_(1)
        cache.attend(0, q2, lens, 0.125, rows=rows, out=out)

    T.manual_seed(0)
    s = T.cuda.Stream()
    s.wait_stream(T.cuda.current_stream())
    graph = T.cuda.CUDAGraph()
    x.normal_()
    with T.cuda.stream(s):
        one()
    T.cuda.current_stream().wait_stream(s)
    with T.cuda.graph(graph, stream=s):
        one()
    for i in range(35):
        x.normal_()
        graph.replay()
    assert lens.tolist() == [36] * n
    _check(T, cache, out, q2, [36] * n, 0.125)
    assert pages.n_free.item() == 40 - 3 * n and sjk.lib().sjk_device_status() == 0


def test_two_streams(T):
    """Calls of one cache on two streams at once keep their own scratch."""
    lens, D = [5000, 4000], 128
    cache, g = _build(T, lens, 16, 4, D, T.bfloat16)
    dl = T.tensor(lens, dtype=T.int32, device="cuda")
    qs = [T.randn((2, 16, D), device="cuda", generator=g).bfloat16() for _ in range(2)]
    want = [cache.attend(0, q, dl, 0.1) for q in qs]
    T.cuda.synchronize()
    streams = [T.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for i in range(20):
        for j, s in enumerate(streams):
            with T.cuda.stream(s):
                outs[j].append(cache.attend(0, qs[j], dl, 0.1))
    T.cuda.synchronize()
    for j in range(2):
        assert all(T.equal(o, want[j]) for o in outs[j])


@pytest.mark.parametrize("dtype,io", [("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("page", [1, 3, 24, 40])
def test_small_pages(T, dtype, io, D, page):
    """Pages that are no multiple of 16 tokens: ragged sequences in any order of rows, a long one, missing pages, windows
    and ids out of range."""
    import random
    r = random.Random(page + D)
    lens = [r.choice([0, 1, 31, 32, 33, 63, 64, 65, r.randint(1, 700)]) for _ in range(40)] + [9001]
    cache, g = _build(T, lens, page, 2, D, _dt(T, dtype), seed=page)
    for i, x in enumerate(lens):
        for _ in range(2 if x > 200 else 0):
            cache.tables[i, r.randrange((x - 1) // page)] = -1                      # (the last page stays)
    order = list(range(len(lens)))
    r.shuffle(order)
    q = T.randn((len(lens), 10, D), device="cuda", generator=g).to(_dt(T, io))
    rows, mine = T.tensor(order, dtype=T.int32, device="cuda"), [lens[i] for i in order]
    dl = T.tensor(mine, dtype=T.int32, device="cuda")
    for window in (0, 50):
        got = cache.attend(0, q, dl, 0.1, window=window, rows=rows)
        _check(T, cache, got, q, mine, 0.1, window, rows=order)
    assert sjk.lib().sjk_device_status() == 0
    at = order.index(len(lens) - 1)
    cache.tables[len(lens) - 1, 4000 // page] = cache.k.shape[1]
    got = cache.attend(0, q, dl, 0.1, rows=rows)
    assert sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE
    cache.tables[len(lens) - 1, 4000 // page] = -1
    _check(T, cache, got[at:at + 1], q[at:at + 1], [9001], 0.1, rows=[len(lens) - 1])


@pytest.mark.parametrize("page,window", [(2 ** 20 + 8, 1000000), (2 ** 20 + 8, 1040000), (2 ** 20, 1000000), (2 ** 20, 1050000)])
def test_longest_sequence(T, page, window):
    """The last positions below 2^31 - 1, in one page and over two, whose tokens are and are no multiple of 16."""
    D, length = 64, 2 ** 31 - 1
    cache = kv16.Cache.alloc(1, 2, page, 1, D, T.bfloat16, 1, 2048)
    g = T.Generator(device="cuda")
    g.manual_seed(page)
    cache.k.normal_(generator=g)
    cache.v.normal_(generator=g)
    cache.tables.fill_(-1)
    cache.tables[0, 2046:] = T.tensor([1, 0], dtype=T.int32, device="cuda")
    q = T.randn((1, 2, D), device="cuda", generator=g).bfloat16()
    got = cache.attend(0, q, T.tensor([length], dtype=T.int32, device="cuda"), 0.5, window=window)
    _check(T, cache, got, q, [length], 0.5, window)
    assert sjk.lib().sjk_device_status() == 0
