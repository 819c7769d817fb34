"""How exact the attention over 16-bit pages is: softmax weights and queries of every size that 32-bit arithmetic keeps,
against the definition in 64 bits.

Error bound of an output element y, with A the same attention over |V|: u |y| for the rounding to the output type, and
(p + 2 e + a) A. p is the relative rounding of a weight: it is the sum of two terms of the cache's type, or of three for
bf16 caches with 32-bit rows: 2^-16 (two bf16 terms of 8 bits), 2^-22 (two f16 terms of 11), 2^-24 (three bf16 terms). e
bounds the error of a score in units of ln 2: 2^-20 (1 + max_t scale sum_d |q_d k_td|). a = 2^-23 (n / 16 + 8): the sums
of n positions, 16 at a time, each of which may drop what lies below 2^-23 of it, and the joins behind them."""
import math

import pytest

import sjk
from test_gpu_kv16 import _build, _dt, _expect

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    import build
    build.build()
    import torch
    assert torch.cuda.is_available()
    return torch


def _check(T, cache, got, q, lens, scale, window=0, rows=None, floor=0.0, few=False):
    """floor: what every element may be off beside the bound. few: one worker holds all of a sequence's few positions: e is
    2^-22 for ex2 and 2^-20 of the products, a one sum that may drop 2^-23 and at most 7 rounded additions and products."""
    split = q.dtype != cache.k.dtype or got.dtype == T.float32
    p = 2.0 ** -22 if cache.k.dtype == T.float16 else 2.0 ** -24 if split else 2.0 ** -16
    u = {T.float32: 2.0 ** -23, T.float16: 2.0 ** -11, T.bfloat16: 2.0 ** -8}[got.dtype]
    tiny = 2.0 ** -25 if got.dtype == T.float16 else 1e-37
    for i, x in enumerate(lens):
        want, mag_v, mag = _expect(T, cache, 0, i if rows is None else rows[i], x, q[i], scale, window)
        e, a = (2.0 ** -22 + 2.0 ** -20 * mag, 2.0 ** -23 + 7 * 2.0 ** -24) if few else (2.0 ** -20 * (1 + mag), 2.0 ** -23 * (x / 16 + 8))
        bound = u * want.abs() * (1 + 2.0 ** -7) + (p + 2 * e + a) * mag_v + tiny + floor
        err = (got[i].double().cpu() - want).abs()
        assert bool((err <= bound).all()), f"sequence {i} of length {x}: worst {float((err / bound).max()):.3g} of the bound"


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("grp", [1, 8, 13, 20])
@pytest.mark.parametrize("page", [16, 5])
def test_weights_of_16_bit_rows(T, dtype, D, grp, page):
    """Queries and outputs of the cache's type: what is off is the rounding of the output, not that of the weights (elements
    that nearly cancel would show it)."""
    lens = [1, 2, 3, 17, 64, 257, 1000]
    cache, g = _build(T, lens, page, 2, D, _dt(T, dtype), seed=grp)
    q = T.randn((len(lens), 2 * grp, D), device="cuda", generator=g).to(_dt(T, dtype))
    got = cache.attend(0, q, T.tensor(lens, dtype=T.int32, device="cuda"), 1 / math.sqrt(D))
    _check(T, cache, got, q, lens, 1 / math.sqrt(D))
    assert sjk.lib().sjk_device_status() == 0


def _peaked(T, dtype, io, out, D, gap, n, spread, many, seed=0):
    """Sequences whose first token stands `gap` nats above the others, with V = 0 there (an attention sink); the others'
    scores spread by `spread` nats. many: entries of that one table row, so that one worker holds a whole sequence."""
    grp, H = 4, 2
    cache, g = _build(T, [n], 16, H, D, _dt(T, dtype), seed=seed)
    q0 = T.randn((H, 1, D), device="cuda", generator=g)
    q = (q0 + 0.05 * T.randn((H, grp, D), device="cuda", generator=g)).reshape(1, H * grp, D).to(_dt(T, io))
    scale = 1 / math.sqrt(D)
    unit = q0[:, 0] / q0[:, 0].norm(dim=-1, keepdim=True)
    first = cache.tables[0, 0].item()
    others = T.arange(n, device="cuda")[1:]
    ids = cache.tables[0, others // 16].long()
    cache.k[0, ids, others % 16] = (spread / q0[:, 0].norm(dim=-1)[None, :, None] * math.sqrt(D) *
                                    T.randn((n - 1, H, 1), device="cuda", generator=g) * unit).to(cache.k.dtype)
    cache.k[0, first, 0] = (unit * gap * math.sqrt(D) / q0[:, 0].norm(dim=-1, keepdim=True)).to(cache.k.dtype)
    cache.v[0, first, 0] = 0
    qs = q.expand(many, -1, -1).contiguous()
    rows = T.zeros(many, dtype=T.int32, device="cuda")
    got = T.full(qs.shape, 9.0, dtype=_dt(T, out), device="cuda")
    cache.attend(0, qs, T.full((many,), n, dtype=T.int32, device="cuda"), scale, rows=rows, out=got)
    return cache, qs, got, scale


@pytest.mark.parametrize("dtype,io,out", [("f16", "f16", "f16"), ("f16", "f32", "f32"), ("f16", "f16", "f32"), ("f16", "bf16", "bf16"),
                                          ("bf16", "bf16", "bf16"), ("bf16", "f32", "f32")])
@pytest.mark.parametrize("gap", [10, 14, 17, 20, 25])
@pytest.mark.parametrize("many", [1, 1300])
@pytest.mark.parametrize("spread", [0.1, 1.0])
def test_tokens_far_below_the_largest(T, dtype, io, out, gap, many, spread):
    """What stands 10 to 25 nats below one token keeps its share: what a weight of an f16 cache loses beside its rounding is
    2^-40 of the largest in its worker's run, so n 2^-40 max |V| at most (l is at least the largest weight); bf16 has the
    range of 32 bits."""
    n, D = 2048, 128
    cache, q, got, scale = _peaked(T, dtype, io, out, D, gap, n, spread, many)
    floor = n * 2.0 ** -40 * float(cache.v[0, cache.tables[0, : n // 16].long()].abs().max()) if dtype == "f16" else 0.0
    some = [0] if many == 1 else [0, many // 2, many - 1]
    _check(T, cache, got[some], q[some], [n] * len(some), scale, rows=[0] * len(some), floor=floor)
    assert sjk.lib().sjk_device_status() == 0


@pytest.mark.parametrize("io,out", [("f16", "f16"), ("f16", "f32"), ("f32", "f32")])
def test_extreme_scores_of_f16_caches(T, io, out):
    """Large scores of both signs over an f16 cache, one token that takes all, scale 0 and a negative scale."""
    lens, D = [70, 700], 128
    cache, g = _build(T, lens, 16, 1, D, T.float16)
    q = (30 * T.randn((2, 4, D), device="cuda", generator=g)).to(_dt(T, io))
    dl = T.tensor(lens, dtype=T.int32, device="cuda")
    floor = 700 * 2.0 ** -40 * 6
    for scale in (1.0, -1.0, 0.0, 1e-3, 1e4, 1e8):
        got = T.full(q.shape, 9.0, dtype=_dt(T, out), device="cuda")
        cache.attend(0, q, dl, scale, out=got)
        if abs(scale) < 100:
            _check(T, cache, got, q, lens, scale, floor=floor)
        else:
            assert bool(T.isfinite(got).all())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("grp", [1, 3, 9])
@pytest.mark.parametrize("small", [8, 12, 16, 20])
def test_queries_with_one_large_channel(T, dtype, D, grp, small):
    """32-bit queries whose first channel, where K is 0, stands 2^small above the others. Two f16 terms keep 2^-39 of the
    largest channel: the scores of an f16 cache may be off by that beside the bound, bf16 has the range of 32 bits."""
    lens = [40, 300]
    cache, g = _build(T, lens, 16, 2, D, _dt(T, dtype), seed=D + small)
    cache.k[..., 0] = 0
    q = 2.0 ** -small * T.randn((2, 2 * grp, D), device="cuda", generator=g)
    q[..., 0] = 1.0
    scale = 2.0 ** small / math.sqrt(D)
    got = cache.attend(0, q, T.tensor(lens, dtype=T.int32, device="cuda"), scale)
    floor = 0.0
    if dtype == "f16":
        live = cache.k[0].nan_to_num(0.0).abs().sum(-1).max()
        floor = float(2 * 2.0 ** -39 * scale * live * cache.v[0].nan_to_num(0.0).abs().max())
    _check(T, cache, got, q, lens, scale, floor=floor)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("big", [1e36, 1e12, 1e-12, 1e-36])
def test_queries_at_the_ends_of_the_range(T, dtype, big):
    lens, D = [70, 700], 128
    cache, g = _build(T, lens, 16, 1, D, _dt(T, dtype))
    q = big * 30 * T.randn((2, 4, D), device="cuda", generator=g)
    got = cache.attend(0, q, T.tensor(lens, dtype=T.int32, device="cuda"), 0.1 / big)
    _check(T, cache, got, q, lens, 0.1 / big, floor=700 * 2.0 ** -40 * 6 + 2.0 ** -39 * 60)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("grp", [1, 2, 5, 16])
def test_weights_of_32_bit_rows(T, dtype, D, grp):
    """Scores of a size of 0.1 or less, whose own error is small: the rounding of the weights shows (with two bf16 terms of
    a weight in place of three, the worst element would be about twice the bound off)."""
    lens = [1, 2, 3, 5, 9]
    cache, g = _build(T, lens, 16, 2, D, _dt(T, dtype), seed=D + grp)
    q = T.randn((len(lens), 2 * grp, D), device="cuda", generator=g)
    got = cache.attend(0, q, T.tensor(lens, dtype=T.int32, device="cuda"), 0.1 / D)
    _check(T, cache, got, q, lens, 0.1 / D, few=True)


def test_graphs_captured_on_one_stream(T):
    """Two graphs of one cache, captured one after the other on the same stream, replayed at once on two streams beside calls
    that run on a third: each has scratch of its own."""
    lens, D = [5000, 4000], 128
    cache, g = _build(T, lens, 16, 4, D, T.bfloat16)
    dl = T.tensor(lens, dtype=T.int32, device="cuda")
    qs = [T.randn((2, 16, D), device="cuda", generator=g).bfloat16() for _ in range(3)]
    want = [cache.attend(0, q, dl, 0.1) for q in qs]
    outs, graphs, s = [[T.empty_like(want[0]) for _ in range(4)] for _ in range(2)], [T.cuda.CUDAGraph() for _ in range(2)], T.cuda.Stream()
    T.cuda.synchronize()
    for j in range(2):
        with T.cuda.graph(graphs[j], stream=s):
            for out in outs[j]:
                cache.attend(0, qs[j], dl, 0.1, out=out)
    assert set(key[0] for key in cache._scratch) == {T.cuda.current_stream().cuda_stream}
    streams = [T.cuda.Stream() for _ in range(3)]
    for _ in range(20):
        for j in range(2):
            with T.cuda.stream(streams[j]):
                graphs[j].replay()
        with T.cuda.stream(streams[2]):
            mine = cache.attend(0, qs[2], dl, 0.1)
        T.cuda.synchronize()
        assert all(T.equal(o, want[j]) for j in range(2) for o in outs[j]) and T.equal(mine, want[2])
        for j in range(2):
            for o in outs[j]:
                o.zero_()
        T.cuda.synchronize()


def test_scratch_of_the_callers(T):
    lens, D = [700, 3], 64
    cache, g = _build(T, lens, 16, 2, D, T.float16)
    dl = T.tensor(lens, dtype=T.int32, device="cuda")
    q = T.randn((2, 8, D), device="cuda", generator=g).half()
    mine = T.empty(cache.scratch_bytes(8), dtype=T.uint8, device="cuda")
    assert T.equal(cache.attend(0, q, dl, 0.1, scratch=mine), cache.attend(0, q, dl, 0.1))
    with pytest.raises(sjk.SjkError):
        cache.attend(0, q, dl, 0.1, scratch=mine[:1024])
