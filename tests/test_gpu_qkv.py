"""sjk_qkv (norm of every head, rotary positions, cache write) against the definition in 64 bits.

Error bound of an element y of a head: u |y| for the one rounding to the output type (u = 2^-8 bf16, 2^-11 f16, 2^-24
f32, plus half of f16's smallest step), and 2^-19 of the row's largest value for the 32-bit arithmetic before it: at
most 512 squares summed in lanes of 16 and a butterfly (under 2^-20 of the mean, halved by the root), a reciprocal
root and three products (2^-22 each), cosine and sine to 2^-22, the angle to pi 2^-24."""
import math

import pytest

import gpu_util as gu
import kv16
import sjk

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.fixture(scope="module")
def T():
    import build
    build.build()
    import torch
    assert torch.cuda.is_available()
    return torch


def _dt(T, name):
    return {"f32": T.float32, "f16": T.float16, "bf16": T.bfloat16}[name]


def _ulp(T, dtype):
    return {T.float32: 2.0 ** -24, T.float16: 2.0 ** -11, T.bfloat16: 2.0 ** -8}[dtype]


def _freq(n_rot, base, scaling, factor):
    step, amp = kv16.rope_steps(n_rot, base=base, scaling=scaling, factor=factor, n_ctx=4096)
    return step, amp


def _want(T, x, w, bias, pos, n_rot, layout, rope):
    """x [n][heads][D] in 64 bits through norm and rotation; the angles from the fixed-point table, exactly."""
    x = x.double().cpu()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * (w.double().cpu() + bias)
    if rope is None:
        return x
    step, amp = rope
    ang = T.tensor([[(int(p) * s % 2 ** 64) * 2.0 ** -64 * 2 * math.pi for s in step] for p in pos.tolist()], dtype=T.float64)
    c, s = (ang.cos() * amp)[:, None], (ang.sin() * amp)[:, None]
    y = x.clone()
    if layout == "half":
        a, b = x[..., : n_rot // 2], x[..., n_rot // 2: n_rot]
        y[..., : n_rot // 2], y[..., n_rot // 2: n_rot] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., 0:n_rot:2], x[..., 1:n_rot:2]
        y[..., 0:n_rot:2], y[..., 1:n_rot:2] = a * c - b * s, a * s + b * c
    return y


def _close(T, got, want, amp=1.0):
    """got within the file's bound of want ([..., D])."""
    u = _ulp(T, got.dtype)
    tiny = 2.0 ** -25 if got.dtype == T.float16 else 0.0
    bound = u * want.abs() * (1 + 2.0 ** -8) + 2.0 ** -19 * max(amp, 1.0) * want.abs().amax(-1, keepdim=True) + tiny
    err = (got.double().cpu() - want).abs()
    assert bool((err <= bound).all()), f"worst {float((err / bound.clamp(min=1e-300)).max()):.3g} of the bound"


def _inputs(T, n, HQ, H, D, dtype, seed, far=5000):
    g = T.Generator(device="cuda")
    g.manual_seed(seed)
    x = T.randn((n, (HQ + 2 * H) * D), dtype=T.float32, device="cuda", generator=g).to(dtype)
    pos = T.randint(0, far, (n,), generator=g, device="cuda").int()
    w = [1 + 0.2 * T.randn(D, device="cuda", generator=g) for _ in range(2)]
    q, k, v = (x[:, a * D: b * D].view(n, b - a, D) for a, b in ((0, HQ), (HQ, HQ + H), (HQ + H, HQ + 2 * H)))
    return q, k, v, pos, w


def _cache(T, n_rows, stride, page, H, D, dtype, seed=1):
    g = T.Generator(device="cuda")
    g.manual_seed(seed)
    pages = n_rows * stride
    c = kv16.Cache.alloc(2, pages, page, H, D, dtype, n_rows, stride)
    c.k.normal_(generator=g)
    c.v.normal_(generator=g)
    c.tables.copy_(T.randperm(pages, generator=g, device="cuda").int().view(n_rows, stride))
    return c


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("layout", ["half", "pair"])
@pytest.mark.parametrize("D,n_rot", [(64, 64), (96, 32), (128, 128), (256, 64), (512, 512), (128, 20), (80, 80), (66, 66), (2, 2), (64, 0)])
def test_rows_and_pages(T, dtype, layout, D, n_rot):
    """Norm, rotation, row outputs and the cache write at once, 5 tokens at scattered positions of 5 table rows."""
    dt = _dt(T, dtype)
    n, HQ, H, page, stride = 5, 6, 2, 24, 7
    q, k, v, pos, w = _inputs(T, n, HQ, H, D, dt, D + n_rot, far=page * stride)
    ct = T.bfloat16 if dt == T.float32 else dt
    cache = _cache(T, n, stride, page, H, D, ct)
    before = cache.k.clone(), cache.v.clone()
    rope = kv16.Rope(n_rot, layout=layout, base=1e4) if n_rot else None
    step = kv16.Qkv(D, rope=rope, q_norm=w[0], k_norm=w[1], norm_bias=0.25, eps=EPS, cache=cache)
    q_out = T.empty((n, HQ, D), dtype=dt, device="cuda")
    k_out, v_out = T.empty((n, H, D), dtype=dt, device="cuda"), T.empty((n, H, D), dtype=T.float32, device="cuda")
    step(q, k, v, pos, q_out=q_out, k_out=k_out, v_out=v_out, layer=1)
    steps = _freq(n_rot, 1e4, "none", 1.0) if n_rot else None
    _close(T, q_out, _want(T, q, w[0], 0.25, pos, n_rot, layout, steps))
    want_k = _want(T, k, w[1], 0.25, pos, n_rot, layout, steps)
    _close(T, k_out, want_k)
    assert T.equal(v_out, v.float())
    assert T.equal(cache.k[0], before[0][0]) and T.equal(cache.v[0], before[1][0])      # the other layer
    at = cache.tables[T.arange(n, device="cuda"), (pos // page).long()].long(), (pos % page).long()
    _close(T, cache.k[1][at], want_k)
    assert T.equal(cache.v[1][at], v.to(ct))
    for now, old in ((cache.k, before[0]), (cache.v, before[1])):                        # and nothing else
        rest = T.ones(now.shape[1:3], dtype=T.bool, device="cuda")
        rest[at] = False
        assert T.equal(now[1][rest], old[1][rest])
    assert sjk.lib().sjk_device_status() == 0


@pytest.mark.parametrize("n", [1, 2, 63, 147, 1183, 1185, 9000])
@pytest.mark.parametrize("D,HQ,H", [(128, 8, 2), (256, 16, 4), (64, 5, 5), (32, 1, 1), (16, 3, 1)])
def test_token_counts(T, n, D, HQ, H):
    """One token to many, on both sides of the kernel's choice of tokens per CTA."""
    q, k, v, pos, w = _inputs(T, n, HQ, H, D, T.bfloat16, n)
    rope = kv16.Rope(D, base=1e6)
    q_out, k_out, v_out = T.empty_like(q), T.empty_like(k), T.empty_like(v)
    kv16.Qkv(D, rope=rope, q_norm=w[0], eps=EPS)(q, k, v, pos, q_out=q_out, k_out=k_out, v_out=v_out)
    steps = _freq(D, 1e6, "none", 1.0)
    some = sorted({0, n // 3, n // 2, n - 1})
    _close(T, q_out[some], _want(T, q[some], w[0], 0.0, pos[some], D, "half", steps))
    _close(T, k_out[some], _want(T, k[some], None, 0.0, pos[some], D, "half", steps))
    assert T.equal(v_out, v)
    # every token: the same values whatever the batch it came in
    one = T.empty_like(q)
    step = kv16.Qkv(D, rope=rope, q_norm=w[0], eps=EPS)
    for t in range(0, n, 100):
        step(q=q[t:t + 100], pos=pos[t:t + 100], q_out=one[t:t + 100])
    assert T.equal(one, q_out)


@pytest.mark.parametrize("scaling,factor", [("linear", 4.0), ("ntk", 8.0), ("yarn", 8.0), ("bands", 8.0)])
@pytest.mark.parametrize("layout", ["half", "pair"])
def test_far_positions(T, scaling, factor, layout):
    """Positions up to 2^31 - 1 lose nothing: the bound is the one of position 0."""
    D = 128
    q, _, _, _, _ = _inputs(T, 6, 4, 1, D, T.float32, 5)
    pos = T.tensor([0, 1, 99999, 1048575, 2 ** 30 + 12345, 2 ** 31 - 1], dtype=T.int32, device="cuda")
    out = T.empty_like(q)
    rope = kv16.Rope(D, layout=layout, base=1e4, scaling=scaling, factor=factor, n_ctx=4096)
    kv16.Qkv(D, rope=rope)(q=q, pos=pos, q_out=out)
    steps = _freq(D, 1e4, scaling, factor)
    _close(T, out, _want(T, q, None, 0.0, pos, D, layout, steps), amp=steps[1])


@pytest.mark.parametrize("D,n_rot", [(128, 128), (128, 64), (96, 20)])
@pytest.mark.parametrize("layout", ["half", "pair"])
def test_in_place(T, D, n_rot, layout):
    """Outputs over the inputs' own rows equal outputs elsewhere, bit for bit."""
    q, k, v, pos, w = _inputs(T, 70, 4, 2, D, T.float16, 3)
    rope = kv16.Rope(n_rot, layout=layout)
    step = kv16.Qkv(D, rope=rope, q_norm=w[0], k_norm=w[1])
    q2, k2 = T.empty_like(q), T.empty_like(k)
    step(q, k, v, pos, q_out=q2, k_out=k2)
    step(q, k, v, pos, q_out=q, k_out=k)
    assert T.equal(q, q2) and T.equal(k, k2)


@pytest.mark.parametrize("case", ["order", "odd stride", "odd start"])
def test_strides(T, case):
    """Heads before tokens, rows off the vector width and rows off 16 bytes give what contiguous rows give, to the bound."""
    n, H, D = 9, 3, 64
    base, _, _, pos, w = _inputs(T, n, H, 1, D, T.bfloat16, 8)
    base = base.contiguous()
    if case == "order":
        x = T.empty((H, n, D), dtype=T.bfloat16, device="cuda").transpose(0, 1)
    elif case == "odd stride":
        x = T.empty((n, H, D + 3), dtype=T.bfloat16, device="cuda")[..., :D]
    else:
        x = T.empty(n * H * D + 1, dtype=T.bfloat16, device="cuda")[1:].view(n, H, D)
    x.copy_(base)
    out = T.empty_like(base)
    kv16.Qkv(D, rope=kv16.Rope(D), q_norm=w[0])(q=x, pos=pos, q_out=out)
    _close(T, out, _want(T, base, w[0], 0.0, pos, D, "half", _freq(D, 1e4, "none", 1.0)))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 66])
def test_padding_and_missing_pages(T, dtype, D):
    """A negative position writes nothing at all; a token whose page is missing, out of range or beyond its table keeps
    its row outputs, leaves the cache alone and sets SJK_DEVICE_PAGE."""
    dt = _dt(T, dtype)
    n, HQ, H, page, stride = 6, 2, 1, 16, 3
    q, k, v, _, w = _inputs(T, n, HQ, H, D, dt, 4)
    cache = _cache(T, 4, stride, page, H, D, dt)
    cache.tables[1, 1] = -1
    cache.tables[2, 0] = cache.k.shape[1]
    rows = T.tensor([0, 0, 1, 2, 3, 4], dtype=T.int32, device="cuda")
    pos = T.tensor([5, -1, 20, 3, page * stride, 1], dtype=T.int32, device="cuda")      # fine, padding, no page, bad page, beyond, bad row
    before = cache.k.clone(), cache.v.clone()
    q_out = T.full((n, HQ, D), 7.0, dtype=dt, device="cuda")
    step = kv16.Qkv(D, rope=kv16.Rope(D), cache=cache)
    assert sjk.lib().sjk_device_status() == 0
    step(q, k, v, pos, q_out=q_out, rows=rows)
    assert sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE
    assert sjk.lib().sjk_device_status() == 0
    assert bool((q_out[1] == 7.0).all())
    live = [0, 2, 3, 4, 5]
    _close(T, q_out[live], _want(T, q[live], None, 0.0, pos[live], D, "half", _freq(D, 1e4, "none", 1.0)))
    p0 = int(cache.tables[0, 0])
    for now, old in ((cache.k, before[0]), (cache.v, before[1])):
        assert not T.equal(now[0, p0, 5], old[0, p0, 5])
        now[0, p0, 5] = old[0, p0, 5]
        assert T.equal(now, old)


def test_values_at_the_edges(T):
    """A row of zeros stays zero under the norm, infinities and NaN stay in their head, and f16 rounds past its range to
    infinity as torch does."""
    D = 64
    x = T.zeros((5, 2, D), dtype=T.float32, device="cuda")
    x[1], x[2, 0, 3], x[3, 0, 5], x[4] = 1.0, math.inf, math.nan, 70000.0
    pos = T.zeros(5, dtype=T.int32, device="cuda")
    out = T.empty((5, 2, D), dtype=T.float16, device="cuda")
    kv16.Qkv(D, rope=kv16.Rope(D))(q=x, pos=pos, q_out=out)
    assert bool((out[0] == 0).all()) and bool((out[1] == 1).all()) and bool(T.isinf(out[4]).all())
    assert bool(T.isfinite(out[2, 1]).all()) and bool(T.isfinite(out[3, 1]).all()) and not bool(T.isfinite(out[2, 0, 3]))
    kv16.Qkv(D, q_norm=T.ones(D, device="cuda"))(q=x, q_out=out)
    assert bool((out[0] == 0).all())
    _close(T, out[1], T.ones((2, D), dtype=T.float64) / math.sqrt(1 + EPS))


def test_another_stream_and_no_tokens(T):
    """The call runs on torch's current stream; an empty batch does nothing."""
    D = 128
    q, _, _, pos, _ = _inputs(T, 300, 8, 1, D, T.bfloat16, 6)
    out = T.zeros_like(q)
    step = kv16.Qkv(D, rope=kv16.Rope(D))
    s = T.cuda.Stream()
    s.wait_stream(T.cuda.current_stream())
    with T.cuda.stream(s):
        step(q=q, pos=pos, q_out=out)
        again = out.clone()
    s.synchronize()
    _close(T, again, _want(T, q, None, 0.0, pos, D, "half", _freq(D, 1e4, "none", 1.0)))
    step(q=q[:0], pos=pos[:0], q_out=out[:0])


def test_rows_feed_the_sealed_cache(T):
    """K and V as 32-bit rows go straight into sjk_store: the staged bytes equal those of the same rows made outside."""
    import ctypes as C
    L = sjk.lib()
    D, H, n = 256, 4, 300
    cfg = sjk.config(D, H, 2048, 512, tail=256, tail_max=512)
    layer = [sjk.Layer(), sjk.Layer()]
    for x in layer:
        sjk.check(L.sj_kvarn_layer_init(C.byref(x), C.byref(cfg)))
    q, k, v, _, w = _inputs(T, n, 16, H, D, T.bfloat16, 9)
    pos = T.arange(n, dtype=T.int32, device="cuda")
    rows = [T.empty((n, H, D), dtype=T.float32, device="cuda") for _ in range(2)]
    kv16.Qkv(D, rope=kv16.Rope(D), k_norm=w[1])(k=k, v=v, pos=pos, k_out=rows[0], v_out=rows[1])
    _close(T, rows[0], _want(T, k, w[1], 0.0, pos, D, "half", _freq(D, 1e4, "none", 1.0)))
    sjk.check(L.sjk_layer_store(C.byref(layer[0]), 0, n, gu.ptr(rows[0]), gu.ptr(rows[1]), 1, None))
    other = rows[0].clone(), v.float().contiguous()
    sjk.check(L.sjk_layer_store(C.byref(layer[1]), 0, n, gu.ptr(other[0]), gu.ptr(other[1]), 1, None))
    size = 128 * H * 2 * D * 2
    assert (gu.d2h_ptr(layer[0].sink, size) == gu.d2h_ptr(layer[1].sink, size)).all()
    for x in layer:
        L.sj_kvarn_layer_free(C.byref(x))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("layout", ["half", "pair"])
@pytest.mark.parametrize("n,D,n_rot", [(1, 128, 20), (700, 96, 24), (2500, 64, 22), (700, 256, 130), (600, 512, 510), (700, 16, 6), (650, 48, 2)])
def test_odd_rotations(T, dtype, layout, n, D, n_rot):
    """Rotating parts that are no multiple of 16 channels, in calls of one token and of many, some of them skipped."""
    dt = _dt(T, dtype)
    HQ, H = 5, 2
    q, k, v, pos, w = _inputs(T, n, HQ, H, D, dt, n + n_rot, far=100000)
    pos[3::7] = -1
    live = pos >= 0
    rope = kv16.Rope(n_rot, layout=layout, base=1e4)
    step = kv16.Qkv(D, rope=rope, q_norm=w[0], norm_bias=0.25, eps=EPS)
    q_out, k_out, v_out = T.full_like(q, 7.0), T.full_like(k, 7.0), T.full_like(v, 7.0)
    step(q, k, v, pos, q_out=q_out, k_out=k_out, v_out=v_out)
    steps = _freq(n_rot, 1e4, "none", 1.0)
    some = [t for t in sorted({0, 1, n // 3, n // 2, n - 2, n - 1}) if 0 <= t < n and int(pos[t]) >= 0]
    _close(T, q_out[some], _want(T, q[some], w[0], 0.25, pos[some], n_rot, layout, steps))
    _close(T, k_out[some], _want(T, k[some], None, 0.0, pos[some], n_rot, layout, steps))
    assert T.equal(v_out[live], v[live])
    for x in (q_out, k_out, v_out):
        assert bool((x[~live] == 7.0).all())
    parts = T.full_like(q, 7.0)                 # every token: the same values whatever the batch it came in
    for t in range(0, n, 100):
        step(q=q[t:t + 100], pos=pos[t:t + 100], q_out=parts[t:t + 100])
    assert T.equal(parts, q_out)


@pytest.mark.parametrize("layout", ["half", "pair"])
def test_odd_rotations_leave_the_rest(T, layout):
    """Infinities, NaN and zeros' signs behind the rotating channels stay as they are and reach no rotating one. (A NaN
    stays a NaN; its payload is the conversion's.)"""
    n, D, n_rot = 700, 64, 20
    q, _, _, pos, _ = _inputs(T, n, 4, 1, D, T.bfloat16, 3)
    q[..., n_rot], q[..., n_rot + 1], q[..., n_rot + 3] = math.inf, math.nan, -0.0
    out = T.empty_like(q)
    kv16.Qkv(D, rope=kv16.Rope(n_rot, layout=layout))(q=q, pos=pos, q_out=out)
    rest, want = out[..., n_rot:].contiguous(), q[..., n_rot:].contiguous()
    assert T.equal(rest.isnan(), want.isnan())
    assert T.equal(rest.view(T.int16)[~want.isnan()], want.view(T.int16)[~want.isnan()])
    assert bool(out[..., :n_rot].isfinite().all())
