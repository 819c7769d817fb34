"""The 16-bit layers' calls on the CPU: rotary tables against their definition, and what the calls refuse before they
reach the device."""
import ctypes as C
import math
from fractions import Fraction

import pytest

import kv16
import sjk


@pytest.fixture(scope="module")
def L():
    import build
    build.build()
    return sjk.lib()


def _definition(n, base=1e4, scaling="none", factor=1.0, n_ctx=0, beta_fast=32.0, beta_slow=1.0, low=1.0, high=4.0):
    """Angle per position of every pair, in 64-bit floats."""
    if scaling == "ntk" and n > 2:
        base = base * factor ** (n / (n - 2))
    out = []
    for i in range(n // 2):
        f = base ** (-2 * i / n)
        if scaling == "linear":
            f /= factor
        elif scaling == "yarn":
            lo = max(math.floor(n * math.log(n_ctx / (beta_fast * 2 * math.pi)) / (2 * math.log(base))), 0)
            hi = min(math.ceil(n * math.log(n_ctx / (beta_slow * 2 * math.pi)) / (2 * math.log(base))), n - 1)
            r = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            f = f / factor * r + f * (1 - r)
        elif scaling == "bands":
            s = min(max((n_ctx * f / (2 * math.pi) - low) / (high - low), 0.0), 1.0)
            f = f / factor * (1 - s) + f * s
        out.append(f)
    return out


@pytest.mark.parametrize("n", [2, 20, 64, 128, 256, 512])
@pytest.mark.parametrize("scaling,factor", [("none", 1.0), ("linear", 4.0), ("ntk", 8.0), ("yarn", 8.0), ("bands", 8.0), ("linear", 0.25)])
def test_rope_steps_match_definition(L, n, scaling, factor):
    """The fixed-point turns are within the 64-bit floats' own error of the definition (2^-50 relative), the amplitude
    within a 32-bit rounding."""
    step, amp = kv16.rope_steps(n, base=5e5, scaling=scaling, factor=factor, n_ctx=8192)
    want = _definition(n, base=5e5, scaling=scaling, factor=factor, n_ctx=8192)
    for s, w in zip(step, want):
        turn = (w / (2 * math.pi)) % 1.0
        assert abs(Fraction(s, 2 ** 64) - Fraction(turn)) <= Fraction(1, 2 ** 64) + Fraction(turn) * Fraction(1, 2 ** 44)
    assert amp == pytest.approx(0.1 * math.log(factor) + 1 if scaling == "yarn" else 1.0, rel=2 ** -23)
    assert kv16.rope_steps(n, base=5e5, scaling=scaling, factor=factor, n_ctx=8192, amp=0.5)[1] == 0.5


def test_rope_first_pair_is_one_radian(L):
    step, _ = kv16.rope_steps(64)
    assert abs(Fraction(step[0], 2 ** 64) * Fraction(math.pi) * 2 - 1) < Fraction(1, 2 ** 50)


@pytest.mark.parametrize("bad", [dict(n_rot=0), dict(n_rot=3), dict(n_rot=514), dict(base=1.0), dict(base=math.inf), dict(amp=-1.0),
                                 dict(scaling="linear", factor=0.0), dict(scaling="yarn", factor=2.0, n_ctx=0),
                                 dict(scaling="yarn", factor=2.0, n_ctx=100, beta_fast=0.5), dict(scaling="bands", factor=2.0, n_ctx=100, low=4.0),
                                 dict(scaling="ntk", factor=math.nan)])
def test_rope_refusals(L, bad):
    with pytest.raises(sjk.SjkError) as e:
        kv16.rope_steps(**{**dict(n_rot=64), **bad})
    assert e.value.rc == -100


P = 0x10000                                      # an aligned address that nothing follows: the calls refuse before


def _cache(**kw):
    c = sjk.Kv16(P, P, 16 * 2 * 64, 2 * 64, 64, kv16.BF16, 64, 2, 16, 8, P, 4, 4)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _rows(n_head=2, type=kv16.BF16, p=P, row=1024, head=64):
    return sjk.Rows(p, row, head, n_head, type)


def _qkv(**kw):
    a = sjk.QkvArgs()
    a.n_tok, a.head_dim, a.eps, a.pos = 3, 64, 1e-6, P
    a.q, a.k, a.v = _rows(4), _rows(), _rows()
    a.q_out = _rows(4)
    a.cache = _cache()
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("rc,bad", [
    (-100, dict(n_tok=-1)), (-120, dict(head_dim=63)), (-120, dict(head_dim=514)), (-120, dict(head_dim=0)),
    (-100, dict(q=_rows(0))), (-100, dict(q=_rows(4, type=3))), (-100, dict(q=_rows(4, type=kv16.F32))),
    (-100, dict(q_out=_rows(2))), (-100, dict(q_out=_rows(4, type=-1))), (-100, dict(q_out=_rows(4, row=2048))),
    (-100, dict(k=sjk.Rows())), (-100, dict(v=sjk.Rows())), (-100, dict(k=_rows(4))), (-100, dict(pos=None)),
    (-100, dict(cache=_cache(head_dim=128))), (-100, dict(cache=_cache(type=kv16.F32))), (-100, dict(cache=_cache(page_tokens=0))),
    (-100, dict(cache=_cache(tables=None))), (-100, dict(cache=_cache(v=None))), (-100, dict(cache=_cache(n_rows=2))),
    (-100, dict(cache=_cache(n_pages=0xFFFFFFFF))), (-100, dict(cache=_cache(slot_stride=-8))),
    (-100, dict(q_norm=P, norm_type=7)), (-100, dict(q_norm=P, eps=-1.0)), (-100, dict(k_norm=P, eps=math.nan)),
    (-129, dict(rope=sjk.RopeC(66, 0, 1.0, P))), (-129, dict(rope=sjk.RopeC(3, 0, 1.0, P))), (-129, dict(rope=sjk.RopeC(64, 2, 1.0, P))),
    (-129, dict(rope=sjk.RopeC(64, 0, 1.0, None))),
])
def test_qkv_refusals(L, rc, bad):
    assert L.sjk_qkv(C.byref(_qkv(**bad)), None) == rc


def test_calls_without_work_return_ok(L):
    assert L.sjk_qkv(C.byref(_qkv(n_tok=0)), None) == 0
    a = _qkv(q_out=sjk.Rows(), k=sjk.Rows(), v=sjk.Rows(), cache=sjk.Kv16())
    assert L.sjk_qkv(C.byref(a), None) == 0      # nobody wants the query heads
    assert L.sjk_qkv(None, None) == -100


def _attend(L, c=None, q=None, out=None, len=P, rows=None, n=2, scale=1.0, window=0, scratch=P, size=1 << 30):
    c = c or _cache()
    return L.sjk_kv16_attend(C.byref(c), C.byref(q or _rows(4)), len, rows, n, scale, window, C.byref(out or _rows(4)), scratch, size, None)


@pytest.mark.parametrize("rc,bad", [
    (-100, dict(n=-1)), (-100, dict(window=-1)), (-100, dict(scale=math.inf)), (-100, dict(scale=math.nan)), (-100, dict(len=None)),
    (-100, dict(q=_rows(3))), (-100, dict(q=_rows(2), out=_rows(4))), (-100, dict(q=_rows(4, p=None))), (-100, dict(out=_rows(4, type=9))),
    (-100, dict(n=5)), (-100, dict(c=_cache(k=P + 8))), (-100, dict(c=_cache(head_stride=60))), (-100, dict(c=_cache(tables=None))),
    (-100, dict(q=_rows(4, p=P + 2))), (-100, dict(q=_rows(4, row=1025))), (-201, dict(c=_cache(head_dim=72))), (-201, dict(c=_cache(head_dim=512))),
    (-102, dict(scratch=None)), (-102, dict(scratch=P + 8)), (-102, dict(size=1024)),
])
def test_attend_refusals(L, rc, bad):
    assert _attend(L, **bad) == rc


def test_attend_scratch_bytes(L):
    c = _cache()
    one = L.sjk_kv16_attend_scratch_bytes(C.byref(c), 4)
    assert 0 < one < 64 << 20 and L.sjk_kv16_attend_scratch_bytes(C.byref(c), 32) >= one
    assert L.sjk_kv16_attend_scratch_bytes(C.byref(c), 3) == 0 and L.sjk_kv16_attend_scratch_bytes(C.byref(c), 0) == 0
    assert _attend(L, n=0) == 0


def _pages(**kw):
    p = sjk.PagesC(P, P, 64, 4, 8, 16)
    p.n_slabs = 1
    p.slabs[0] = sjk.Slab(P, 4096, 4096 * 64, 2)
    for k, v in kw.items():
        if k == "slab":
            p.slabs[0] = v
        else:
            setattr(p, k, v)
    return p


@pytest.mark.parametrize("bad", [dict(ledger=None), dict(ledger=P + 4), dict(n_pages=0), dict(n_pages=(1 << 20) + 1), dict(tables=None),
                                 dict(n_rows=0), dict(table_stride=0), dict(page_tokens=0), dict(n_slabs=5), dict(n_slabs=-1),
                                 dict(slab=sjk.Slab(None, 4096, 4096 * 64, 2)), dict(slab=sjk.Slab(P + 8, 4096, 4096 * 64, 2)),
                                 dict(slab=sjk.Slab(P, 4100, 4096 * 64, 2)), dict(slab=sjk.Slab(P, 4096, 8, 2)), dict(slab=sjk.Slab(P, 4096, 4096 * 64, 0))])
def test_pages_refusals(L, bad):
    p = C.byref(_pages(**bad))
    assert L.sjk_pages_fork(p, P, P, 1, P, None) == -100
    assert L.sjk_pages_extend(p, P, P, None, 1, 1, P, None) == -100
    assert L.sjk_pages_free(p, P, None, None, 1, None) == -100
    assert L.sjk_pages_compact(p, None, None) == -100


def test_pages_argument_refusals(L):
    p = C.byref(_pages())
    assert L.sjk_pages_fork(p, P, P, -1, P, None) == -100 and L.sjk_pages_fork(p, P, P, 1, None, None) == -100
    assert L.sjk_pages_extend(p, P, P, None, 1, 1025, P, None) == -100 and L.sjk_pages_extend(p, P, P, None, -1, 1, P, None) == -100
    assert L.sjk_pages_extend(p, P, P, None, 1, 1, None, None) == -100
    assert L.sjk_pages_free(p, None, None, None, 1, None) == -100 and L.sjk_pages_copy(p, P, None, 1, None) == -100
    for rc in (L.sjk_pages_fork(p, None, None, 0, None, None), L.sjk_pages_extend(p, None, None, None, 1, 0, None, None),
               L.sjk_pages_free(p, None, None, None, 0, None), L.sjk_pages_copy(p, None, None, 0, None)):
        assert rc == 0
    assert L.sjk_pages_bytes(64) >= 16 + 64 * 8
