"""Outputs that lie over inputs which other parts of the same launch still read are refused, before anything reaches the device."""
import ctypes as C

import pytest

import sjk
from test_kv16 import P, _cache, _rows


@pytest.fixture(scope="module")
def L():
    import build
    build.build()
    return sjk.lib()


LEN, PATH, COUNT, ROWS, NEW = (P + i * 4096 for i in range(5))


def _keep(L, new, n=2, width=4, rows=ROWS):
    return L.sjk_kv16_keep(C.byref(_cache()), 1, 0, LEN, PATH, COUNT, rows, width, n, new, None)


@pytest.mark.parametrize("new", [LEN, LEN + 4, LEN - 4, COUNT, COUNT + 4, COUNT - 4, PATH, PATH + 28, PATH - 4, ROWS, ROWS + 4, ROWS - 4])
def test_keep_refuses_new_lengths_over_its_inputs(L, new):
    assert _keep(L, new) == -100
    assert _keep(L, new, n=0) == 0


def _maps(L, n=2, n_tok=8, masks=P + 0x5000, rows=ROWS, c=None, **out):
    step = sjk.Kv16Step(*(P + 0x10000 + i * 0x1000 for i in range(5)))
    for k, v in out.items():
        setattr(step, k, v)
    return L.sjk_kv16_maps(C.byref(c or _cache()), LEN, COUNT, rows, masks, n, n_tok, C.byref(step), None)


@pytest.mark.parametrize("what", ["first", "row", "pos", "at", "slot"])
@pytest.mark.parametrize("over", [LEN, COUNT, ROWS, P + 0x5000])
def test_maps_refuse_outputs_over_inputs(L, what, over):
    """(The inputs are 8 bytes, the masks 64; outputs 12, 32 or 64.)"""
    size = {"first": 12, "slot": 64}.get(what, 32)
    last = over + (64 if over == P + 0x5000 else 8)
    for at in (over, last - 8, over - size + 8):
        assert _maps(L, **{what: at}) == -100


@pytest.mark.parametrize("bad", [dict(n=-1), dict(n=8193), dict(n_tok=-1), dict(rows=ROWS + 2), dict(masks=P + 0x5004), dict(first=NEW + 1), dict(row=NEW + 2),
                                 dict(pos=NEW + 3), dict(at=NEW + 2), dict(slot=NEW + 4), dict(n=5, rows=None), dict(c=_cache(tables=None)), dict(c=_cache(page_tokens=0))])
def test_maps_refusals_of_lists_apart(L, bad):
    assert _maps(L, **bad) == -100


@pytest.mark.parametrize("over", [dict(blocks=LEN), dict(blocks=LEN + 4), dict(blocks=LEN - 60), dict(count=LEN), dict(count=LEN + 4), dict(count=LEN - 12)])
def test_select_refuses_lists_over_lengths(L, over):
    """(Lengths 8 bytes, lists 2 x 2 x 4 numbers, counts 2 x 2.)"""
    a = dict(dict(blocks=PATH, count=COUNT), **over)
    assert L.sjk_kv16_select(C.byref(_cache()), P + 0x8000, C.byref(_rows(4)), LEN, ROWS, 2, 4, 1, 1, a["blocks"], a["count"], P + 0x20000, 1 << 30, None) == -100
