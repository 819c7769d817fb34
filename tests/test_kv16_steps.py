"""The calls for several new tokens a sequence and for chosen pages on the CPU: what they refuse before they reach the device,
and what kv16 checks and passes on around them."""
import ctypes as C
import math

import pytest
import torch

import kv16
import sjk
from test_kv16 import P, _cache, _qkv, _rows
from test_kv16_host import Gpu, Host, _heads, _i32, host  # noqa: F401
from test_kv16_host import _cache as _host_cache


@pytest.fixture(scope="module")
def L():
    import build
    build.build()
    return sjk.lib()


def test_qkv_at_refusals(L):
    assert L.sjk_qkv_at(C.byref(_qkv(n_tok=0)), P, None) == 0
    assert L.sjk_qkv_at(C.byref(_qkv(n_tok=0)), None, None) == 0
    assert L.sjk_qkv_at(C.byref(_qkv(n_tok=0)), P + 2, None) == -100
    assert L.sjk_qkv_at(None, P, None) == -100
    assert L.sjk_qkv_at(C.byref(_qkv(pos=None)), P, None) == -100


def _maps(L, c=None, len=P, add=P, rows=None, masks=None, n=2, n_tok=8, **out):
    step = sjk.Kv16Step(P, P, P, P, P)
    for k, v in out.items():
        setattr(step, k, v)
    return L.sjk_kv16_maps(C.byref(c or _cache()), len, add, rows, masks, n, n_tok, C.byref(step), None)


@pytest.mark.parametrize("bad", [dict(n=-1), dict(n=8193), dict(n_tok=-1), dict(len=None), dict(add=None), dict(len=P + 2), dict(add=P + 1),
                                 dict(rows=P + 2), dict(masks=P + 4), dict(first=P + 1), dict(row=P + 2), dict(pos=P + 3), dict(at=P + 2),
                                 dict(slot=P + 4), dict(n=5), dict(c=_cache(tables=None)), dict(c=_cache(page_tokens=0))])
def test_maps_refusals(L, bad):
    assert _maps(L, **bad) == -100
    assert L.sjk_kv16_maps(None, P, P, None, None, 1, 1, C.byref(sjk.Kv16Step()), None) == -100
    assert L.sjk_kv16_maps(C.byref(_cache()), P, P, None, None, 1, 1, None, None) == -100


def _tree(L, c=None, q=None, out=None, n_tok=8, first=P, len=P, rows=None, masks=P, n=2, nodes=4, scale=1.0, window=0, scratch=P, size=1 << 30):
    return L.sjk_kv16_attend_tree(C.byref(c or _cache()), C.byref(q or _rows(4)), n_tok, first, len, rows, masks, n, nodes, scale, window,
                                  C.byref(out or _rows(4)), scratch, size, None)


@pytest.mark.parametrize("rc,bad", [
    (-100, dict(n=-1)), (-100, dict(n_tok=-1)), (-100, dict(nodes=-1)), (-100, dict(window=-1)), (-100, dict(scale=math.inf)),
    (-100, dict(scale=math.nan)), (-100, dict(len=None)), (-100, dict(len=P + 2)), (-100, dict(first=P + 1)), (-100, dict(rows=P + 2)),
    (-100, dict(masks=P + 4)), (-100, dict(q=_rows(3), out=_rows(3))), (-100, dict(q=_rows(2), out=_rows(4))), (-100, dict(q=_rows(4, p=None))),
    (-100, dict(out=_rows(4, p=None))), (-100, dict(q=_rows(4, type=kv16.F32))), (-100, dict(out=_rows(4, type=kv16.F32))),
    (-100, dict(q=_rows(4, type=kv16.F16))), (-100, dict(q=_rows(4, p=P + 8))), (-100, dict(q=_rows(4, row=1025))), (-100, dict(q=_rows(4, head=66))),
    (-100, dict(out=_rows(4, p=P + 1))), (-100, dict(c=_cache(k=P + 8))), (-100, dict(c=_cache(head_stride=60))), (-100, dict(c=_cache(tables=None))),
    (-100, dict(n=5)), (-100, dict(first=None, n_tok=9)), (-201, dict(c=_cache(head_dim=72))), (-201, dict(nodes=65)),
    (-201, dict(q=_rows(4096), out=_rows(4096), nodes=64)), (-102, dict(scratch=None)), (-102, dict(scratch=P + 8)), (-102, dict(size=1024)),
])
def test_tree_refusals(L, rc, bad):
    assert _tree(L, **bad) == rc


def test_tree_without_work(L):
    assert _tree(L, n=0, n_tok=0, len=None, q=_rows(4, p=None), out=_rows(4, p=None), scratch=None) == 0
    assert _tree(L, n_tok=0, nodes=0, first=None, q=_rows(4, p=None), out=_rows(4, p=None), scratch=None) == 0
    assert 0 < L.sjk_kv16_attend_tree_scratch_bytes(C.byref(_cache())) < 64 << 20
    assert L.sjk_kv16_attend_tree_scratch_bytes(C.byref(_cache(head_dim=80))) == 0 and L.sjk_kv16_attend_tree_scratch_bytes(None) == 0


def _keep(L, c=None, layers=1, stride=0, len=P, path=P, count=P, rows=None, width=4, n=2, new=2 * P):
    return L.sjk_kv16_keep(C.byref(c or _cache()), layers, stride, len, path, count, rows, width, n, new, None)


@pytest.mark.parametrize("bad", [dict(layers=0), dict(layers=65536), dict(stride=-8), dict(len=None), dict(path=None), dict(count=None), dict(width=0),
                                 dict(width=257), dict(n=-1), dict(n=5), dict(len=P + 1), dict(path=P + 2), dict(count=P + 2), dict(rows=P + 1),
                                 dict(new=P + 2), dict(new=P), dict(new=P + 4), dict(new=P - 4), dict(c=_cache(v=None))])
def test_keep_refusals(L, bad):
    assert _keep(L, **bad) == -100
    assert _keep(L, n=0, len=None, path=None, count=None, new=None) == 0


def _bounds(L, c=None, layers=1, stride=0, bounds=P, bstride=0, first=P, end=P, rows=None, n=2):
    return L.sjk_kv16_bounds(C.byref(c or _cache()), layers, stride, bounds, bstride, first, end, rows, n, None)


@pytest.mark.parametrize("rc,bad", [(-100, dict(layers=0)), (-100, dict(stride=-1)), (-100, dict(bounds=None)), (-100, dict(bounds=P + 8)),
                                    (-100, dict(bstride=-8)), (-100, dict(layers=2, stride=8, bstride=8)), (-100, dict(layers=2, stride=4, bstride=1 << 30)),
                                    (-100, dict(first=None)), (-100, dict(end=None)), (-100, dict(first=P + 1)), (-100, dict(end=P + 2)),
                                    (-100, dict(rows=P + 2)), (-100, dict(n=-1)), (-100, dict(n=5)), (-100, dict(c=_cache(k=P + 8))),
                                    (-100, dict(c=_cache(slot_stride=130))), (-201, dict(c=_cache(head_dim=72)))])
def test_bounds_refusals(L, rc, bad):
    assert _bounds(L, **bad) == rc
    assert _bounds(L, n=0, first=None, end=None) == 0


def _select(L, c=None, bounds=P, q=None, len=P, rows=None, n=2, budget=4, sink=1, recent=1, blocks=P, count=P, scratch=P, size=1 << 30):
    return L.sjk_kv16_select(C.byref(c or _cache()), bounds, C.byref(q or _rows(4)), len, rows, n, budget, sink, recent, blocks, count, scratch, size, None)


@pytest.mark.parametrize("rc,bad", [
    (-100, dict(bounds=None)), (-100, dict(bounds=P + 8)), (-100, dict(q=_rows(3))), (-100, dict(q=_rows(4, type=5))), (-100, dict(q=_rows(4, p=P + 1))),
    (-100, dict(q=_rows(4, p=None))), (-100, dict(len=None)), (-100, dict(len=P + 2)), (-100, dict(rows=P + 1)), (-100, dict(n=-1)), (-100, dict(n=5)),
    (-100, dict(budget=0)), (-100, dict(sink=-1)), (-100, dict(recent=-1)), (-100, dict(sink=3, recent=2)), (-100, dict(sink=2 ** 31 - 1, recent=2 ** 31 - 1)),
    (-100, dict(blocks=None)), (-100, dict(blocks=P + 2)), (-100, dict(count=P + 1)), (-201, dict(c=_cache(head_dim=80))), (-102, dict(scratch=None)),
    (-102, dict(scratch=P + 4)), (-102, dict(size=16)),
])
def test_select_refusals(L, rc, bad):
    assert _select(L, **bad) == rc
    assert _select(L, n=0, len=None, blocks=None, count=None, scratch=None, q=_rows(4, p=None)) == 0


def _attend(L, c=None, q=None, out=None, len=P, rows=None, blocks=P, n=2, budget=4, scale=1.0, scratch=P, size=1 << 30):
    return L.sjk_kv16_attend_blocks(C.byref(c or _cache()), C.byref(q or _rows(4)), len, rows, blocks, n, budget, scale, C.byref(out or _rows(4)), scratch,
                                    size, None)


@pytest.mark.parametrize("rc,bad", [
    (-100, dict(n=-1)), (-100, dict(budget=0)), (-100, dict(scale=math.nan)), (-100, dict(len=None)), (-100, dict(blocks=None)), (-100, dict(len=P + 1)),
    (-100, dict(blocks=P + 2)), (-100, dict(rows=P + 2)), (-100, dict(q=_rows(3), out=_rows(3))), (-100, dict(q=_rows(2))), (-100, dict(q=_rows(4, p=None))),
    (-100, dict(out=_rows(4, type=9))), (-100, dict(n=5)), (-100, dict(c=_cache(k=P + 8))), (-100, dict(q=_rows(4, p=P + 2))), (-201, dict(c=_cache(head_dim=72))),
    (-102, dict(scratch=None)), (-102, dict(scratch=P + 8)), (-102, dict(size=1024)),
])
def test_attend_blocks_refusals(L, rc, bad):
    assert _attend(L, **bad) == rc


def test_attend_blocks_without_work(L):
    assert _attend(L, n=0, len=None, blocks=None, scratch=None) == 0
    c = C.byref(_cache())
    a = L.sjk_kv16_attend_blocks_scratch_bytes(c, 4, 2, 4)
    assert 0 < a < L.sjk_kv16_attend_blocks_scratch_bytes(c, 4, 2, 4000) and L.sjk_kv16_attend_blocks_scratch_bytes(c, 3, 2, 4) == 0
    assert L.sjk_kv16_attend_blocks_scratch_bytes(c, 4, 2, 0) == 0 and L.sjk_kv16_select_scratch_bytes(c, -1) == 0
    # sizes that 32 bits do not hold
    big = _cache(n_rows=1 << 20, table_stride=1 << 20, n_head_kv=8)
    assert L.sjk_kv16_select_scratch_bytes(C.byref(big), 1 << 12) > 1 << 38


# ---- from Python ------------------------------------------------------------------------------------------------------

class Steps(Host):
    """Notes the new calls as well."""

    def __getattr__(self, name):
        if name.startswith("sjk_kv16_") and not name.endswith("_bytes"):
            return lambda *a: self._note(name[9:], stream=a[-1], args=a)
        if name == "sjk_qkv_at":
            return lambda a, at, st: self._note("qkv_at", stream=st, at=at, pos=a._obj.pos)
        return getattr(self.lib, name)


@pytest.fixture
def steps(host, monkeypatch):  # noqa: F811
    h = Steps(host.lib)
    h.device = 0
    monkeypatch.setattr(kv16, "_L", h)
    monkeypatch.setattr(kv16, "_current_device", lambda: host.device)
    monkeypatch.setattr(kv16, "_capturing", lambda: h.capturing)
    h.outer = host
    return h


def _masks(n, index=0, dtype=torch.int64):
    return Gpu(torch.zeros(n, dtype=dtype), index)


def _wrong_tree(c):
    q, lens = _heads(8, 4), _i32(2)
    yield dict(q=_heads(8, 4, index=1), lens=lens)
    yield dict(q=q, lens=_i32(2, 1))
    yield dict(q=q, lens=lens, masks=_masks(7))
    yield dict(q=q, lens=lens, masks=_masks(8, dtype=torch.int32))
    yield dict(q=q, lens=lens, masks=_masks(8, 1))
    yield dict(q=q, lens=lens, first=_i32(2))
    yield dict(q=q, lens=_i32(3))                            # 8 tokens of 3 sequences, no `first`
    yield dict(q=q, lens=lens, nodes=5)
    yield dict(q=q, lens=lens, rows=_i32(3))
    yield dict(q=q, lens=lens, out=_heads(7, 4))
    yield dict(q=q, lens=lens, scratch=Gpu(torch.zeros(1 << 20, dtype=torch.uint8), 1))


def test_tree_arguments(steps):
    c = _host_cache()
    for bad in _wrong_tree(c):
        bad.setdefault("masks", None)
        bad.setdefault("out", _heads(8, 4))
        with pytest.raises(ValueError):
            c.attend_tree(0, scale=0.1, **bad)
    assert steps.calls == []
    q, lens, m = _heads(8, 4), _i32(2), _masks(8)
    out = _heads(8, 4)
    assert c.attend_tree(0, q, lens, m, 0.5, out=out, window=7) is out
    call = steps.calls[-1]["args"]
    assert call[2] == 8 and call[3] is None and call[6] == m.data_ptr() and call[7:9] == (2, 4) and call[9:11] == (0.5, 7) and call[13] == c.tree_scratch_bytes()
    c.attend_tree(0, q, lens, None, 0.5, first=_i32(3), out=out)
    assert steps.calls[-1]["args"][8] == 64 and steps.calls[-1]["args"][6] is None
    steps.calls.clear()
    c.attend_tree(0, _heads(0, 4), _i32(0), None, 0.5, out=_heads(0, 4))
    c.attend_tree(0, _heads(0, 4), lens, None, 0.5, first=_i32(3), out=_heads(0, 4))
    assert steps.calls == []


def test_keep_and_maps_arguments(steps):
    c = _host_cache()
    path = Gpu(torch.zeros((2, 3), dtype=torch.int32))
    for kw in (dict(lens=_i32(2), path=_i32(6), count=_i32(2)), dict(lens=_i32(2), path=path, count=_i32(3)), dict(lens=_i32(3), path=path, count=_i32(3)),
               dict(lens=_i32(2), path=path, count=_i32(2), rows=_i32(1)), dict(lens=_i32(2), path=path, count=_i32(2), new_lens=_i32(3)),
               dict(lens=_i32(2), path=Gpu(torch.zeros((3, 2), dtype=torch.int32).T), count=_i32(2)), dict(lens=_i32(2, 1), path=path, count=_i32(2))):
        kw.setdefault("new_lens", _i32(2))
        with pytest.raises(ValueError):
            c.keep(**kw)
    new = _i32(2)
    assert c.keep(_i32(2), path, _i32(2), new_lens=new) is new and steps.calls[-1]["args"][7:10] == (3, 2, new.data_ptr())
    steps.calls.clear()
    m = kv16.Maps(c, 2, 9)
    for kw in (dict(lens=_i32(3), add=_i32(2)), dict(lens=_i32(2), add=_i32(1)), dict(lens=_i32(2), add=_i32(2), rows=_i32(3)),
               dict(lens=_i32(2), add=_i32(2), masks=_masks(8)), dict(lens=_i32(2, 1), add=_i32(2))):
        with pytest.raises(ValueError):
            m(**kw)
    assert steps.calls == []
    assert m(_i32(2), _i32(2), masks=_masks(9)) is m and steps.calls[-1]["args"][5:7] == (2, 9)
    assert (m.first.numel(), m.rows.numel(), m.pos.numel(), m.at.numel(), m.slots.numel()) == (3, 9, 9, 9, 9)


def test_blocks_arguments(steps):
    c = _host_cache()
    good = torch.zeros((1, 8, 2, 2, 64), dtype=torch.bfloat16)
    for bad in (good.half(), good[:, :7], good.transpose(2, 3)):
        with pytest.raises(ValueError, match="bounds"):
            kv16.Blocks(c, bounds=Gpu(bad))
    with pytest.raises(ValueError, match="bounds"):
        kv16.Blocks(c, bounds=Gpu(good, 1))

    class Bounds(Gpu):                           # (iterated over by layer)
        def __iter__(self):
            return iter(self.t)

    b = kv16.Blocks(c, bounds=Bounds(good))
    q, lens = _heads(2, 4), _i32(2)
    room = lambda *s: Gpu(torch.zeros(s, dtype=torch.int32))  # noqa: E731
    for kw in (dict(budget=0), dict(budget=3, sink=2, recent=2), dict(budget=3, sink=-1), dict(budget=3, blocks=room(2, 2, 4)), dict(budget=3, count=room(2)),
               dict(budget=3, lens=_i32(3)), dict(budget=3, q=_heads(2, 4, index=1)), dict(budget=3, rows=_i32(3))):
        with pytest.raises(ValueError):
            b.select(0, **{"q": q, "lens": lens, "blocks": None if "blocks" not in kw else kw["blocks"],
                           **{"blocks": room(2, 2, max(kw.get("budget", 3), 1)), "count": room(2, 2)}, **kw})
    for kw in (dict(blocks=room(2, 4)), dict(blocks=room(2, 3, 4)), dict(lens=_i32(1)), dict(out=_heads(3, 4)), dict(rows=_i32(1))):
        with pytest.raises(ValueError):
            b.attend(0, **{"q": q, "lens": lens, "blocks": room(2, 2, 4), "scale": 0.1, "out": _heads(2, 4), **kw})
    with pytest.raises(ValueError):
        b.update(_i32(2), _i32(3))
    assert steps.calls == []
    lists, count = b.select(0, q, lens, 5, blocks=room(2, 2, 5), count=room(2, 2))
    out = _heads(2, 4)
    assert b.attend(0, q, lens, lists, 0.1, out=out) is out
    b.update(_i32(2), _i32(2))
    assert [x["name"] for x in steps.calls] == ["select", "attend_blocks", "bounds"]
    assert steps.calls[0]["args"][1] == good.data_ptr() and steps.calls[0]["args"][5:9] == (2, 5, 1, 1)


def test_scratch_by_stream_and_capture(steps, monkeypatch):
    """Calls of a stream share memory that grows, calls of another one and captured calls do not use it."""
    c = _host_cache()
    q, lens, out = _heads(8, 4), _i32(2), _heads(8, 4)
    where = lambda: (c.attend_tree(0, q, lens, None, 0.1, out=out), steps.calls[-1]["args"][12])[1]  # noqa: E731
    a = where()
    assert where() == a
    monkeypatch.setattr(kv16, "_stream", lambda d: 2000 + d)
    b = where()
    assert b != a and where() == b
    steps.capturing = True
    x = torch.empty(8, dtype=torch.uint8)
    assert where() not in (a, b) and x is not None
    steps.capturing = False
    assert where() == b
    s = kv16._Scratch(0)
    assert s.get(1, 100)[1] == s.get(1, 50)[1] and s.get(1, 200)[2] == 200 and s.get(1, 100)[2] == 200


def test_qkv_passes_cache_positions(steps):
    c = _host_cache()
    step = kv16.Qkv(64, cache=c)
    k, pos, at = _heads(3, 2), _i32(3), _i32(3)
    with pytest.raises(ValueError):
        step(k=k, v=k, pos=pos, at=_i32(2))
    step(k=k, v=k, pos=pos, at=at)
    assert steps.calls[-1]["name"] == "qkv_at" and steps.calls[-1]["at"] == at.data_ptr() and steps.calls[-1]["pos"] == pos.data_ptr()


@pytest.mark.parametrize("there,current", [(0, 1), (1, 0), (1, 1)])
def test_calls_run_on_their_tensors_device(steps, there, current):
    steps.outer.device = current
    seen = []
    steps._note = lambda name, **kw: seen.append((name, steps.outer.device, kw["stream"])) or 0
    c = _host_cache(there)
    lens, out = _i32(2, there), _heads(8, 4, index=there)
    c.attend_tree(0, _heads(8, 4, index=there), lens, None, 0.1, out=out)
    c.keep(lens, Gpu(torch.zeros((2, 3), dtype=torch.int32), there), _i32(2, there), new_lens=_i32(2, there))

    class Bounds(Gpu):
        def __iter__(self):
            return iter(self.t)

    b = kv16.Blocks(c, bounds=Bounds(torch.zeros((1, 8, 2, 2, 64), dtype=torch.bfloat16), there))
    lists = Gpu(torch.zeros((2, 2, 5), dtype=torch.int32), there)
    b.select(0, _heads(2, 4, index=there), lens, 5, blocks=lists, count=Gpu(torch.zeros((2, 2), dtype=torch.int32), there))
    b.attend(0, _heads(2, 4, index=there), lens, lists, 0.1, out=_heads(2, 4, index=there))
    b.update(lens, lens)
    kv16.Maps(c, 2, 4)(lens, lens)
    assert [x[0] for x in seen] == ["attend_tree", "keep", "select", "attend_blocks", "bounds", "maps"]
    assert all(x[1:] == (there, 1000 + there) for x in seen) and steps.outer.device == current
