"""What kv16 does on the host around a call: tensors and devices it refuses, the device it launches on, threads that share
an object, scratch memory. On the CPU: tensors that say they are a GPU's, and a library that notes the calls."""
import ctypes as C
import math
import threading
import time
import types
from collections import Counter

import pytest
import torch

import kv16
import sjk


class Gpu:
    """A CPU tensor that says it is GPU `index`'s."""
    is_cuda = True

    def __init__(self, t, index=0):
        self.t, self.index = t, index

    device = property(lambda self: types.SimpleNamespace(index=self.index))

    def get_device(self):
        return self.index

    def __getitem__(self, i):
        return Gpu(self.t[i], self.index)

    def __getattr__(self, name):
        return getattr(self.t, name)


class Host:
    """Stands for the library and for the current device."""

    def __init__(self, lib):
        self.lib, self.device, self.calls, self.capturing, self.during = lib, 0, [], False, lambda: None

    def __getattr__(self, name):
        return getattr(self.lib, name)

    def _note(self, name, **kw):
        self.calls.append(dict(name=name, device=self.device, **kw))
        return 0

    def sjk_pages_init(self, p, st):
        return self._note("init", stream=st)

    def sjk_pages_fork(self, p, src, dst, n, status, st):
        return self._note("fork", stream=st)

    def sjk_pages_extend(self, p, rows, lens, add, add_all, n, status, st):
        return self._note("extend", stream=st)

    def sjk_pages_free(self, p, rows, g0, g1, n, st):
        return self._note("free", stream=st)

    def sjk_pages_compact(self, p, info, st):
        return self._note("compact", stream=st)

    def sjk_pages_copy(self, p, src, dst, n, st):
        return self._note("copy", stream=st)

    def sjk_rope_init(self, r, cfg):
        r._obj.n_rot, r._obj.amp, r._obj.step = cfg._obj.n_rot, 1.0, 0x10000
        return self._note("rope")

    def sjk_rope_free(self, r):
        pass

    def sjk_kv16_attend(self, c, q, lens, rows, n, scale, window, out, scratch, size, st):
        self.during()
        return self._note("attend", stream=st, scratch=scratch, size=size, q=(q._obj.p, q._obj.row_stride, q._obj.n_head), out=out._obj.p,
                          lens=lens, n=n)

    def sjk_qkv(self, a, st):
        self.during()
        a = a._obj
        return self._note("qkv", stream=st, q=(a.q.p, a.q.row_stride, a.q.n_head), q_out=a.q_out.p, n=a.n_tok, pos=a.pos, rows=a.rows)


@pytest.fixture
def host(monkeypatch):
    import build
    build.build()
    h = Host(sjk.lib())

    class device:                                # torch.cuda.device
        def __init__(self, i):
            self.i = i

        def __enter__(self):
            self.before, h.device = h.device, self.i

        def __exit__(self, *a):
            h.device = self.before

    def on_host(make):
        return lambda *a, device=None, **kw: make(*a, **kw)

    monkeypatch.setattr(kv16, "_L", h)
    monkeypatch.setattr(kv16, "_stream", lambda d: 1000 + d)
    monkeypatch.setattr(kv16, "_current_device", lambda: h.device, raising=False)
    monkeypatch.setattr(kv16, "_capturing", lambda: h.capturing, raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: h.device)
    for name in ("empty", "zeros"):
        monkeypatch.setattr(torch, name, on_host(getattr(torch, name)))
    return h


def _i32(n, index=0):
    return Gpu(torch.zeros(n, dtype=torch.int32), index)


def _heads(n, heads, D=64, dtype=torch.bfloat16, index=0):
    return Gpu(torch.zeros((n, heads, D), dtype=dtype), index)


def _cache(index=0, tables=None):
    kv = [Gpu(torch.zeros((1, 8, 16, 2, 64), dtype=torch.bfloat16), index) for _ in range(2)]
    return kv16.Cache(*kv, Gpu(torch.full((4, 4), -1, dtype=torch.int32), index if tables is None else tables))


def test_slabs_in_host_memory_are_refused(host):
    tables = Gpu(torch.full((4, 4), -1, dtype=torch.int32))
    on, off = Gpu(torch.zeros((1, 8, 64))), torch.zeros((1, 8, 64))
    kv16.Pages(tables, 16, slabs=[on])
    for slabs in ([off], [on, off]):
        with pytest.raises(ValueError, match="slabs"):
            kv16.Pages(tables, 16, slabs=slabs)


@pytest.mark.parametrize("there", [0, 1])
@pytest.mark.parametrize("current", [0, 1])
def test_calls_run_on_their_tensors_device(host, there, current):
    """Whatever device is current, a call launches on its tensors' device, on that device's stream, and leaves the current
    device as it was."""
    host.device = there
    rope = kv16.Rope(64)
    host.device = current
    cache = _cache(there)
    pages = cache.pages()
    q, n = _heads(3, 4, index=there), _i32(3, there)
    cache.attend(0, q, n, 1.0, out=_heads(3, 4, index=there))
    step = kv16.Qkv(64, rope=rope, cache=cache)
    step(k=_heads(3, 2, index=there), v=_heads(3, 2, index=there), pos=n)
    kv16.Qkv(64)(q=q, q_out=q)
    pages.fork(n, n)
    pages.extend(n, n, 1)
    pages.free(n)
    pages.compact()
    pages.copy(n, n)
    assert [c["name"] for c in host.calls] == ["rope", "init", "attend", "qkv", "qkv", "fork", "extend", "free", "compact", "copy"]
    assert all(c["device"] == there for c in host.calls) and all(c["stream"] == 1000 + there for c in host.calls[1:])
    assert host.device == current


def test_rope_on_a_named_device(host):
    assert kv16.Rope(64, device=1).device == 1 and kv16.Rope(64, device="cuda:1").device == 1 and kv16.Rope(64).device == 0
    assert [c["device"] for c in host.calls] == [1, 1, 0] and host.device == 0


def test_tensors_of_another_device_are_refused(host):
    cache, q, n = _cache(0), _heads(3, 4), _i32(3)
    pages = cache.pages()
    far_q, far_n, host_q, host_n = _heads(3, 4, index=1), _i32(3, 1), q.t, n.t
    host.calls.clear()

    def refused(call, *a, **kw):
        with pytest.raises(ValueError):
            call(*a, **kw)
        assert host.calls == []

    for fq, fn in ((far_q, far_n), (host_q, host_n)):
        refused(cache.attend, 0, fq, n, 1.0, out=q)
        refused(cache.attend, 0, q, fn, 1.0, out=q)
        refused(cache.attend, 0, q, n, 1.0, out=fq)
        refused(cache.attend, 0, q, n, 1.0, out=q, rows=fn)
        step = kv16.Qkv(64, cache=cache)
        kv = _heads(3, 2)
        refused(step, fq, kv, kv, n, q_out=q)
        refused(step, q, kv, kv, n, q_out=fq)
        refused(step, q, kv, kv, fn, q_out=q)
        refused(step, q, kv, kv, n, q_out=q, rows=fn)
        refused(kv16.Qkv(64), q=q, q_out=fq)
        refused(kv16.Qkv(64), q=host_q, q_out=host_q)
        refused(pages.fork, fn, n)
        refused(pages.fork, n, fn)
        refused(pages.extend, n, fn, 1)
        refused(pages.free, n, first=fn)
        refused(pages.copy, fn, fn)
    refused(kv16.Cache, cache.k, Gpu(cache.v.t, 1), cache.tables)
    refused(_cache, 0, tables=1)
    refused(kv16.Pages, Gpu(cache.tables.t, 1), 16, slabs=[cache.k])
    # what a Qkv is made of
    rope = kv16.Rope(64, device=1)
    host.calls.clear()
    w = Gpu(torch.ones(64), 1)
    refused(kv16.Qkv, 64, rope=rope, cache=cache)
    refused(kv16.Qkv, 64, q_norm=w, cache=cache)
    refused(kv16.Qkv, 64, q_norm=w, k_norm=Gpu(torch.ones(64), 0))
    refused(kv16.Qkv(64, rope=rope), q=q, q_out=q, pos=n)
    refused(kv16.Qkv(64, q_norm=w), q=q, q_out=q)


def _from_threads(*calls):
    """Each call in its own thread, all started together; what they raised."""
    gate, errors = threading.Barrier(len(calls)), []

    def one(call):
        gate.wait()
        try:
            call()
        except Exception as e:                   # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=one, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
        assert not t.is_alive()
    assert errors == []


def test_threads_on_one_cache(host):
    """Threads that share a cache: every launch has the pointers, strides and heads of one call."""
    cache = _cache()
    kinds = [(3, 4), (2, 8), (4, 6), (1, 2)]
    args = [(_heads(n, h), _heads(n, h), _i32(n)) for n, h in kinds]
    host.during = lambda: time.sleep(0.002)      # the library runs outside the interpreter's lock
    for q, out, n in args:                       # scratch is there before
        cache.attend(0, q, n, 1.0, out=out)
    host.calls.clear()

    def calls(q, out, n):
        def run():
            for _ in range(20):
                cache.attend(0, q, n, 1.0, out=out)
        return run

    _from_threads(*(calls(*a) for a in args))
    want = {(q.data_ptr(), q.stride(0), q.shape[1]): (out.data_ptr(), n.data_ptr(), n.shape[0]) for q, out, n in args}
    assert Counter(c["q"] for c in host.calls) == {k: 20 for k in want}
    for c in host.calls:
        assert want[c["q"]] == (c["out"], c["lens"], c["n"])


def test_threads_on_one_qkv(host):
    step = kv16.Qkv(64)
    kinds = [(3, 4), (2, 8), (4, 6), (1, 2)]
    args = [(_heads(n, h), _heads(n, h), _i32(n)) for n, h in kinds]
    host.during = lambda: time.sleep(0.002)

    def calls(q, out, pos):
        def run():
            for _ in range(20):
                step(q=q, q_out=out, pos=pos)
        return run

    _from_threads(*(calls(*a) for a in args))
    want = {(q.data_ptr(), q.stride(0), q.shape[1]): (out.data_ptr(), pos.data_ptr(), q.shape[0]) for q, out, pos in args}
    assert Counter(c["q"] for c in host.calls) == {k: 20 for k in want}
    for c in host.calls:
        assert want[c["q"]] == (c["q_out"], c["pos"], c["n"])


def test_scratch_of_captured_calls(host):
    """Calls that are captured get scratch of their own, which the graph's memory pool holds; two graphs captured on one
    stream and calls that run there do not share it. Calls that run keep theirs by stream and heads."""
    cache, q, n = _cache(), _heads(3, 4), _i32(3)
    made, keep = [], torch.empty

    def call():
        host.calls.clear()
        cache.attend(0, q, n, 1.0, out=q)
        return host.calls[0]["scratch"], host.calls[0]["size"]

    first = call()
    assert call() == first and first[1] >= sjk.lib().sjk_kv16_attend_scratch_bytes(C.byref(cache.layers[0]), 4)
    with pytest.MonkeyPatch.context() as m:
        m.setattr(torch, "empty", lambda *a, **kw: made.append(keep(*a, **kw)) or made[-1])
        host.capturing = True
        one = call()                             # (this test holds what was allocated)
        two = call()
        host.capturing = False
    assert len(made) == 2 and [one[0], two[0]] == [x.data_ptr() for x in made]
    assert len({first[0], one[0], two[0]}) == 3 and one[1] == two[1] == first[1] and call() == first
    # a graph captured before any call has run leaves nothing behind for those that run
    other = _cache()
    host.capturing = True
    other.attend(0, q, n, 1.0, out=q)
    assert other._scratch == {}


def test_scratch_of_the_callers(host):
    cache, q, n = _cache(), _heads(3, 4), _i32(3)
    size = cache.scratch_bytes(4)
    assert size == sjk.lib().sjk_kv16_attend_scratch_bytes(C.byref(cache.layers[0]), 4)
    mine = Gpu(torch.empty(size, dtype=torch.uint8))
    for host.capturing in (False, True):
        host.calls.clear()
        cache.attend(0, q, n, 1.0, out=q, scratch=mine)
        assert (host.calls[0]["scratch"], host.calls[0]["size"]) == (mine.data_ptr(), size) and cache._scratch == {}
    host.calls.clear()
    for bad in (mine.t, Gpu(mine.t, 1), Gpu(torch.empty(size, dtype=torch.int32)), Gpu(torch.empty((2, size), dtype=torch.uint8)[:, ::2])):
        with pytest.raises(ValueError, match="scratch"):
            cache.attend(0, q, n, 1.0, out=q, scratch=bad)
    with pytest.raises(ValueError):
        cache.scratch_bytes(3)
    assert host.calls == []


def test_stacks_that_do_not_fit_are_refused(host):
    tables, slab = Gpu(torch.full((4, 4), -1, dtype=torch.int32)), Gpu(torch.zeros((1, 8, 64)))
    ids = torch.arange(7, -1, -1, dtype=torch.int32)
    p = kv16.Pages(tables, 16, slabs=[slab], ids=ids, n_free=3)
    assert p.n_free.item() == 3 and torch.equal(p.ids, ids)
    for n_free in (None, 0, 8):
        assert kv16.Pages(tables, 16, slabs=[slab], ids=ids, n_free=n_free).n_free.item() == (8 if n_free is None else n_free)
    for bad in (dict(ids=ids, n_free=9), dict(ids=ids, n_free=-1), dict(ids=ids[:1]), dict(ids=ids[:7], n_free=3), dict(ids=ids[None])):
        with pytest.raises(ValueError):
            kv16.Pages(tables, 16, slabs=[slab], **bad)


def test_copies_beyond_the_claim_counter_are_refused():
    """Segments are claimed by a 32-bit counter: a call with more of them is refused before its launch (it would never end)."""
    L = sjk.lib()
    p = sjk.PagesC(0x10000, 0x10000, 64, 4, 8, 16)
    p.n_slabs = 2
    p.slabs[0] = p.slabs[1] = sjk.Slab(0x10000, 64 << 10, 0, 1 << 22)        # 4 segments a page and layer
    for n in (128, 256, 2 ** 31 - 1):
        assert L.sjk_pages_copy(C.byref(p), 0x10000, 0x10000, n, None) == -201
    p.n_pages = 1 << 10
    assert L.sjk_pages_extend(C.byref(p), 0x10000, 0x10000, None, 1, 512, 0x10000, None) == -201
    assert L.sjk_pages_compact(C.byref(p), None, None) == -201


@pytest.mark.parametrize("factor,amp", [(1e-5, 1.0), (0.25, 1.0), (1.0, 1.0), (1.5, 0.1 * math.log(1.5) + 1), (40.0, 0.1 * math.log(40.0) + 1)])
def test_yarn_amplitude(factor, amp):
    """The default amplitude is 0.1 ln(factor) + 1 for contexts that grow and 1 for others."""
    assert kv16.rope_steps(64, scaling="yarn", factor=factor, n_ctx=4096)[1] == pytest.approx(amp, rel=2 ** -23)
    assert kv16.rope_steps(64, scaling="yarn", factor=factor, n_ctx=4096, amp=0.7)[1] == pytest.approx(0.7, rel=2 ** -23)


def test_addresses_off_their_types_are_refused():
    """Pointers that are no multiple of what they point at would fault on the device: every call refuses them. (Calls without
    work, which nothing launches.)"""
    L, P = sjk.lib(), 0x10000

    def rows(heads, type, p=P):
        return sjk.Rows(p, 1024, 64, heads, type)

    def cache(**kw):
        c = sjk.Kv16(P, P, 16 * 2 * 64, 2 * 64, 64, kv16.BF16, 64, 2, 16, 8, P, 4, 4)
        for k, v in kw.items():
            setattr(c, k, v)
        return c

    def qkv(**kw):
        a = sjk.QkvArgs()
        a.n_tok, a.head_dim, a.eps, a.pos = 0, 64, 1e-6, P
        a.q, a.k, a.v, a.q_out = rows(4, kv16.BF16), rows(2, kv16.BF16), rows(2, kv16.BF16), rows(4, kv16.F32, 2 * P)
        a.cache = cache()
        for k, v in kw.items():
            setattr(a, k, v)
        return L.sjk_qkv(C.byref(a), None)

    assert qkv() == qkv(rope=sjk.RopeC(64, 0, 1.0, P), rows=P, q_norm=P, k_norm=P, norm_type=kv16.F32) == 0
    for bad in (dict(q=rows(4, kv16.BF16, P + 1)), dict(q_out=rows(4, kv16.F32, P + 2)), dict(k=rows(2, kv16.BF16, P + 3)), dict(pos=P + 2),
                dict(rows=P + 1), dict(q_norm=P + 2, norm_type=kv16.F32), dict(k_norm=P + 1, norm_type=kv16.F16), dict(cache=cache(k=P + 1)),
                dict(cache=cache(v=P + 1)), dict(cache=cache(tables=P + 2))):
        assert qkv(**bad) == -100, bad
    assert qkv(rope=sjk.RopeC(64, 0, 1.0, P + 4)) == -129

    def attend(c=None, q=None, out=None, lens=P, rws=None):
        c, q, out = c or cache(), q or rows(4, kv16.F32), out or rows(4, kv16.F32)
        return L.sjk_kv16_attend(C.byref(c), C.byref(q), lens, rws, 0, 1.0, 0, C.byref(out), P, 1 << 30, None)

    assert attend() == attend(rws=P) == 0
    for bad in (dict(q=rows(4, kv16.F32, P + 2)), dict(q=rows(4, kv16.F16, P + 1)), dict(out=rows(4, kv16.F32, P + 2)),
                dict(out=rows(4, kv16.BF16, P + 1)), dict(lens=P + 2), dict(rws=P + 1), dict(c=cache(tables=P + 1))):
        assert attend(**bad) == -100, bad

    p = sjk.PagesC(P, P, 64, 4, 8, 16)
    r = C.byref(p)
    assert L.sjk_pages_fork(r, P, P, 0, P, None) == L.sjk_pages_extend(r, P, P, P, 1, 0, P, None) == L.sjk_pages_free(r, P, P, P, 0, None) == 0
    assert L.sjk_pages_copy(r, P, P, 0, None) == 0
    for x in (P + 1, P + 2):
        assert L.sjk_pages_fork(r, x, P, 0, P, None) == -100 and L.sjk_pages_fork(r, P, x, 0, P, None) == -100
        assert L.sjk_pages_fork(r, P, P, 0, x, None) == -100
        assert L.sjk_pages_extend(r, x, P, None, 1, 0, P, None) == -100 and L.sjk_pages_extend(r, P, x, None, 1, 0, P, None) == -100
        assert L.sjk_pages_extend(r, P, P, x, 1, 0, P, None) == -100 and L.sjk_pages_extend(r, P, P, None, 1, 0, x, None) == -100
        assert L.sjk_pages_free(r, x, None, None, 0, None) == -100 and L.sjk_pages_free(r, P, x, None, 0, None) == -100
        assert L.sjk_pages_free(r, P, None, x, 0, None) == -100 and L.sjk_pages_compact(r, x, None) == -100
        assert L.sjk_pages_copy(r, x, P, 0, None) == -100 and L.sjk_pages_copy(r, P, x, 0, None) == -100
    p.tables = P + 2
    assert L.sjk_pages_fork(r, P, P, 0, P, None) == -100
