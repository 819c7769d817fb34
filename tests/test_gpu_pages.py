"""sjk_pages_* (fork, extend with copy on write, free, compact, copy) against a model in Python that serves the same
calls one entry at a time: the same tables, share counts, stack and page contents."""
import ctypes as C
import random

import numpy as np
import pytest

import gpu_util as gu
import kv16
import sjk

pytestmark = pytest.mark.gpu
FULL, ARG, CORRUPT = -110, -100, -107


@pytest.fixture(scope="module")
def T():
    import build
    build.build()
    import torch
    assert torch.cuda.is_available()
    return torch


class Model:
    """Entries one at a time."""

    def __init__(self, n_pages, rows, stride, page):
        self.stack = list(range(n_pages - 1, -1, -1))
        self.owners = [0] * n_pages
        self.tables = [[-1] * stride for _ in range(rows)]
        self.data = list(range(1000, 1000 + n_pages))       # what a page holds
        self.page = page

    def fork(self, src, dst):
        out = []
        for i, (s, d) in enumerate(zip(src, dst)):
            rows = range(len(self.tables))
            if s not in rows or d not in rows or d in src or d in dst[:i] or any(e != -1 for e in self.tables[d]):
                out.append(ARG)
                continue
            self.tables[d] = list(self.tables[s])
            for e in self.tables[d]:
                if e != -1:
                    self.owners[e] += 1
            out.append(0)
        return out

    def extend(self, rows, lens, adds):
        if len(set(rows)) < len(rows) or any(r not in range(len(self.tables)) for r in rows) or \
                any(n < 0 or a < 0 or (a and (n + a - 1) // self.page >= len(self.tables[0])) for n, a in zip(lens, adds)):
            return ARG
        stack, owners, tables, data = list(self.stack), list(self.owners), [list(t) for t in self.tables], list(self.data)
        for r, n, a in zip(rows, lens, adds):
            for g in range(n // self.page, (n + a - 1) // self.page + 1) if a else ():
                e = tables[r][g]
                if e != -1 and owners[e] == 1:
                    continue
                if not stack:
                    return FULL
                new = stack.pop()
                if e != -1:
                    owners[e] -= 1
                    if g * self.page < n:
                        data[new] = data[e]
                owners[new] = 1
                tables[r][g] = new
        self.stack, self.owners, self.tables, self.data = stack, owners, tables, data
        return 0

    def free(self, rows, first, end):
        gone = set()
        for r, a, b in zip(rows, first, end):
            for g in range(max(a, 0), min(b, len(self.tables[r]))):
                e = self.tables[r][g]
                self.tables[r][g] = -1
                if e != -1:
                    self.owners[e] -= 1
                    if self.owners[e] == 0:
                        gone.add(e)
        self.stack += sorted(gone, reverse=True)

    def compact(self):
        n = len(self.owners)
        top = n - len(self.stack)
        free = set(self.stack)
        to = [e for e in range(top) if e in free]
        frm = [e for e in range(top, n) if e not in free]
        new = dict(zip(frm, to))
        for a, b in new.items():
            self.owners[b], self.owners[a], self.data[b] = self.owners[a], 0, self.data[a]
        self.tables = [[new.get(e, e) for e in t] for t in self.tables]
        self.stack = list(range(n - 1, top - 1, -1))
        return [top, len(to)]


class Device:
    def __init__(self, T, n_pages, rows, stride, page, layers=2, extra=(1,)):
        self.T = T
        self.tables = T.full((rows, stride), -1, dtype=T.int32, device="cuda")
        # slabs of unlike page sizes, int32 words that say (page, layer)
        self.slabs = [T.zeros((layers, n_pages, w), dtype=T.int32, device="cuda") for w in (4, 4100, 8192)]
        for s in self.slabs:
            s += (1000 + T.arange(n_pages, device="cuda", dtype=T.int32))[None, :, None]
            s += (T.arange(layers, device="cuda", dtype=T.int32) * 100000)[:, None, None]
        self.p = kv16.Pages(self.tables, page, slabs=self.slabs)

    def i32(self, x):
        return self.T.tensor(x, dtype=self.T.int32, device="cuda")

    def same(self, m):
        assert self.tables.tolist() == m.tables
        free = self.p.n_free.item()
        assert self.p.ids[:free].tolist() == m.stack
        assert self.p.shares.tolist() == [max(o - 1, 0) for o in m.owners]
        for s in self.slabs:
            first = s[:, :, 0]
            assert bool((s == first[..., None]).all())
            for layer in range(s.shape[0]):
                held = [e for e, o in enumerate(m.owners) if o]
                got = (first[layer] - 100000 * layer).tolist()
                assert [got[e] for e in held] == [m.data[e] for e in held]


@pytest.mark.parametrize("n_pages,rows,stride,page,seed", [(12, 8, 6, 4, 0), (40, 8, 6, 4, 1), (300, 33, 40, 1, 2), (1000, 64, 17, 16, 3),
                                                           (33, 5, 9, 7, 4), (5000, 200, 30, 5, 5)])
def test_random_calls(T, n_pages, rows, stride, page, seed):
    r = random.Random(seed)
    m, d = Model(n_pages, rows, stride, page), Device(T, n_pages, rows, stride, page)
    lens = [0] * rows
    seen = set()
    for call in range(60):
        kind = r.choice(["extend", "extend", "extend", "fork", "free", "compact"])
        if kind == "extend":
            some = r.sample(range(rows), r.randint(1, rows))
            adds = [r.choice([0, 1, 1, 2, r.randint(0, 3 * page)]) for _ in some]
            adds = [min(a, stride * page - lens[i]) for a, i in zip(adds, some)]
            one = r.random() < 0.3 and all(lens[i] < stride * page for i in some)
            got = d.p.extend(d.i32(some), d.i32([lens[i] for i in some]), 1 if one else d.i32(adds))
            want = m.extend(some, [lens[i] for i in some], [1] * len(some) if one else adds)
            assert got.item() == want
            seen.add(want)
            if want == 0:
                for i, a in zip(some, adds):
                    lens[i] += 1 if one else a
        elif kind == "fork":
            empty = [i for i in range(rows) if all(e == -1 for e in m.tables[i])]
            held = [i for i in range(rows) if i not in empty] or [0]
            dst = r.sample(empty, min(len(empty), r.randint(1, 6))) or [0]
            src = [r.choice(held) for _ in dst]
            if r.random() < 0.2:
                dst[-1] = r.choice(held)                    # not empty
            got = d.p.fork(d.i32(src), d.i32(dst)).tolist()
            want = m.fork(src, dst)
            assert got == want
            for s, t, w in zip(src, dst, want):
                if w == 0:
                    lens[t] = lens[s]
        elif kind == "free":
            some = r.sample(range(rows), r.randint(1, max(1, rows // 3)))
            cut = r.random() < 0.5
            first = [-(-r.randint(0, lens[i]) // page) if cut else 0 for i in some]
            if cut:
                d.p.free(d.i32(some), first=d.i32(first))
            else:
                d.p.free(d.i32(some))
            m.free(some, first, [stride] * len(some))
            for i, f in zip(some, first):
                lens[i] = min(lens[i], f * page)
        else:
            assert d.p.compact().tolist() == m.compact()
        if call % 7 == 0 or call == 59:
            d.same(m)
    assert 0 in seen and (n_pages > 12 or FULL in seen)
    assert sjk.lib().sjk_device_status() == 0


def test_last_owner_keeps_the_page(T):
    """All owners of a partly filled page write on: the last in the call keeps it, the others copy; a truncated owner's
    shared page that holds nothing of it any more is replaced without a copy."""
    m, d = Model(16, 4, 3, 4), Device(T, 16, 4, 3, 4)
    for x in (m, d):
        n = (lambda v: v) if x is m else d.i32
        (x if x is m else x.p).extend(n([0]), n([0]), n([6]))
        (x if x is m else x.p).fork(n([0, 0, 0]), n([3, 1, 2]))
    assert d.p.extend(d.i32([3, 0, 2, 1]), d.i32([6, 6, 6, 6]), 1).item() == m.extend([3, 0, 2, 1], [6] * 4, [1] * 4) == 0
    d.same(m)
    assert d.tables[1, 1].item() == 1                       # row 1 came last
    assert d.p.extend(d.i32([0]), d.i32([0]), 3).item() == m.extend([0], [0], [3]) == 0      # written anew from position 0
    d.same(m)


def test_extend_is_all_or_nothing(T):
    m, d = Model(5, 3, 8, 2), Device(T, 5, 3, 8, 2)
    assert d.p.extend(d.i32([0]), d.i32([0]), 5).item() == m.extend([0], [0], [5]) == 0
    d.p.fork(d.i32([0]), d.i32([1]))
    m.fork([0], [1])
    for rows, lens, adds, rc in (([0, 1], [5, 5], [3, 4], FULL), ([2], [0], [16], FULL), ([0, 0], [5, 5], [1, 1], ARG), ([3], [0], [1], ARG),
                                 ([-1], [0], [1], ARG), ([2], [-1], [1], ARG), ([2], [0], [17], ARG), ([2], [2 ** 31 - 1], [2 ** 31 - 1], ARG)):
        assert d.p.extend(d.i32(rows), d.i32(lens), d.i32(adds)).item() == rc == m.extend(rows, lens, adds)
        d.same(m)
    assert d.p.extend(d.i32([1, 0, 2]), d.i32([5, 5, 0]), d.i32([1, 0, 2])).item() == m.extend([1, 0, 2], [5, 5, 0], [1, 0, 2]) == 0
    d.same(m)
    d.tables[2, 0] = 5
    assert d.p.extend(d.i32([1, 2]), d.i32([6, 0]), 1).item() == CORRUPT
    assert d.p.fork(d.i32([2]), d.i32([2])).tolist() == [ARG]
    d.p.free(d.i32([1]))
    m.free([1], [0], [8])
    assert d.p.fork(d.i32([2]), d.i32([1])).tolist() == [CORRUPT]
    assert sjk.lib().sjk_device_status() == 0
    d.p.free(d.i32([2, 7, -3]))                             # the entry that is no page goes, rows out of range are reported
    assert sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE
    m.tables[2][0] = -1
    d.same(m)


def test_fork_refusals(T):
    m, d = Model(12, 5, 4, 2), Device(T, 12, 5, 4, 2)
    d.p.extend(d.i32([0, 1]), d.i32([0, 0]), 4)
    m.extend([0, 1], [0, 0], [4, 4])
    for src, dst in (([0, 0], [2, 2]), ([0, 3], [3, 4]), ([0, 5, -1], [5, 3, 4]), ([0], [1]), ([0], [0])):
        assert d.p.fork(d.i32(src), d.i32(dst)).tolist() == m.fork(src, dst)
        d.same(m)


@pytest.mark.parametrize("first,end", [([0, 2], [1, 4]), ([-5, 3], [2, 100]), ([2, 2], [2, 1]), ([0, 0], [-1, 9])])
def test_free_ranges_and_repeats(T, first, end):
    """Ranges are cut to the table; a row named twice gives an entry up once."""
    m, d = Model(20, 3, 5, 2), Device(T, 20, 3, 5, 2)
    d.p.extend(d.i32([0, 1]), d.i32([0, 0]), 9)
    m.extend([0, 1], [0, 0], [9, 9])
    d.p.fork(d.i32([0]), d.i32([2]))
    m.fork([0], [2])
    d.p.free(d.i32([2, 1]), first=d.i32(first), end=d.i32(end))
    m.free([2, 1], first, end)
    d.same(m)
    d.p.free(d.i32([0, 0, 0, 1]))
    m.free([0, 0, 0, 1], [0] * 4, [5] * 4)
    d.same(m)


@pytest.mark.parametrize("n_pages", [1, 31, 32, 33, 1025, 70000, 1 << 20])
def test_compact_sizes(T, n_pages):
    """Every bitmap shape, from one page to the most a ledger holds."""
    tables = T.full((2, n_pages), -1, dtype=T.int32, device="cuda")
    slab = (1000 + T.arange(n_pages, dtype=T.int32, device="cuda")).view(1, n_pages, 1).expand(1, n_pages, 4).contiguous()
    p = kv16.Pages(tables, 1, slabs=[slab])
    i32 = lambda x: T.tensor(x, dtype=T.int32, device="cuda")  # noqa: E731
    assert p.extend(i32([0]), i32([0]), n_pages).item() == 0
    assert T.equal(tables[0], T.arange(n_pages, dtype=T.int32, device="cuda"))
    keep = T.rand(n_pages, device="cuda") < 0.3
    tables[1] = T.where(keep, -1, tables[0])
    tables[0] = T.where(keep, tables[0], -1)
    p.free(i32([1]))
    used = int(keep.sum())
    held = tables[0][keep].clone()
    assert p.n_free.item() == n_pages - used
    assert T.equal(p.ids[: n_pages - used], (~keep).nonzero()[:, 0].int().flip(0))
    moved = int((held >= used).sum())
    assert p.compact().tolist() == [used, moved]
    now = tables[0][keep]
    assert T.equal(now.sort().values, T.arange(used, dtype=T.int32, device="cuda"))
    assert T.equal(slab[0, now.long(), 3], held + 1000)
    assert T.equal(p.ids[: n_pages - used], T.arange(n_pages - 1, used - 1, -1, dtype=T.int32, device="cuda"))
    assert p.compact().tolist() == [used, 0] and sjk.lib().sjk_device_status() == 0


def test_copy_and_its_bounds(T):
    d = Device(T, 10, 2, 3, 4)
    d.p.copy(d.i32([1, 3, 10, 4]), d.i32([2, 7, 5, -1]))
    for s in d.slabs:
        for layer in range(2):
            assert [x - 100000 * layer for x in s[layer, :, 0].tolist()] == [1000, 1001, 1001, 1003, 1004, 1005, 1006, 1003, 1008, 1009]
            assert bool((s[layer] == s[layer, :, :1]).all())
    assert sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE


def test_reserve_batch_on_a_ledger(T):
    """sjk_pool_reserve_batch works on a ledger's memory, and its blocks can be forked and freed."""
    L = sjk.lib()
    d = Device(T, 12, 3, 4, 2)
    req = (sjk.BlockReq * 1)(sjk.BlockReq(d.tables[0].data_ptr(), 0, 3))
    st = T.ones(1, dtype=T.int32, device="cuda")
    sjk.check(L.sjk_pool_reserve_batch(C.c_void_p(d.p._buf.data_ptr()), req, 1, gu.ptr(st), None))
    assert st.item() == 0 and d.tables[0].tolist() == [0, 1, 2, -1] and d.p.n_free.item() == 9
    assert d.p.fork(d.i32([0]), d.i32([1])).tolist() == [0]
    d.p.free(d.i32([0]))
    assert d.p.n_free.item() == 9
    d.p.free(d.i32([1]))
    assert d.p.ids[:12].tolist() == list(range(11, -1, -1))


def test_forked_sealed_sequence(T):
    """The record pool under a ledger: a sealed sequence's table forked, the pool compacted, and attention through the
    fork's table gives the bits it gave through the first."""
    L = sjk.lib()
    D, H, npos, n_ub, tail, tail_max, n_layers = 256, 4, 1536, 128, 256, 512, 2
    cfg = sjk.config(D, H, 4096, n_ub, bits_k=3, bits_v=3, body=1, tail=tail, tail_max=tail_max)
    pool = sjk.Pool()
    n_blocks = 64
    sjk.check(L.sj_kvarn_pool_init(C.byref(pool), C.byref(cfg), n_layers, n_blocks))
    for i in range(20):                                     # scattered blocks: ids above the used number are handed out
        L.sj_kvarn_pool_alloc(C.byref(pool))
    s = gu.DevSeq(cfg, n_layers, pool)
    rng = np.random.default_rng(0)
    for pos in range(0, npos, n_ub):
        sjk.check(s.begin_ubatch(pos, n_ub))
        k, v = (T.from_numpy(rng.standard_normal((n_layers, n_ub, H, D)).astype(np.float32)).cuda() for _ in range(2))
        sjk.check(L.sjk_seq_store(C.byref(s.s), pos, n_ub, gu.ptr(k), gu.ptr(v), 0, 1, None))
    T.cuda.synchronize()
    groups = (s.pol.B - 128) // 128
    assert groups >= 4
    block = H * pool.lay.bytes
    # a ledger over the slab: the host pool's stack, one more table row for the fork
    tables = T.full((2, int(s.s.layers[0].n_groups)), -1, dtype=T.int32, device="cuda")
    tables[0, :groups] = T.tensor([int(s.s.blocks[g]) for g in range(groups)], dtype=T.int32, device="cuda")
    size = L.sjk_pages_bytes(n_blocks)
    ledger = T.empty(size, dtype=T.uint8, device="cuda")
    p = sjk.PagesC(ledger.data_ptr(), tables.data_ptr(), n_blocks, 2, tables.shape[1], 128)
    p.n_slabs = 1
    p.slabs[0] = sjk.Slab(pool.body, block, block * n_blocks, n_layers)
    sjk.check(L.sjk_pages_init(C.byref(p), None))
    for i in range(20):                                     # what stood for other sequences is free again
        L.sj_kvarn_pool_release(C.byref(pool), i)
    sjk.check(L.sjk_pool_dev_load(gu.ptr(ledger), C.byref(pool), None))
    q = T.randn((16, D), device="cuda")
    view = sjk.view_of(s.s.layers[1])

    def attend(row):
        view.blocks = tables[row].data_ptr()
        out = T.empty_like(q)
        n = L.sjk_attend_scratch_bytes(C.byref(view), npos, 1, 16)
        scratch = T.empty(n, dtype=T.uint8, device="cuda")
        sjk.check(L.sjk_attend(C.byref(view), s.pol.B, npos, npos - 1, 1, 16, gu.ptr(q), 1 / 16, gu.ptr(out), gu.ptr(scratch), n, None))
        return out

    want = attend(0)
    i32 = lambda x: T.tensor(x, dtype=T.int32, device="cuda")  # noqa: E731
    st, info = i32([1]), i32([0, 0])
    a, b, one = i32([0]), i32([1]), i32([0])
    sjk.check(L.sjk_pages_fork(C.byref(p), a.data_ptr(), b.data_ptr(), 1, st.data_ptr(), None))
    assert st.item() == 0 and T.equal(attend(1), want)
    sjk.check(L.sjk_pages_free(C.byref(p), one.data_ptr(), None, None, 1, None))
    sjk.check(L.sjk_pages_compact(C.byref(p), info.data_ptr(), None))
    assert info.tolist() == [groups, groups]
    assert sorted(tables[1, :groups].tolist()) == list(range(groups))
    assert T.equal(attend(1), want)
    sjk.check(L.sjk_pool_dev_store(gu.ptr(ledger), C.byref(pool), None))
    assert pool.n_free == n_blocks - groups and pool.free_ids[pool.n_free - 1] == groups
    assert L.sjk_device_status() == 0
    s.close()
    L.sj_kvarn_pool_free(C.byref(pool))
