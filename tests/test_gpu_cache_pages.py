"""sjk_pages_* on ledgers whose stack was damaged from outside (nothing is followed beyond its array, nothing half done), and
over caches of other layouts."""
import pytest

import kv16
import sjk
from test_gpu_pages import CORRUPT, FULL, Device, Model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    import build
    build.build()
    import torch
    assert torch.cuda.is_available()
    return torch


def _pair(T, n_pages=20, rows=4, stride=8, page=2):
    m, d = Model(n_pages, rows, stride, page), Device(T, n_pages, rows, stride, page)
    assert d.p.extend(d.i32([0, 1]), d.i32([0, 0]), 5).item() == m.extend([0, 1], [0, 0], [5, 5]) == 0
    d.p.fork(d.i32([0]), d.i32([2]))
    m.fork([0], [2])
    return m, d


@pytest.mark.parametrize("n_free", [21, 1 << 20, -1])
def test_more_free_ids_than_pages(T, n_free):
    m, d = _pair(T)
    was = d.p.n_free.item()
    d.p.n_free.fill_(n_free)
    before = d.p._buf.clone(), d.tables.clone()
    assert d.p.extend(d.i32([3]), d.i32([0]), 3).item() == CORRUPT
    assert d.p.compact().tolist()[1] == 0 and sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE
    ids = slice(4, 24)
    assert T.equal(d.p._buf[ids], before[0][ids]) and T.equal(d.tables, before[1]) and T.equal(d.p.n_free, before[0][:1])
    d.p.n_free.fill_(was)
    d.same(m)
    assert d.p.extend(d.i32([3]), d.i32([0]), 3).item() == m.extend([3], [0], [3]) == 0
    d.same(m)


def test_pages_given_back_to_a_torn_stack(T):
    m, d = _pair(T)
    for n_free in (20, 25, -1):                             # full although rows hold pages; beyond the pool
        d.p.n_free.fill_(n_free)
        d.p.free(d.i32([1 if n_free == 20 else 0]))
        assert sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE and d.p.n_free.item() == 20


@pytest.mark.parametrize("depth,bad", [(0, 20), (2, 1 << 30), (3, -1)])
def test_ids_of_the_stack_that_are_no_pages(T, depth, bad):
    """An extend that would hand such an id out does nothing; one that takes the ids above it works."""
    m, d = _pair(T)
    at = d.p.n_free.item() - 1 - depth
    was = d.p.ids[at].item()
    d.p.ids[at] = bad
    assert d.p.extend(d.i32([3, 0]), d.i32([0, 5]), d.i32([2 * depth + 1, 1])).item() == CORRUPT
    d.p.ids[at] = was
    d.same(m)
    d.p.ids[at] = bad
    if depth:
        assert d.p.extend(d.i32([3]), d.i32([0]), 2 * depth).item() == m.extend([3], [0], [2 * depth]) == 0
    d.p.ids[at] = was
    d.same(m)
    assert sjk.lib().sjk_device_status() == 0


def test_bad_ids_deep_in_a_large_request(T):
    """More pages than the bookkeeping has threads."""
    m, d = Model(900, 3, 700, 1), Device(T, 900, 3, 700, 1)
    at = 900 - 1 - 600
    was = d.p.ids[at].item()
    d.p.ids[at] = 900
    assert d.p.extend(d.i32([0]), d.i32([0]), 601).item() == CORRUPT
    d.p.ids[at] = was
    d.same(m)
    d.p.ids[at] = 900
    assert d.p.extend(d.i32([0]), d.i32([0]), 600).item() == m.extend([0], [0], [600]) == 0
    d.p.ids[at] = was
    d.same(m)
    assert d.p.extend(d.i32([1]), d.i32([0]), 301).item() == FULL == m.extend([1], [0], [301])
    d.same(m)


@pytest.mark.parametrize("layout", ["heads first", "interleaved"])
def test_ledgers_over_other_layouts(T, layout):
    """Caches whose K and V are views of whole pages: the ledger's slab is the tensor that they came from."""
    n, page, H, D = 12, 16, 2, 64
    if layout == "heads first":
        slabs = [T.zeros((1, n, H, page, D), dtype=T.bfloat16, device="cuda") for _ in range(2)]
        k, v = (x.transpose(2, 3) for x in slabs)
    else:
        slabs = [T.zeros((1, n, page, H, 2, D), dtype=T.bfloat16, device="cuda")]
        k, v = slabs[0][..., 0, :], slabs[0][..., 1, :]
    cache = kv16.Cache(k, v, T.full((2, 4), -1, dtype=T.int32, device="cuda"))
    pages = kv16.Pages(cache.tables, page, slabs=slabs)
    i32 = lambda x: T.tensor(x, dtype=T.int32, device="cuda")  # noqa: E731
    pages.extend(i32([0]), i32([0]), 20)
    T.manual_seed(0)
    rows = [T.randn((21, H, D), device="cuda").bfloat16() for _ in range(2)]
    step = kv16.Qkv(D, cache=cache)
    step(k=rows[0][:20], v=rows[1][:20], pos=T.arange(20, dtype=T.int32, device="cuda"), rows=i32([0] * 20))
    q = T.randn((1, 4, D), device="cuda").bfloat16()
    want = cache.attend(0, q, i32([20]), 0.125, rows=i32([0]))
    assert pages.fork(i32([0]), i32([1])).tolist() == [0]
    assert pages.extend(i32([1]), i32([20]), 1).item() == 0         # splits the last page, which gets its contents
    assert cache.tables[:, :2].tolist() == [[0, 1], [0, 2]]
    step(k=rows[0][20:], v=rows[1][20:], pos=i32([20]), rows=i32([1]))
    assert T.equal(cache.attend(0, q, i32([20]), 0.125, rows=i32([0])), want)
    assert T.equal(cache.attend(0, q, i32([20]), 0.125, rows=i32([1])), want)
    at = cache.tables[1].long()
    got = T.cat((cache.k[0, at[0]], cache.k[0, at[1], :5]))
    assert T.equal(got, rows[0])
    assert sjk.lib().sjk_device_status() == 0
