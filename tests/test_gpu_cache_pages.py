"""sjk_pages_* on ledgers whose stack was damaged from outside: nothing is followed beyond its array, nothing half done."""
import pytest

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
