"""Edges of the calls for several new tokens and for chosen pages: what lies behind a list's end, sequences of one
position, and positions past the last one that 32 bits number."""
import pytest

import kv16
import sjk
from test_gpu_blocks import _cache, _check, _ints

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    import build
    build.build()
    import torch
    assert torch.cuda.is_available()
    return torch


def test_nothing_counts_behind_a_list(T):
    """Entries behind a list's -1 are not looked at: whatever they are, the result is that of the list and nothing is reported."""
    lens = [200, 90]
    cache, g = _cache(T, lens, 16, 2, 64, T.bfloat16)
    blocks = kv16.Blocks(cache)
    q = T.randn((2, 4, 64), device="cuda", generator=g).bfloat16()
    tail = [5, 4, 2 ** 31 - 1, -2 ** 31, -9, 3, 3, 100] * 6
    for head in ([], [3], [0, 5], list(range(6))):
        mine = [[(head + [-1] + tail)[:40]] * 2] * 2
        out = blocks.attend(0, q, _ints(T, lens), _ints(T, mine), 0.1)
        _check(T, cache, out, q, lens, [[head] * 2] * 2, 0.1)
        assert sjk.lib().sjk_device_status() == 0
    # what ends a list without a -1 is reported, as before, wherever in the list it is
    for at in (1, 31, 32, 33, 39):
        for wrong in (0, -2, 13):
            cache, g = _cache(T, [40 * 16], 16, 1, 64, T.bfloat16)
            mine = list(range(40))
            mine[at] = wrong if wrong != 13 else 10 ** 6
            q1 = T.randn((1, 2, 64), device="cuda", generator=g).bfloat16()
            out = kv16.Blocks(cache).attend(0, q1, _ints(T, [640]), _ints(T, [[mine]]), 0.1)
            _check(T, cache, out, q1, [640], [[mine[:at]]], 0.1)
            assert sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE


def test_lists_over_short_sequences(T):
    """Lists over sequences of one position and of none."""
    lens = [1, 0, 17, 1]
    cache, g = _cache(T, [max(x, 1) for x in lens], 16, 2, 64, T.bfloat16)
    q = T.randn((4, 6, 64), device="cuda", generator=g).bfloat16()
    lists = [[[0, -1, -1]] * 2, [[-1, -1, -1]] * 2, [[1, -1, -1], [0, 1, -1]], [[-1, -1, -1], [0, -1, -1]]]
    out = kv16.Blocks(cache).attend(0, q, _ints(T, lens), _ints(T, lists), 0.1)
    _check(T, cache, out, q, lens, lists, 0.1)
    assert bool((out[0] != 0).any()) and bool((out[3, 3:] != 0).any()) and sjk.lib().sjk_device_status() == 0
    # (a list over a sequence without positions: its pages lie behind it)
    out = kv16.Blocks(cache).attend(0, q, _ints(T, [-3, 0, 1, 1]), _ints(T, [[[0, -1, -1]] * 2] * 4), 0.1)
    _check(T, cache, out, q, [0, 0, 1, 1], [[[]] * 2, [[]] * 2, [[0]] * 2, [[0]] * 2], 0.1)
    assert sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE


def test_kept_positions_end_at_2_31(T):
    """Paths that reach past position 2^31 - 2 are left out, as the maps leave such tokens out, however long the table row is."""
    page, D = 2 ** 20, 64
    cache = kv16.Cache.alloc(1, 2, page, 1, D, T.bfloat16, 1, 2050)
    g = T.Generator(device="cuda")
    g.manual_seed(1)
    cache.k.normal_(generator=g)
    cache.v.normal_(generator=g)
    cache.tables.fill_(-1)
    cache.tables[0, 2047:2049] = _ints(T, [1, 0])
    length, k, v = 2 ** 31 - 6, cache.k.clone(), cache.v.clone()
    for path in ([0, 2, 6], [1, 3, 5], [7]):
        new = cache.keep(_ints(T, [length]), _ints(T, [path]), _ints(T, [len(path)]))
        assert new.tolist() == [length] and sjk.lib().sjk_device_status() == sjk.DEVICE_PAGE
        assert T.equal(cache.k, k) and T.equal(cache.v, v)
    new = cache.keep(_ints(T, [length]), _ints(T, [[1, 4]]), _ints(T, [2]))
    assert new.tolist() == [length + 2] and sjk.lib().sjk_device_status() == 0
    place = page - 6
    assert T.equal(cache.k[0, 1, place: place + 2], k[0, 1, [place + 1, place + 4]]) and T.equal(cache.v[0, 1, place: place + 2], v[0, 1, [place + 1, place + 4]])


def test_new_lengths_beside_the_inputs(T):
    """Lengths, paths, counts, rows and new lengths side by side in one buffer."""
    cache, g = _cache(T, [60, 60, 60], 16, 1, 64, T.bfloat16)
    k, v = cache.k.clone(), cache.v.clone()
    buf = _ints(T, [50, 51, 52] + [1, 3, 0, 2, 4, 5] + [2, 1, 2] + [7, 7, 7] + [2, 1, 0])
    lens, path, count, new, rows = buf[:3], buf[3:9].view(3, 2), buf[9:12], buf[12:15], buf[15:]
    assert cache.keep(lens, path, count, rows=rows, new_lens=new) is new
    assert buf.tolist() == [50, 51, 52, 1, 3, 0, 2, 4, 5, 2, 1, 2, 52, 52, 54, 2, 1, 0] and sjk.lib().sjk_device_status() == 0
    for row, length, p in ((2, 50, [1, 3]), (1, 51, [0]), (0, 52, [4, 5])):
        for j, t in enumerate(p):
            a, b = ((int(cache.tables[row, x // 16]), x % 16) for x in (length + t, length + j))
            assert T.equal(cache.k[0, b[0], b[1]], k[0, a[0], a[1]]) and T.equal(cache.v[0, b[0], b[1]], v[0, a[0], a[1]])
