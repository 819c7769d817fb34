"""The choice of pages (sjk_kv16_select) among scores that lie close together, in all three forms of the choice: tables of up to
2,048 pages, up to 8,192, and more. Scores here are sums of a few terms that 64 bits hold exactly, whatever the order, so the lists
have to be those of a plain sort; lists and counts are full of other numbers before the call."""
import random

import pytest

import kv16
import sjk

pytestmark = pytest.mark.gpu
SENTINEL = -77
STRIDES = [64, 3000, 9000]


@pytest.fixture(scope="module")
def T():
    import build
    build.build()
    import torch
    assert torch.cuda.is_available()
    return torch


def _pages(T, dtype, stride, keys, D=64):
    """A sequence per entry of `keys` (a page of one token per key: its first channels), and their bounds."""
    n, most = len(keys), max(len(k) for k in keys)
    cache = kv16.Cache.alloc(1, n * most, 1, 1, D, dtype, n, stride)
    cache.tables[:, :most] = T.arange(n * most, device="cuda").int().view(n, most)
    wide = max(len(x) for k in keys for x in k)
    rows = [list(x) + [0.0] * (wide - len(x)) for k in keys for x in k + [[0.0]] * (most - len(k))]
    cache.k[0, :, 0, 0, :wide] = T.tensor(rows, dtype=T.float64).to(dtype).cuda()
    blocks = kv16.Blocks(cache)
    lens = T.tensor([len(k) for k in keys], dtype=T.int32, device="cuda")
    blocks.update(T.zeros_like(lens), lens)
    return blocks, lens


def _queries(T, rows, dtype, D=64):
    q = T.zeros((len(rows), 1, D), dtype=T.float64)
    for i, r in enumerate(rows):
        q[i, 0, : len(r)] = T.tensor(r, dtype=T.float64)
    return q.to(dtype).cuda()


def _choose(scores, budget):
    pick = sorted(sorted(range(len(scores)), key=lambda b: (-scores[b], b))[:budget])
    return pick + [-1] * (budget - len(pick))


def _check(T, blocks, lens, q, scores, budget):
    n = len(scores)
    lists, count = (T.full(s, SENTINEL, dtype=T.int32, device="cuda") for s in ((n, 1, budget), (n, 1)))
    blocks.select(0, q, lens, budget, sink=0, recent=0, blocks=lists, count=count)
    assert lists[:, 0].tolist() == [_choose(s, budget) for s in scores], f"budget {budget}"
    assert count[:, 0].tolist() == [min(budget, len(s)) for s in scores]


@pytest.mark.parametrize("stride", STRIDES)
def test_some_units_apart(T, stride):
    """Two pages at the border some units of the last place apart, others some hundred above."""
    keys = [[0.5, 0.0], [1.25, 0.0]] + [[1.0, float(h)] for h in (19, 29, 48, 109, 187)]
    blocks, lens = _pages(T, T.bfloat16, stride, [keys])
    q = _queries(T, [[1.0, 2.0 ** -50]], T.bfloat16)
    scores = [[a + b * 2.0 ** -50 for a, b in keys]]
    for budget in range(1, len(keys) + 2):
        _check(T, blocks, lens, q, scores, budget)
    assert sjk.lib().sjk_device_status() == 0


@pytest.mark.parametrize("stride", STRIDES)
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("spread", [1, 8, 200])
def test_one_large_term(T, stride, dtype, spread):
    """Scores with a large term in common (of three sizes) and small differences, ties among them; every budget."""
    r = random.Random(stride + spread)
    n, pages = 12, 50
    keys = [[[r.choice([1.0, 1.0, 1.0, 1.5, 0.25]), float(r.randint(-spread, spread)), r.randint(0, 3) / 4] for _ in range(pages - i)] for i in range(n)]
    blocks, lens = _pages(T, getattr(T, dtype), stride, keys)
    size = [2.0 ** r.choice([20, 30, 38, 43, 45, 47]) for _ in range(n)]
    q = _queries(T, [[s, 1.0, 0.25] for s in size], T.float32)
    scores = [[a * s + b + c / 4 for a, b, c in k] for k, s in zip(keys, size)]
    for budget in range(1, pages + 1):
        _check(T, blocks, lens, q, scores, budget)
    assert sjk.lib().sjk_device_status() == 0


@pytest.mark.parametrize("pages,stride", [(2048, 2048), (8192, 8192), (20000, 20001)])
def test_long_lists_close_together(T, pages, stride):
    """As many pages as each form of the choice takes, in clusters around one large term."""
    r = random.Random(pages)
    keys = [[[1.0, float(r.randint(0, 255)), r.randint(0, 15) / 16] for _ in range(pages)]]
    blocks, lens = _pages(T, T.bfloat16, stride, keys)
    for size in (2.0 ** 36, 2.0 ** 44):
        q = _queries(T, [[size, 1.0, 0.25]], T.float32)
        scores = [[a * size + b + c / 4 for a, b, c in k] for k in keys]
        for budget in (1, 2, 16, 128, 777, pages // 2, pages - 1):
            _check(T, blocks, lens, q, scores, budget)
    assert sjk.lib().sjk_device_status() == 0
