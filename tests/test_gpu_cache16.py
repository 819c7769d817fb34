"""How exact the attention over 16-bit pages is: softmax weights and queries of every size that 32-bit arithmetic keeps,
against the definition in 64 bits.

Error bound of an output element y, with A the same attention over |V|: u |y| for the rounding to the output type, and
(p + 2 e + a) A. p is the relative rounding of a weight: it is the sum of two terms of the cache's type, or of three for
bf16 caches with 32-bit rows: 2^-16 (two bf16 terms of 8 bits), 2^-22 (two f16 terms of 11), 2^-24 (three bf16 terms). e
bounds the error of a score in units of ln 2: 2^-20 (1 + max_t scale sum_d |q_d k_td|). a = 2^-23 (n / 16 + 8): the sums
of n positions, 16 at a time, each of which may drop what lies below 2^-23 of it, and the joins behind them."""
import math

import pytest

import sjk
from test_gpu_kv16 import _build, _dt, _expect

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    import build
    build.build()
    import torch
    assert torch.cuda.is_available()
    return torch


def _check(T, cache, got, q, lens, scale, window=0, rows=None, floor=0.0):
    """floor: what every element may be off beside the bound."""
    split = q.dtype != cache.k.dtype or got.dtype == T.float32
    p = 2.0 ** -22 if cache.k.dtype == T.float16 else 2.0 ** -24 if split else 2.0 ** -16
    u = {T.float32: 2.0 ** -23, T.float16: 2.0 ** -11, T.bfloat16: 2.0 ** -8}[got.dtype]
    tiny = 2.0 ** -25 if got.dtype == T.float16 else 1e-37
    for i, x in enumerate(lens):
        want, mag_v, mag = _expect(T, cache, 0, i if rows is None else rows[i], x, q[i], scale, window)
        bound = u * want.abs() * (1 + 2.0 ** -7) + (p + 2.0 ** -19 * (1 + mag) + 2.0 ** -23 * (x / 16 + 8)) * mag_v + tiny + floor
        err = (got[i].double().cpu() - want).abs()
        assert bool((err <= bound).all()), f"sequence {i} of length {x}: worst {float((err / bound).max()):.3g} of the bound"


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("grp", [1, 8, 13, 20])
@pytest.mark.parametrize("page", [16, 5])
def test_weights_of_16_bit_rows(T, dtype, D, grp, page):
    """Queries and outputs of the cache's type: what is off is the rounding of the output, not that of the weights (elements
    that nearly cancel would show it)."""
    lens = [1, 2, 3, 17, 64, 257, 1000]
    cache, g = _build(T, lens, page, 2, D, _dt(T, dtype), seed=grp)
    q = T.randn((len(lens), 2 * grp, D), device="cuda", generator=g).to(_dt(T, dtype))
    got = cache.attend(0, q, T.tensor(lens, dtype=T.int32, device="cuda"), 1 / math.sqrt(D))
    _check(T, cache, got, q, lens, 1 / math.sqrt(D))
    assert sjk.lib().sjk_device_status() == 0
