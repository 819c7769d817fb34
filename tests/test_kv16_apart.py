"""Outputs that lie over inputs which other parts of the same launch still read are refused, before anything reaches the device."""
import ctypes as C

import pytest

import sjk
from test_kv16 import P, _cache


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
