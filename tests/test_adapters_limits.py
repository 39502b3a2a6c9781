"""Sizes of adapters beyond what a grid has room for are refused before anything is launched."""
import ctypes

import pytest

from logssms_b200.ops import build

TOO_LARGE = -3


def call(rows, width, features, rank, adapters, code):
    f = build.load("adapters").lb_add_adapters
    p, n, i = ctypes.c_void_p, ctypes.c_long, ctypes.c_int
    f.argtypes = [p, n, p, n, p, n, n, p, n, n, p, p, p, p, n, p, p, n, i, i, i, i, i, p, p]
    launches = i(7)
    code = f(0, features, 0, width, 0, rank * width, width, 0, features * rank, rank, 0, 0, 0, 0, features, 0, 0, rows, width, features, rank,
             adapters, code, ctypes.byref(launches), 0)
    assert launches.value == 0
    return code


@pytest.mark.parametrize("rows,rank,adapters,code", [(1, 65535 * 64 + 1, 1, 0), (1, 65535 * 64 + 1, 1, 1), (4, 65535 * 8 + 1, 8, 0), (512, 65535 * 64 + 1, 8, 0)])
def test_ranks_past_a_grids_limit(rows, rank, adapters, code):
    assert call(rows, 1, 1, rank, adapters, code) == TOO_LARGE


@pytest.mark.parametrize("code", [0, 1])
def test_features_past_a_grids_limit(code):
    assert call(1, 1, 65535 * 64 + 1, 8, 1, code) == TOO_LARGE
