"""Windowed decode over the 4-bit cache where a CTA's run holds several blocks of a unit: a window begins inside a block, or two blocks, of which
its warps take two or four tiles at once. Stages of one to four blocks, windows from every tile of a block on, sinks that end inside one; the rows of every
form of the kernel (four, eight, sixteen), with and without weights. Tolerances: those of test_kv4_gpu.py."""
import pytest
import torch

import mm_rs_with_catlass_b200 as catcoc
from test_kv4_gpu import DEV, _attend, _make

pytestmark = pytest.mark.gpu

EVEN, ODD, RAGGED = [4096] * 16, [4100] * 16, [4001 - 211 * i for i in range(16)]


def _windowed(lens, heads, group, q_len, d, window, sinks, dtype=torch.bfloat16, weights=False):
    cache, table, kv_lens, k, v, ends, g = _make(lens, heads, d, seed=window + sinks, dtype=dtype)
    catcoc.kv4_append(cache, k, v, table, kv_lens, ends=ends)
    q = torch.randn(len(lens) * q_len, heads * group, d, device=DEV, generator=g).to(dtype)
    w = torch.rand(len(lens), heads, table.shape[1] * 64, device=DEV, generator=g) if weights else None
    return _attend(q, cache, table, kv_lens, q_len=q_len, window=window, sinks=sinks, weights=w)


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("d,group,q_len", [(128, 4, 1), (128, 1, 3), (128, 8, 1), (128, 4, 2), (128, 16, 1), (64, 1, 1), (64, 4, 2), (64, 3, 4)])
@pytest.mark.parametrize("lens,window,sinks", [(EVEN, 1000, 4), (ODD, 1024, 4), (RAGGED, 777, 0), (RAGGED, 1024, 70)])
def test_windows_over_runs(lens, window, sinks, d, group, q_len, weights):
    _windowed(lens, 8, group, q_len, d, window, sinks, weights=weights)


@pytest.mark.parametrize("start", range(0, 128, 9))
def test_windows_that_begin_anywhere(start):
    """The first token of the window at every kind of place among the tiles of two blocks."""
    for d, dtype in ((128, torch.bfloat16), (64, torch.float16)):
        for n in (4096, 4100, 2017):
            _windowed([n] * 6, 8, 4, 1, d, n - 1024 - start, 33, dtype=dtype, weights=start % 2 == 1)


def test_long_window_of_one_sequence():
    """Runs of many stages of one unit, the window's start in the first of them."""
    for group, d in ((4, 128), (8, 128), (2, 64)):
        for window in (60000, 60001, 60017, 60040):
            _windowed([70001], 2, group, 1, d, window, 130)
