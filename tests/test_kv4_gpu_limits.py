"""The longest rows of the block table that decode takes: 2^24 tokens, with weights, 65536 blocks of the kernel that adds them."""
import math

import pytest
import torch

import mm_rs_with_catlass_b200 as catcoc
from mm_rs_with_catlass_b200.ops import kv4
from test_kv4_gpu import DEV, _make, _ok

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("short", [0, 300])
def test_the_longest_row(short):
    """All pages of the table are one: each of its tokens has one part in 2^18 of the probability that it has in a sequence of one page (or, of the last
    ones, none)."""
    pages, d = 1 << 18, 64
    cache, table, one, k, v, ends, g = _make([64], 1, d, seed=1)
    catcoc.kv4_append(cache, k, v, table, one, ends=ends)
    q = torch.randn(1, 1, d, device=DEV, generator=g).bfloat16()
    long, n = table[:, :1].repeat(1, pages).contiguous(), pages * 64 - short
    w = torch.zeros(1, 1, pages * 64, device=DEV)
    out = catcoc.kv4_decode(q, cache, long, torch.tensor([n], dtype=torch.int32, device=DEV), weights=w)
    _ok()
    want, prob = kv4.kv4_decode_reference(q, cache, table, one)
    count = torch.zeros(pages * 64, dtype=torch.float64, device=DEV)
    count[:n] = 1
    part = prob[0, 0, :64].repeat(pages) * count
    expect = part / part.sum()
    key, value = (x[0, 0, :64] for x in kv4.kv4_read_reference(cache, table, one))
    zero = kv4._parts(cache)[1][table[0].long(), 0].contiguous().view(torch.bfloat16).double()[0, :, 1]
    x = q[0, 0].double()
    big = ((x.abs() * (key.abs() + 2 * zero.abs()[:, None])).sum(-1) * d ** -0.5 * 1.4427).max()
    assert prob[0, 0, :64].min() > 2.0 ** -20 * prob[0, 0, :64].max()           # (no probability is rounded away against the largest)
    # a probability and their sum as in test_kv4_gpu.py; a lane adds up 2^24 / (1000 warps x 8) of them one after the other, half a step each: 2^-13
    e = 2 * (math.log(2) * big * 2.0 ** -19 + 2.0 ** -21) + 2.0 ** -13 + 2.0 ** -15
    assert ((w[0, 0].double() - expect).abs() <= e * expect).all() and (w[0, 0, n:] == 0).all()
    # s <= 2 top / 15, |z| <= top: 8 s <= 1.1 top and 31 s + |z| <= 5.2 top; the tokens left out move the mean by at most 2 top x 300 / 2^24
    top = value.abs().max()
    assert ((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -12 * 1.1 + (e + 2.0 ** -20) * 5.2 + 2.0 ** -14) * top).all()
