"""Eviction of sequences that are longer than the 4096 tokens which a CTA holds in its registers: the weights pass several times, in stretches; equal weights, of
which the first stay, over the ends of stretches; moves in place, in the launch that picks, and in one of their own."""
import math

import pytest
import torch

import mm_rs_with_catlass_b200 as catcoc
from mm_rs_with_catlass_b200.ops import kv4
from test_kv4_gpu import DEV, _make, _ok

pytestmark = pytest.mark.gpu


def _kept(w, n, keep, recent, sinks):
    """Positions that stay of a head's ``n`` tokens, in order."""
    if n <= keep:
        return list(range(n))
    w = w.tolist()
    heavy = sorted(range(sinks, n - recent), key=lambda i: (w[i] != w[i], -w[i] if w[i] == w[i] else 0.0, i))[:keep - sinks - recent]
    return sorted([*range(sinks), *heavy, *range(n - recent, n)])


def _golden(cache, w, table, lens, keep, recent, sinks, out_table, out_w):
    kept = torch.full((len(lens), cache.shape[1], keep), -1, dtype=torch.int32, device=DEV)
    new, new_w = cache.clone(), out_w.clone()
    for b, n in enumerate(lens):
        for h in range(cache.shape[1]):
            at = torch.tensor(_kept(w[b, h, :n], n, keep, recent, sinks), dtype=torch.long, device=DEV)
            to = torch.arange(len(at), device=DEV)
            kept[b, h, :len(at)] = at.int()
            for src, dst in zip(kv4._parts(cache), kv4._parts(new)):
                dst[out_table[b, to // 64].long(), h, to % 64] = src[table[b, at // 64].long(), h, at % 64]
            new_w[b, h, :len(at)], new_w[b, h, len(at):] = w[b, h, at], 0.0
    return kept, new, new_w


def _weights(g, batch, heads, room, kind):
    w = torch.randn(batch, heads, room, device=DEV, generator=g).exp_()
    if kind == "equal":                    # few values: the border lies among thousands of equal ones
        w = torch.randint(0, 3, w.shape, device=DEV, generator=g).float() * 0.25
    elif kind == "zero":                   # none was looked at: the first ones stay
        w.zero_()
    elif kind == "rising":                 # the last stretch takes nearly all places; its own order is that of the numbers
        w = torch.arange(room, device=DEV).float().expand(w.shape).clone()
    else:
        w[torch.rand(w.shape, device=DEV, generator=g) < 0.3] = 0.0
        w[torch.rand(w.shape, device=DEV, generator=g) < 0.2] = 0.5
        w[0, 0, [40, 4095, 4096]] = torch.tensor([math.inf, -0.0, math.nan], device=DEV)
        w[:, :, 7] = -1.0
    return w


CASES = [([4097], 2048, 100, 4, 2, "mixed"), ([4096, 4097, 8192, 8193, 1], 4000, 64, 1, 2, "mixed"), ([20000], 10000, 256, 4, 2, "mixed"),
         ([20000, 300], 9000, 0, 0, 1, "equal"), ([12289], 5000, 5, 2, 1, "zero"), ([16384], 12000, 4096, 4096, 1, "rising"), ([9000], 1, 0, 0, 3, "equal"),
         ([5000], 4999, 10, 0, 1, "rising"), ([8192] * 2, 4097, 8, 8, 40, "mixed")]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,keep,recent,sinks,heads,kind", CASES)
def test_long_sequences(lens, keep, recent, sinks, heads, kind, d):
    cache, table, kv_lens, k, v, ends, g = _make(lens, heads, d, seed=keep)
    catcoc.kv4_append(cache, k, v, table, kv_lens, ends=ends)
    w = _weights(g, len(lens), heads, table.shape[1] * 64, kind)
    args = dict(recent=recent, sinks=sinks)
    want = _golden(cache, w, table, lens, keep, recent, sinks, table, w)
    got_cache, got_w = cache.clone(), w.clone()
    kept, new = catcoc.kv4_evict(got_cache, got_w, table, kv_lens, keep, **args)
    _ok()
    assert new.tolist() == [min(n, keep) for n in lens] and torch.equal(kept, want[0])
    assert torch.equal(got_cache, want[1]) and torch.equal(got_w.nan_to_num(-7.0), want[2].nan_to_num(-7.0))
    # into other pages, behind the old ones
    width = (keep + 63) // 64
    more = torch.cat((cache, torch.randint(0, 256, (len(lens) * width, *cache.shape[1:]), dtype=torch.uint8, device=DEV, generator=g)))
    new_table = (cache.shape[0] + torch.randperm(len(lens) * width, device=DEV, generator=g)).view(len(lens), width).int()
    new_w = torch.full((len(lens), heads, width * 64 + 3), 9.0, device=DEV)
    want = _golden(more, w, table, lens, keep, recent, sinks, new_table, new_w)
    before = w.clone()
    kept, new = catcoc.kv4_evict(more, w, table, kv_lens, keep, out_table=new_table, out_weights=new_w, **args)
    _ok()
    assert new.tolist() == [min(n, keep) for n in lens] and torch.equal(kept, want[0])
    assert torch.equal(more, want[1]) and torch.equal(new_w.nan_to_num(-7.0), want[2].nan_to_num(-7.0)) and torch.equal(w.nan_to_num(-7.0), before.nan_to_num(-7.0))
