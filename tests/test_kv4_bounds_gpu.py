"""The 4-bit cache at the ends of what its tables name: lengths that a row cannot hold, and pages that are not in the cache."""
import math

import pytest
import torch

import mm_rs_with_catlass_b200 as catcoc
from mm_rs_with_catlass_b200.ops import kv4
from mm_rs_with_catlass_b200.ops._common import StatusError, local_status, raise_on_status
from test_kv4_gpu import DEV, _make

pytestmark = pytest.mark.gpu


def _noted(call):
    result = call()
    torch.cuda.synchronize()
    with pytest.raises(StatusError):
        raise_on_status(local_status(torch.device("cuda", 0)), "kv4")
    return result


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("new,length", [(1, 193), (5, 195), (5, 200), (5, 197), (200, 193), (1, 0x7fffffff), (5, -1), (5, 3), (1, -0x80000000), (200, -0x80000000)])
def test_append_outside_of_the_tables_row(new, length, ragged, d):
    """Three pages hold 192 tokens. Tokens whose positions lie outside of them change no byte of the cache; the others are written, and so are those of the
    other sequences."""
    cache, table, _, _, _, _, g = _make([192, 192], 2, d, seed=new)
    k, v = (torch.randn(2 * new, 2, d, device=DEV, generator=g).bfloat16() for _ in range(2))
    for bad in (0, 1):
        lens = [192, 192]
        if new > 192:
            lens = [new, new]
        lens[bad] = length
        want = cache.clone()
        for b in (0, 1):
            places = [lens[b] - new + t for t in range(new)]
            rows = [t for t in range(new) if 0 <= places[t] < 192]
            if rows:                       # (they are consecutive, the last one at places[rows[-1]])
                kept = slice(b * new + rows[0], b * new + rows[-1] + 1)
                kv4.kv4_append_reference(want, k[kept], v[kept], table[b:b + 1], torch.tensor([places[rows[-1]] + 1], device=DEV))
        got = cache.clone()
        ends = torch.tensor([new, 2 * new], dtype=torch.int32, device=DEV) if ragged else None
        _noted(lambda: catcoc.kv4_append(got, k, v, table, torch.tensor(lens, dtype=torch.int32, device=DEV), ends=ends))
        assert torch.equal(got, want)


def _without(q, cache, table, kv_lens, there, q_len, window, sinks):
    """(output, probabilities summed over a KV head's rows, tolerance of the output) in 64 bits over the tokens of the pages that are ``there [B, pages]``. The bounds
    are those of test_kv4_gpu.py, with s code at most |value| + |z|."""
    d, heads, room = q.shape[2], cache.shape[1], table.shape[1] * 64
    batch, group, scale = table.shape[0], q.shape[1] // cache.shape[1], q.shape[2] ** -0.5
    out, tol = (torch.zeros(q.shape, dtype=torch.float64, device=DEV) for _ in range(2))
    sums = torch.zeros(batch, heads, room, dtype=torch.float64, device=DEV)
    for b in range(batch):
        n = int(kv_lens[b])
        k, v = (x[0, :, :n] for x in kv4.kv4_read_reference(cache, table[b:b + 1], kv_lens[b:b + 1]))
        params = [p[table[b].long()].transpose(1, 2).flatten(0, 1)[:n].contiguous().view(torch.bfloat16).double().unflatten(-1, (-1, 2)).transpose(0, 1)
                  for p in kv4._parts(cache)[1::2]]                                                # [heads, n, groups, 2]
        s, z = ([p[..., i].repeat_interleave(64, -1) for p in params] for i in (0, 1))
        j = torch.arange(n, device=DEV)
        for t in range(q_len):
            p = n - q_len + t
            seen = (j <= p) & there[b].repeat_interleave(64)[:n]
            if window is not None:
                seen = seen & ((p - j < window) | (j < sinks))
            if not bool(seen.any()):
                continue
            x = q[b * q_len + t].double().view(heads, group, d)
            prob = torch.softmax(torch.einsum("hgd,hnd->hgn", x, k[:, seen]) * scale, -1)
            row = torch.einsum("hgn,hnd->hgd", prob, v[:, seen])
            big = (torch.einsum("hgd,hnd->hgn", x.abs(), k[:, seen].abs() + 2 * z[0][:, seen].abs()) * scale * 1.4427).amax(-1, keepdim=True)
            e = 2 * (math.log(2) * big * 2.0 ** -19 + 2.0 ** -21)
            unit = s[1][:, seen]
            centred = torch.einsum("hgn,hnd->hgd", prob, (v[:, seen] - z[1][:, seen] - 8 * unit).abs())
            abs_v = torch.einsum("hgn,hnd->hgd", prob, v[:, seen].abs() + 2 * z[1][:, seen].abs() + 16 * unit)
            floor = 2.0 ** -38 * 15 * n * 15 * unit.amax(1)[:, None]
            out[b * q_len + t] = row.reshape(-1, d)
            tol[b * q_len + t] = (2.0 ** -12 * centred + (e + 2.0 ** -20) * abs_v + floor + torch.finfo(q.dtype).eps / 2 * row.abs()).reshape(-1, d)
            sums[b, :, :n][:, seen] += prob.sum(1)
    return out, sums, tol


@pytest.mark.parametrize("window,sinks", [(None, 0), (900, 70)])
@pytest.mark.parametrize("d,group,q_len", [(128, 4, 1), (128, 8, 1), (128, 16, 1), (64, 3, 2), (64, 16, 1)])
@pytest.mark.parametrize("kind", ["few", "many", "long"])
def test_decode_leaves_out_what_is_not_in_the_cache(d, group, q_len, window, sinks, kind):
    """Attention is that over the other pages' tokens, and their weights alone change; stages of which some blocks or all are missing, sequences
    without the first page, the last, or any. What the missing blocks' places in shared memory held before does not show."""
    lens = {"many": [2100 - 97 * i for i in range(16)], "few": [700, 300, 64, 333, 190, 77, 1, 500], "long": [45000, 44001, 64, 333, 190, 77, 1, 500]}[kind]
    heads = {"many": 4, "few": 1, "long": 8}[kind]            # (long: runs of more than 32 blocks, whose names come 32 at a time)
    cache, table, kv_lens, k, v, ends, g = _make(lens, heads, d, seed=group, extra=1)
    catcoc.kv4_append(cache, k, v, table, kv_lens, ends=ends)
    there = torch.rand(table.shape, device=DEV, generator=g) > 0.15
    there[0], there[1] = True, True
    there[0, 1:6], there[1, 4], there[2], there[3, 0], there[4, (lens[4] - 1) // 64], there[7] = False, False, False, False, False, True
    names = torch.tensor([-1, cache.shape[0], 0x7fffffff, -0x80000000], dtype=torch.int32, device=DEV)
    bad = torch.where(there, table, names[torch.randint(0, 4, table.shape, device=DEV, generator=g)])
    q = torch.randn(len(lens) * q_len, heads * group, d, device=DEV, generator=g).bfloat16()
    base = torch.rand(len(lens), heads, table.shape[1] * 64, device=DEV, generator=g)
    want, sums, tol = _without(q, cache, table, kv_lens, there, q_len, window, sinks)
    w = base.clone()
    args = dict(q_len=q_len, window=window, sinks=sinks)
    # other numbers first, so that a place that is read in vain holds something large
    catcoc.kv4_decode(q, torch.full_like(cache, 0x47), table, kv_lens, **args)
    plain = _noted(lambda: catcoc.kv4_decode(q, cache, bad, kv_lens, **args))
    out = _noted(lambda: catcoc.kv4_decode(q, cache, bad, kv_lens, weights=w, **args))
    assert torch.equal(out, plain) and (out[2 * q_len:3 * q_len] == 0).all()
    off = (out.double() - want).abs()
    assert (off <= tol + 1e-30).all(), float((off / (tol + 1e-30)).max())
    assert torch.equal(w[sums == 0], base[sums == 0])
    err = (w.double() - base.double() - sums).abs()
    assert (err <= (math.log(2) * 2.0 ** -18 * 600 + 2.0 ** -20) * sums + 2.0 ** -23 * (base + sums)).all()
