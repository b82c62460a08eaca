"""The 4-bit cache on the GPU against its goldens in 64 bits: what the pages hold behind a sequence, pages in any order, lengths of
zero, one and around the ends of pages and tiles, ragged batches, windows and sinks, rows that see nothing, heads that share a KV
head, extreme ranges, arguments that only the device can see, streams and graphs.

Tolerances of the attention. The scores are sums of D products of whole codes in fp32, in four steps per group, plus the zeros'
part: off by at most 2^-19 of M = scale log2(e) sum_c |q_c| (s code + |z|) (the matrix unit drops what lies 2^-23 under its largest term,
16 terms and 8 steps, twice that for the fp32 steps around it), and exp2 is off by 2^-22: a probability is off by e = ln 2 (2^-19 M) + 2^-21 of
itself, their sum by as much. The probabilities times scales are rounded to 11 bits (half a step: 2^-12), or where they lie 2^-23
under the largest to 2^-38 of it, which n tokens can add up; they are the weights of code - 8. The fp32 sums of the codes and of the eights,
which are as large as 16 p s, are off by 2^-20 of that. The output is rounded once, by half a step of its type."""
import math

import pytest
import torch

import mm_rs_with_catlass_b200 as catcoc
from mm_rs_with_catlass_b200.ops import kv4
from mm_rs_with_catlass_b200.ops._common import StatusError, local_status, raise_on_status

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ok():
    torch.cuda.synchronize()
    raise_on_status(local_status(torch.device("cuda", 0)), "kv4")


def _make(lens, heads, d, seed=0, extra=0, gain=1.0, dtype=torch.bfloat16, width=None):
    """A cache in which the sequences' tokens lie on pages in any order, among pages of random bytes (scales and zeros that are no numbers
    among them), and the tokens."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    width = max(1, (max(lens) + 63) // 64) + extra if width is None else width
    pages = len(lens) * width + 3
    cache = torch.randint(0, 256, (pages, heads, 72 * d), dtype=torch.uint8, device=DEV, generator=g)
    table = torch.randperm(pages, device=DEV, generator=g)[:len(lens) * width].view(len(lens), width).int().contiguous()
    kv_lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
    n = sum(lens)
    k, v = ((torch.randn(n, heads, d, device=DEV, generator=g) * gain).to(dtype) for _ in range(2))
    ends = torch.tensor(lens, device=DEV).cumsum(0).int()
    return cache, table, kv_lens, k, v, ends, g


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [1, 3, 8])
def test_append_writes_what_the_golden_writes(d, dtype, heads):
    for lens in ([1], [64, 65, 0, 1, 200], [5] * 37):
        cache, table, kv_lens, k, v, ends, g = _make(lens, heads, d, seed=heads, dtype=dtype)
        want = kv4.kv4_append_reference(cache.clone(), k, v, table, kv_lens, ends=ends)
        # the same tokens as parts of a projection's rows, and rows that TMA-like loads cannot take
        fused = torch.cat((v, k, v), 1)
        odd = torch.empty(k.shape[0], heads, d + 3, dtype=dtype, device=DEV)
        odd[..., 1:d + 1] = k
        for kk, vv in ((k, v), (fused[:, heads:2 * heads], fused[:, 2 * heads:]), (odd[..., 1:d + 1], v)):
            got = cache.clone()
            assert catcoc.kv4_append(got, kk, vv, table, kv_lens, ends=ends) is got
            assert torch.equal(got, want)
    _ok()


def test_append_extreme_values():
    for dtype, values in ((torch.bfloat16, [0.0, 1.0, -1.0, 3e38, -3e38, 2.0 ** -130, 1e-20, math.inf, math.nan]),
                          (torch.float16, [0.0, 1.0, -1.0, 65504.0, -65504.0, 2.0 ** -24, math.inf, -math.inf, math.nan])):
        n = len(values) ** 2
        k = torch.zeros(n, 2, 128, dtype=dtype, device=DEV)
        for i, a in enumerate(values):
            for j, b in enumerate(values):
                k[i * len(values) + j, 0, ::3], k[i * len(values) + j, 1, 1::2] = a, b
        table, lens = torch.tensor([[1, 0]], dtype=torch.int32, device=DEV), torch.tensor([n], dtype=torch.int32, device=DEV)
        cache = catcoc.kv4_cache(2, 2, 128)
        want = kv4.kv4_append_reference(cache.clone(), k, -k, table, lens)
        got = catcoc.kv4_append(cache, k, -k, table, lens)
        for x, y in zip(kv4.kv4_read_reference(got, table, lens, count=n), kv4.kv4_read_reference(want, table, lens, count=n)):
            assert torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0)) and torch.equal(x.isnan(), y.isnan())
    _ok()


def test_append_leaves_the_rest_alone():
    """Tokens behind the last sequence are left out, and of a page only the new tokens' bytes change."""
    cache, table, kv_lens, k, v, ends, g = _make([70, 3, 129], 2, 128, seed=4)
    tail = torch.cat((k, k[:50])), torch.cat((v, v[:50]))
    want = kv4.kv4_append_reference(cache.clone(), k, v, table, kv_lens, ends=ends)
    assert torch.equal(catcoc.kv4_append(cache.clone(), *tail, table, kv_lens, ends=ends), want)
    # without ends: the last 2 of each
    want = kv4.kv4_append_reference(cache.clone(), k[:6], v[:6], table, kv_lens)
    assert torch.equal(catcoc.kv4_append(cache.clone(), k[:6], v[:6], table, kv_lens), want)
    assert torch.equal(catcoc.kv4_append(cache.clone(), k[:0], v[:0], table, kv_lens), cache)
    # a sequence without new tokens between two others, over more than 32 sequences
    many = torch.zeros(70, dtype=torch.int32, device=DEV)
    many[[0, 31, 32, 33, 69]] = torch.tensor([3, 1, 1, 2, 4], dtype=torch.int32, device=DEV)
    ends, lens = many.cumsum(0).int(), many + 60
    table = torch.arange(140, device=DEV).view(70, 2).int()
    cache = torch.randint(0, 256, (140, 2, 72 * 64), dtype=torch.uint8, device=DEV, generator=g)
    k, v = (torch.randn(11 + 40, 2, 64, device=DEV, generator=g).half() for _ in range(2))
    want = kv4.kv4_append_reference(cache.clone(), k[:11], v[:11], table, lens, ends=ends)
    assert torch.equal(catcoc.kv4_append(cache.clone(), k, v, table, lens, ends=ends), want)
    _ok()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_read(d, dtype):
    lens = [130, 0, 64, 1]
    cache, table, kv_lens, k, v, ends, _ = _make(lens, 3, d, seed=2, dtype=dtype)
    catcoc.kv4_append(cache, k, v, table, kv_lens, ends=ends)
    start = torch.tensor([100, 0, -3, 1], dtype=torch.int32, device=DEV)
    for s, count in ((None, None), (None, 1), (None, 500), (start, 7), (start, 33)):
        got = catcoc.kv4_read(cache, table, kv_lens, start=s, count=count, dtype=dtype)
        # s * code + z in fp32 (the product is exact), rounded once more
        want = kv4.kv4_read_reference(cache, table, kv_lens, start=s, count=count)
        for x, y in zip(got, want):
            assert x.shape == y.shape and x.dtype == dtype and torch.equal(x, y.float().to(dtype))
    _ok()


def _attend(q, cache, table, kv_lens, *, weights=None, q_len=1, window=None, sinks=0, scale=None):
    """A call against the golden, with the bounds from the top of this file. Returns the output."""
    base = None if weights is None else weights.clone()
    out = catcoc.kv4_decode(q, cache, table, kv_lens, q_len=q_len, window=window, sinks=sinks, weights=weights, scale=scale)
    _ok()
    assert out.shape == q.shape and out.dtype == q.dtype
    args = dict(q_len=q_len, window=window, sinks=sinks, scale=scale)
    want, sums = kv4.kv4_decode_reference(q, cache, table, kv_lens, weights=base, **args)
    d, heads = q.shape[2], cache.shape[1]
    group = q.shape[1] // heads
    # M and the sums of p s code and of p |v| need the parts of the values: caches with the zeros left out, and with all signs positive
    parts = kv4._parts(cache)
    eps = torch.finfo(q.dtype).eps
    for b in range(table.shape[0]):
        n = int(kv_lens[b])
        if not n:
            assert (out[b * q_len:(b + 1) * q_len] == 0).all()
            continue
        pages = table[b, :(n + 63) // 64].long()
        codes, params = [[parts[2 * i + j][pages].transpose(1, 2).flatten(0, 1)[:n] for i in (0, 1)] for j in (0, 1)]
        zeros = [p.clone().view(torch.bfloat16).unflatten(-1, (-1, 2)) for p in params]
        for z in zeros:
            z[..., 1] = 0
        scaled = [kv4.dequantise_reference(c, z.flatten(-2).view(torch.uint8)).transpose(0, 1) for c, z in zip(codes, zeros)]   # s code [heads, n, D]
        steps = [p.contiguous().view(torch.bfloat16).double().unflatten(-1, (-1, 2))[..., 0].repeat_interleave(64, -1).transpose(0, 1) for p in params]
        offs = [p.contiguous().view(torch.bfloat16).double().unflatten(-1, (-1, 2))[..., 1].abs().repeat_interleave(64, -1).transpose(0, 1) for p in params]
        k_all, v_all = kv4.kv4_read_reference(cache, table[b:b + 1], kv_lens[b:b + 1])
        k_all, v_all = k_all[0, :, :n], v_all[0, :, :n]
        j = torch.arange(n, device=DEV)
        for t in range(q_len):
            p = n - q_len + t
            seen = j <= p if window is None else (j <= p) & ((p - j < window) | (j < sinks))
            row = slice(b * q_len + t, b * q_len + t + 1)
            if not bool(seen.any()):
                assert (out[row] == 0).all()
                continue
            x = q[b * q_len + t].double().view(heads, group, d)
            sc = 1 / math.sqrt(d) if scale is None else scale
            big = (torch.einsum("hgd,hnd->hgn", x.abs(), scaled[0][:, seen] + offs[0][:, seen]) * sc * 1.4427).amax(-1)       # [heads, group]
            prob = torch.softmax(torch.einsum("hgd,hnd->hgn", x, k_all[:, seen]) * sc, -1)
            e = 2 * (math.log(2) * big * 2.0 ** -19 + 2.0 ** -21)                                                                 # [heads, group]
            unit = steps[1][:, seen]                                                                                              # s
            centred = torch.einsum("hgn,hnd->hgd", prob, (scaled[1][:, seen] - 8 * unit).abs())
            abs_v = torch.einsum("hgn,hnd->hgd", prob, scaled[1][:, seen] + offs[1][:, seen]) + 16 * torch.einsum("hgn,hnd->hgd", prob, unit)
            floor = 2.0 ** -38 * 15 * int(seen.sum()) * scaled[1][:, seen].amax(1)[:, None]
            tol = (2.0 ** -12 * centred + (e[..., None] + 2.0 ** -20) * abs_v + floor).view(heads * group, d) + eps / 2 * want[b * q_len + t].abs() + 1e-30
            off = (out[b * q_len + t].double() - want[b * q_len + t]).abs()
            assert (off <= tol).all(), (b, t, float((off / tol).max()))
    if weights is not None:
        err = (weights.double() - sums).abs()
        lim = (math.log(2) * 2.0 ** -18 * 600 + 2.0 ** -20) * (sums - base.double()) + 2.0 ** -23 * sums.abs() + 1e-30   # M below 600 where weights are tested
        assert (err <= lim).all(), float((err / lim).max())
    return out


LENS = [[1], [2, 15, 16, 17], [63, 64, 65], [0, 300, 1, 0], [129, 700, 5, 1000]]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", LENS)
def test_lengths(d, lens):
    for dtype, heads, group in ((torch.bfloat16, 2, 4), (torch.float16, 1, 7)):
        cache, table, kv_lens, k, v, ends, g = _make(lens, heads, d, seed=len(lens), dtype=dtype, extra=1)
        catcoc.kv4_append(cache, k, v, table, kv_lens, ends=ends)
        q = torch.randn(len(lens), heads * group, d, device=DEV, generator=g).to(dtype)
        _attend(q, cache, table, kv_lens)


@pytest.mark.parametrize("group,q_len", [(1, 1), (8, 1), (9, 1), (16, 1), (3, 3), (5, 4), (17, 2), (1, 64), (2, 20)])
def test_rows(group, q_len):
    for d in (64, 128):
        cache, table, kv_lens, k, v, ends, g = _make([200, 33, 90], 2, d, seed=group)
        catcoc.kv4_append(cache, k, v, table, kv_lens, ends=ends)
        q = torch.randn(3 * q_len, 2 * group, d, device=DEV, generator=g).bfloat16()
        w = torch.rand(3, 2, table.shape[1] * 64, device=DEV, generator=g)
        _attend(q, cache, table, kv_lens, q_len=q_len, weights=w)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (64, 64), (100, 3), (129, 70), (1000, 5), (1 << 31, 1 << 31), (50, 10000)])
def test_windows(window, sinks):
    for d, q_len in ((128, 1), (64, 3), (128, 20)):
        lens = [700, 64, 1, 128, 333]
        cache, table, kv_lens, k, v, ends, g = _make(lens, 2, d, seed=window % 97, extra=2)
        catcoc.kv4_append(cache, k, v, table, kv_lens, ends=ends)
        q = torch.randn(len(lens) * q_len, 8, d, device=DEV, generator=g).bfloat16()
        w = torch.zeros(len(lens), 2, table.shape[1] * 64 + 5, device=DEV)
        _attend(q, cache, table, kv_lens, q_len=q_len, window=window, sinks=sinks, weights=w)


def test_long_and_many():
    """Runs that end inside a unit and runs of many units; sequences that fill whole runs."""
    for lens, heads, group in (([20011], 1, 4), ([9000, 9000], 8, 2), ([100] * 130, 4, 4), ([5000] + [3] * 60, 2, 16)):
        cache, table, kv_lens, k, v, ends, g = _make(lens, heads, 128, seed=1)
        catcoc.kv4_append(cache, k, v, table, kv_lens, ends=ends)
        q = torch.randn(len(lens), heads * group, 128, device=DEV, generator=g).bfloat16()
        _attend(q, cache, table, kv_lens, weights=torch.zeros(len(lens), heads, table.shape[1] * 64, device=DEV))


@pytest.mark.parametrize("d", [64, 128])
def test_ranges(d):
    """Scores and scales over wide ranges: the references of the maxima and of the scales move, forwards and backwards."""
    lens = [500, 300]
    for dtype in (torch.bfloat16, torch.float16):
        for ramp_k, ramp_v, gain_q in ((0.0, 0.0, 1.0), (2.0, 9.0, 1.0), (-2.0, -9.0, 1.0), (0.0, -20.0, 1.0), (0.0, 12.0, 1e-3), (-1.0, 0.0, 30.0)):
            if dtype == torch.float16 and abs(ramp_v) > 12:
                continue
            cache, table, kv_lens, k, v, ends, g = _make(lens, 2, d, seed=3, dtype=torch.float32)
            at = torch.cat([torch.linspace(0, 1, n, device=DEV) for n in lens])[:, None, None]
            k, v = (k * torch.exp2(at * ramp_k)).to(dtype), (v * torch.exp2(at * ramp_v)).to(dtype)
            catcoc.kv4_append(cache, k, v, table, kv_lens, ends=ends)
            q = (torch.randn(2, 6, d, device=DEV, generator=g) * gain_q).to(dtype)
            _attend(q, cache, table, kv_lens)
    if d == 128:    # values over nearly all of bf16's range, and queries at its ends
        cache, table, kv_lens, k, v, ends, g = _make([200], 1, d, seed=5)
        v = (v.float() * torch.exp2(torch.linspace(-100, 100, 200, device=DEV))[:, None, None]).bfloat16()
        catcoc.kv4_append(cache, k * 2.0 ** -60, v, table, kv_lens, ends=ends)
        _attend((torch.randn(1, 4, d, device=DEV, generator=g) * 2.0 ** 60).bfloat16(), cache, table, kv_lens)
        catcoc.kv4_append(cache, k, v, table, kv_lens, ends=ends)
        _attend((torch.randn(1, 4, d, device=DEV, generator=g) * 2.0 ** -125).bfloat16(), cache, table, kv_lens)
        _attend(torch.zeros(1, 4, d, device=DEV).bfloat16(), cache, table, kv_lens)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_is_not_seen_does_not_count(bad):
    """Tokens that are no numbers outside of a row's window change no bit of it; inside they show."""
    n, d = 400, 128
    cache, table, kv_lens, k, v, ends, g = _make([n], 2, d, seed=8)
    catcoc.kv4_append(cache, k, v, table, kv_lens, ends=ends)
    q = torch.randn(3, 8, d, device=DEV, generator=g).bfloat16()
    args = dict(q_len=3, window=100, sinks=5)
    w0, w1 = (torch.zeros(1, 2, table.shape[1] * 64, device=DEV) for _ in range(2))
    want = catcoc.kv4_decode(q, cache, table, kv_lens, weights=w0, **args)
    hidden = list(range(5, n - 102))
    for x in (k, v):
        x[hidden, :, 3] = bad
    catcoc.kv4_append(cache, k, v, table, kv_lens, ends=ends)
    got = catcoc.kv4_decode(q, cache, table, kv_lens, weights=w1, **args)
    assert torch.equal(got, want) and torch.equal(w0, w1)
    # the newest token: the last row alone sees it; with V only, in the group of 64 channels alone
    v[n - 1, 0, 70] = bad
    catcoc.kv4_append(cache, k, v, table, kv_lens, ends=ends)
    got = catcoc.kv4_decode(q, cache, table, kv_lens, **args)
    assert torch.equal(got[:2], want[:2]) and torch.equal(got[2, 4:], want[2, 4:])
    assert got[2, :4, 64:].isnan().all() and got[2, :4, :64].isfinite().all()
    assert (got[2, :4, :64].float() - want[2, :4, :64].float()).abs().max() <= 2.0 ** -8 * want[2, :4, :64].float().abs().max()
    k[n - 1, 1, 0] = bad
    catcoc.kv4_append(cache, k, v, table, kv_lens, ends=ends)
    got = catcoc.kv4_decode(q, cache, table, kv_lens, **args)
    assert torch.equal(got[:2], want[:2]) and got[2, 4:].isnan().all()
    q[1, 0, 0] = math.nan
    assert catcoc.kv4_decode(q, cache, table, kv_lens, **args)[1, 0].isnan().all()
    _ok()


def test_arguments_in_memory():
    """Buffers of the caller: strided and unaligned queries, out, scale; results do not depend on the page order."""
    cache, table, kv_lens, k, v, ends, g = _make([300, 77], 2, 64, seed=6)
    catcoc.kv4_append(cache, k, v, table, kv_lens, ends=ends)
    rows = torch.randn(2, 10, 64, device=DEV, generator=g).bfloat16()
    q = rows[:, 1:9]
    want = _attend(q.contiguous(), cache, table, kv_lens, scale=0.3)
    out = torch.empty(2, 8, 64, dtype=torch.bfloat16, device=DEV)
    assert catcoc.kv4_decode(q, cache, table, kv_lens, scale=0.3, out=out) is out and torch.equal(out, want)
    flat = torch.empty(2 * 8 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:]
    flat.copy_(q.reshape(-1))
    assert torch.equal(catcoc.kv4_decode(flat.view(2, 8, 64), cache, table, kv_lens, scale=0.3), want)
    order = torch.randperm(cache.shape[0], device=DEV, generator=g)
    moved = torch.empty_like(cache)
    moved[order] = cache
    assert torch.equal(catcoc.kv4_decode(q, moved, order[table.long()].int(), kv_lens, scale=0.3), want)


def test_bad_pages_and_lengths_are_noted():
    """Names and lengths that the host cannot see: the access is left out, the other sequences' results stand, the status tells."""
    cache, table, kv_lens, k, v, ends, g = _make([300, 77], 2, 64, seed=6)
    catcoc.kv4_append(cache, k, v, table, kv_lens, ends=ends)
    q = torch.randn(2, 8, 64, device=DEV, generator=g).bfloat16()
    want = catcoc.kv4_decode(q, cache, table, kv_lens)
    w = torch.rand(2, 2, table.shape[1] * 64, device=DEV, generator=g)
    before = cache.clone()

    def noted(call):
        result = call()
        torch.cuda.synchronize()
        with pytest.raises(StatusError):
            raise_on_status(local_status(torch.device("cuda", 0)), "kv4")
        return result
    for name in (-1, cache.shape[0], 0x7fffffff, -0x80000000):
        bad = table.clone()
        bad[0, 1] = name
        assert torch.equal(noted(lambda: catcoc.kv4_decode(q, cache, bad, kv_lens))[1], want[1])
        x, y = noted(lambda: catcoc.kv4_read(cache, bad, kv_lens)), catcoc.kv4_read(cache, table, kv_lens)
        assert all(torch.equal(a[1], b[1]) and torch.equal(a[0, :, :64], b[0, :, :64]) and (a[0, :, 64:128] == 0).all() for a, b in zip(x, y))
        noted(lambda: catcoc.kv4_append(cache, k, v, bad, kv_lens, ends=ends))
        assert torch.equal(cache, before)                                 # the others' tokens again
        noted(lambda: catcoc.kv4_evict(cache.clone(), w.clone(), bad, kv_lens, 290))
    for n in (-5, table.shape[1] * 64 + 1, 0x7fffffff):
        lens = kv_lens.clone()
        lens[0] = n
        assert torch.equal(noted(lambda: catcoc.kv4_decode(q, cache, table, lens))[1], want[1])
        noted(lambda: catcoc.kv4_read(cache, table, lens, count=3))
        noted(lambda: catcoc.kv4_evict(cache.clone(), w.clone(), table, lens, 50))
    lens = kv_lens.clone()
    lens[1] = 3                                                         # 77 new tokens of a sequence of three
    noted(lambda: catcoc.kv4_append(cache, k, v, table, lens, ends=ends))
    _ok()


EVICT = [([300], 100, 20, 4), ([300, 64, 100, 101, 0, 1], 100, 20, 4), ([1500, 1025, 700], 513, 0, 0), ([200, 90], 80, 80, 0), ([200], 70, 60, 10),
         ([200, 65], 1, 0, 0), ([200, 65], 1, 1, 0), ([200], 199, 5, 5), ([3000], 2900, 10, 1), ([100, 50], 300, 3, 3)]


def _evict_weights(g, batch, heads, room):
    w = torch.randn(batch, heads, room, device=DEV, generator=g).exp_()
    w[torch.rand(w.shape, device=DEV, generator=g) < 0.3] = 0.0
    w[torch.rand(w.shape, device=DEV, generator=g) < 0.2] = 0.5           # many equal ones
    return w


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,keep,recent,sinks", EVICT)
def test_evict(lens, keep, recent, sinks, d):
    for heads in (1, 3):
        cache, table, kv_lens, k, v, ends, g = _make(lens, heads, d, seed=keep)
        catcoc.kv4_append(cache, k, v, table, kv_lens, ends=ends)
        w = _evict_weights(g, len(lens), heads, table.shape[1] * 64)
        w[:, :, 7 % min(len(w[0, 0]), 7 + 1)] = -1.0                      # whole order of the numbers
        w[0, 0, 40], w[0, 0, 41], w[0, 0, 42] = math.inf, -0.0, math.nan
        want_cache, want_w = cache.clone(), w.clone()
        want = kv4.kv4_evict_reference(want_cache, want_w, table, kv_lens, keep, recent=recent, sinks=sinks)
        # in place: nothing but the first positions changes
        got_cache, got_w = cache.clone(), w.clone()
        got = catcoc.kv4_evict(got_cache, got_w, table, kv_lens, keep, recent=recent, sinks=sinks)
        _ok()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(got_cache, want_cache) and torch.equal(got_w.nan_to_num(-7.0), want_w.nan_to_num(-7.0))
        # into other pages, behind the old ones
        width = (keep + 63) // 64
        more = torch.cat((cache, torch.randint(0, 256, (len(lens) * width, *cache.shape[1:]), dtype=torch.uint8, device=DEV, generator=g)))
        new_table = (cache.shape[0] + torch.randperm(len(lens) * width, device=DEV, generator=g)).view(len(lens), width).int()
        new_w = torch.full((len(lens), heads, width * 64 + 3), 9.0, device=DEV)
        ref_cache, ref_w = more.clone(), new_w.clone()
        want = kv4.kv4_evict_reference(ref_cache, w, table, kv_lens, keep, recent=recent, sinks=sinks, out_table=new_table, out_weights=ref_w)
        got = catcoc.kv4_evict(more, w, table, kv_lens, keep, recent=recent, sinks=sinks, out_table=new_table, out_weights=new_w)
        _ok()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(more, ref_cache) and torch.equal(new_w.nan_to_num(-7.0), ref_w.nan_to_num(-7.0))


def _serve(seed, steps=40, keep=96):
    """A short serving loop: a prompt, then steps that append, attend with a window's worth of sums, and evict when there is no room."""
    lens = [150, 70, 1]
    cache, table, kv_lens, k, v, ends, g = _make(lens, 2, 128, seed=seed, width=4)
    return cache, table, kv_lens, k, v, ends, g, keep, steps


def test_a_serving_loop():
    """Prompt, steps, evictions: the whole run against the goldens run side by side on a second cache."""
    cache, table, kv_lens, k, v, ends, g, keep, steps = _serve(11)
    other = cache.clone()
    w = torch.zeros(3, 2, 256, device=DEV)
    catcoc.kv4_append(cache, k, v, table, kv_lens, ends=ends)
    kv4.kv4_append_reference(other, k, v, table, kv_lens, ends=ends)
    assert torch.equal(cache, other)
    evictions = 0
    for step in range(steps):
        kv_lens = kv_lens + 1
        k, v = (torch.randn(3, 2, 128, device=DEV, generator=g).bfloat16() for _ in range(2))
        catcoc.kv4_append(cache, k, v, table, kv_lens)
        kv4.kv4_append_reference(other, k, v, table, kv_lens)
        assert torch.equal(cache, other)
        q = torch.randn(3, 8, 128, device=DEV, generator=g).bfloat16()
        _attend(q, cache, table, kv_lens, weights=w)
        if step % 13 == 12:
            golden_w = w.clone()
            want, want_lens = kv4.kv4_evict_reference(other, golden_w, table, kv_lens, keep, recent=16, sinks=4)
            kept, kv_lens = catcoc.kv4_evict(cache, w, table, kv_lens, keep, recent=16, sinks=4)
            assert torch.equal(kept, want) and torch.equal(kv_lens, want_lens) and torch.equal(cache, other) and torch.equal(w, golden_w)
            evictions += 1
    assert evictions == 3
    # the first sequences are full: a dense continuation over what was kept
    x, y = catcoc.kv4_read(cache, table, kv_lens, count=keep)
    assert x.shape == (3, 2, keep, 128) and x.isfinite().all() and y.isfinite().all()
    q = torch.randn(1, 8, 5, 128, device=DEV, generator=g).bfloat16()
    assert catcoc.flash_attention(q, x[:1], y[:1]).isfinite().all()


def _calls(seed):
    lens = [500, 64, 1200, 3]
    cache, table, kv_lens, k, v, ends, g = _make(lens, 4, 128, seed=seed)
    q = torch.randn(4, 16, 128, device=DEV, generator=g).bfloat16()
    w = torch.rand(4, 4, table.shape[1] * 64, device=DEV, generator=g)
    work = cache.clone()

    def step():
        ww = w.clone()
        catcoc.kv4_append(work, k, v, table, kv_lens, ends=ends)
        out = catcoc.kv4_decode(q, work, table, kv_lens, weights=ww)
        kept, n = catcoc.kv4_evict(work, ww, table, kv_lens, 300, recent=50, sinks=4)
        return out, ww, kept, n, *catcoc.kv4_read(work, table, n, count=300)
    return [q, k, v], step


def test_two_streams():
    calls = [_calls(seed)[1] for seed in (1, 2)]
    want = [[x.clone() for x in c()] for c in calls]
    _ok()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[], []]
    for _ in range(12):
        for s, c, out in zip(streams, calls, got):
            with torch.cuda.stream(s):
                out.append(c())
    _ok()
    for x, out in zip(want, got):
        assert all(torch.equal(a, b) for y in out for a, b in zip(x, y))


def test_captured_calls_replay_on_new_contents():
    inputs, call = _calls(3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = call()
        second = call()
    for scale in (1.0, 0.5, -2.0):
        for x in inputs:
            x.mul_(scale)
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        a, b = [x.clone() for x in first], [x.clone() for x in second]
        want = call()
        assert all(torch.equal(x, z) and torch.equal(y, z) for x, y, z in zip(a, b, want))
    _ok()
    del graph
