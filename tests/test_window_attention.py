"""Attention with a sliding window and sinks against a plain computation in 64 bits, where the walk over key blocks can go wrong: windows
and sinks of one key, of whole blocks and one more or less, beyond all keys; positions that begin inside a block; tiles whose windows begin
in different blocks; query heads packed into tiles; keys cut into slices; the kernel for few rows; all types and head dimensions.

Tolerance: a probability is rounded to the operands' type (half a step, eps / 2 of itself; in fp16 at least 2^-25 of the largest) and is
off by e = 2 ln 2 2^-19 M + 2^-21 of itself for scores that are off by 2^-19 of M = scale log2(e) sum_c |q_c k_c|; the output is rounded once."""
import math

import pytest
import torch

import mm_rs_with_catlass_b200 as catcoc
from mm_rs_with_catlass_b200 import _native as N

BIG = 1 << 31


def _scratch(b, hq, hk, sq, sk, d, window, sinks):
    """(few-rows kernel?, scratch bytes)"""
    need = int(N.lib().catcoc_window_route(b, hq, hk, sq, sk, d, min(window, 1 << 30), min(sinks, 1 << 30)))
    return need >= 0, need if need >= 0 else -1 - need


def _visible(sq, sk, window, sinks, device="cpu"):
    p = torch.arange(sk - sq, sk, device=device)[:, None]
    j = torch.arange(sk, device=device)[None]
    return (j <= p) & ((p - j < window) | (j < sinks))


def _run(b, hq, hk, sq, sk, d, dtype, window, sinks, seed=0, gain=None, scale=None):
    from mm_rs_with_catlass_b200.ops._common import local_status, raise_on_status
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v = (torch.randn(b, h, s, d, device="cuda", generator=g).to(dtype) for h, s in ((hq, sq), (hk, sk), (hk, sk)))
    if gain is not None:
        k = (k.float() * torch.linspace(*gain, sk, device="cuda")[:, None]).to(dtype)
    out = catcoc.flash_attention(q, k, v, causal=True, window=window, sinks=sinks, scale=scale)
    torch.cuda.synchronize()
    raise_on_status(local_status(torch.device("cuda", 0)), "windowed attention")
    assert out.shape == q.shape and out.dtype == dtype
    seen = _visible(sq, sk, window, sinks, "cuda")
    sc, eps = d ** -0.5 if scale is None else scale, torch.finfo(dtype).eps
    for i in range(b):
        for h in range(hq):
            x, kk, vv = q[i, h].double(), k[i, h // (hq // hk)].double(), v[i, h // (hq // hk)].double()
            prob = torch.softmax((x @ kk.t() * sc).masked_fill(~seen, -math.inf), -1)
            want = prob @ vv
            big = ((x.abs() @ kk.abs().t()) * sc * 1.4427).masked_fill(~seen, 0).amax(-1, keepdim=True)
            e = 2 * math.log(2) * 2.0 ** -19 * big + 2.0 ** -21
            tol = (eps / 2 + 2 * e) * (prob @ vv.abs()) + eps / 2 * want.abs() + 1e-30
            if dtype == torch.float16:
                tol = tol + 2.0 ** -25 * (seen.double() @ vv.abs())
            off = (out[i, h].double() - want).abs()
            assert (off <= tol).all(), (i, h, float((off / tol).max()), (off / tol).amax(-1).argmax())
    return out


def test_refusals():
    from mm_rs_with_catlass_b200.ops import attention
    q = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16)
    real, attention.cm.require_cuda = attention.cm.require_cuda, lambda *t: torch.device("cpu")
    try:
        for args in (dict(window=4), dict(causal=True, window=0), dict(causal=True, window=-1), dict(causal=True, window=4, sinks=-1),
                     dict(causal=True, sinks=4), dict(sinks=1)):
            with pytest.raises(ValueError):
                catcoc.flash_attention(q, q, q, **args)
        with pytest.raises(ValueError):
            catcoc.flash_attention(q, q[:, :, :3], q[:, :, :3], causal=True, window=2)      # fewer keys than queries
    finally:
        attention.cm.require_cuda = real
    call = N.lib().catcoc_window_attention
    assert call(16, 16, 16, 16, None, 1, 1, 1, 4, 4, 64, N.FMT_BF16, 0, 0, 1.0, 16, 0, None) == N.E_BAD_ARG
    assert call(16, 16, 16, 16, None, 1, 1, 1, 4, 4, 64, N.FMT_BF16, 1, -1, 1.0, 16, 0, None) == N.E_BAD_ARG
    assert call(16, 16, 16, 16, None, 1, 1, 1, 400, 300, 64, N.FMT_BF16, 1, 0, 1.0, 16, 0, None) == N.E_BAD_ARG


def test_few_rows_want_an_aligned_output():
    """Few query rows: they are stored 16 bytes at a time."""
    at = 1 << 20
    call = N.lib().catcoc_window_attention
    assert call(at, at, at, at + 8, at, 1, 4, 1, 1, 300, 64, N.FMT_BF16, 64, 4, 1.0, at, 0, None) == N.E_ALIGNMENT


def test_scratch_goes_by_what_is_visible():
    assert _scratch(16, 32, 8, 1, 4096, 128, 64, 0) == (True, 0)                   # two blocks a sequence: whole runs
    assert _scratch(1, 8, 8, 512, 16384, 128, 4096, 64)[1] > 0                     # 34 blocks a tile, few tiles: slices
    assert _scratch(1, 8, 8, 512, 16384, 128, 512, 64) == (False, 0)
    assert _scratch(1, 8, 8, 300, 16384, 128, BIG, 0)[1] == int(N.lib().catcoc_flash_attention_workspace_bytes(1, 8, 8, 300, 16384, 128, 1))


def test_reference_window():
    from mm_rs_with_catlass_b200.ops.attention import attention_reference
    torch.manual_seed(0)
    q, k, v = (torch.randn(1, 2, s, 64) for s in (5, 9, 9))
    got = attention_reference(q, k, v, causal=True, window=3, sinks=2)
    seen = _visible(5, 9, 3, 2)
    want = torch.softmax((q @ k.transpose(-1, -2) / 8).masked_fill(~seen, -math.inf), -1) @ v
    assert torch.allclose(got, want, atol=1e-6) and seen.sum(1).tolist() == [5] * 5


WINDOWS = [(1, 0), (1, 1), (5, 4), (127, 0), (128, 128), (129, 1), (256, 130), (300, 300), (BIG, 0), (60, BIG)]


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("sq,sk", [(129, 129), (256, 256), (300, 300), (512, 700), (700, 1301), (1024, 1024)])
def test_windows_over_tiles(sq, sk, window, sinks):
    _run(1, 3, 3, sq, sk, 128, torch.bfloat16, window, sinks, seed=sq)
    _run(2, 2, 1, sq, sk, 64, torch.float16, window, sinks, seed=sq + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("sq,sk", [(1, 1), (1, 300), (3, 1000), (16, 16), (32, 2049)])
def test_few_rows(sq, sk, window, sinks):
    assert _scratch(2, 8, 2, sq, sk, 128, window, sinks)[0]
    _run(2, 8, 2, sq, sk, 128, torch.bfloat16, window, sinks, seed=sk)
    _run(1, 7, 7, sq, sk, 64, torch.float16, window, sinks, seed=sk + 1)
    _run(40, 8, 4, sq, sk, 64, torch.bfloat16, window, sinks, seed=sk + 2)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("case", [(1, 16, 2, 100, 2000), (2, 32, 4, 64, 700), (1, 8, 1, 300, 900), (16, 32, 4, 100, 1000), (2, 6, 2, 131, 131)])
@pytest.mark.parametrize("window,sinks", [(90, 0), (200, 17), (700, 129)])
def test_packed_heads(case, d, window, sinks):
    _run(*case, d, torch.bfloat16, window, sinks, seed=case[3])


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("case", [(1, 16, 4, 512, 8192, 4096, 64), (1, 8, 8, 170, 5000, 3000, 0), (1, 4, 1, 300, 9000, 2500, 700), (1, 1, 1, 2300, 2301, 2000, 1)])
def test_slices(case, d):
    few, scratch = _scratch(*case[:5], d, *case[5:])
    assert not few and scratch > 0
    for dtype in (torch.bfloat16, torch.float16):
        _run(*case[:5], d, dtype, *case[5:], seed=case[3])


@pytest.mark.gpu
@pytest.mark.parametrize("gain", [(0.2, 6.0), (6.0, 0.2)])
def test_moving_maxima(gain):
    for d in (64, 128):
        _run(1, 2, 2, 900, 1500, d, torch.bfloat16, 400, 30, seed=2, gain=gain)
        _run(2, 8, 2, 2, 1500, d, torch.float16, 400, 30, seed=3, gain=gain, scale=0.2)


@pytest.mark.gpu
def test_a_window_over_everything_is_causal_attention():
    for case in ((2, 8, 2, 700, 900), (2, 8, 2, 1, 900)):
        for d in (64, 128):
            g = torch.Generator(device="cuda").manual_seed(d)
            b, hq, hk, sq, sk = case
            q, k, v = (torch.randn(b, h, s, d, device="cuda", generator=g).bfloat16() for h, s in ((hq, sq), (hk, sk), (hk, sk)))
            want = catcoc.flash_attention(q, k, v, causal=True)
            for args in (dict(window=sk), dict(window=BIG, sinks=BIG), dict(window=1, sinks=sk)):
                assert torch.equal(catcoc.flash_attention(q, k, v, causal=True, **args), want)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_blocks_outside_of_the_windows_are_not_read(bad):
    """Keys and values that are no numbers in blocks which no row of a tile sees: the tile's rows keep their bits."""
    for sq, sk in ((2000, 2000), (1, 2000), (170, 5000)):
        for d in (64, 128):
            g = torch.Generator(device="cuda").manual_seed(d)
            q, k, v = (torch.randn(1, h, s, d, device="cuda", generator=g).bfloat16() for h, s in ((2, sq), (2, sk), (2, sk)))
            want = catcoc.flash_attention(q, k, v, causal=True, window=200, sinks=5)
            k[:, :, 128:1024] = bad
            v[:, :, 128:1024] = bad
            got = catcoc.flash_attention(q, k, v, causal=True, window=200, sinks=5)
            # a tile of 128 rows whose first position's window begins at 1024 or later
            clean = [t for t in range(0, sq, 128) if t + sk - sq - 199 >= 1024]
            assert clean and all(torch.equal(got[:, :, t:t + 128], want[:, :, t:t + 128]) for t in clean)


@pytest.mark.gpu
def test_strided_operands_streams_and_graphs():
    """Heads of a fused projection, an output of the caller's, two streams at once, a captured call on new contents."""
    g = torch.Generator(device="cuda").manual_seed(5)
    calls = []
    for sq in (600, 2, 300):
        qkv = torch.randn(2, sq + 700, 12, 64, device="cuda", generator=g).bfloat16()
        q, k, v = qkv[:, :sq, :8].transpose(1, 2), qkv[:, :, 8:10].transpose(1, 2), qkv[:, :, 10:].transpose(1, 2)
        if sq == 300:
            q, k, v = (torch.randn(1, h, s, 128, device="cuda", generator=g).bfloat16() for h, s in ((8, 300), (2, 6000), (2, 6000)))
        window = 3000 if sq == 300 else 250
        calls.append((q, lambda q=q, k=k, v=v, w=window: catcoc.flash_attention(q, k, v, causal=True, window=w, sinks=9)))
    assert _scratch(1, 8, 2, 300, 6000, 128, 3000, 9)[1] > 0
    want = [c().clone() for _, c in calls]
    out = torch.empty_like(want[0])
    q, k, v = (calls[0][1].__defaults__[i] for i in range(3))
    assert catcoc.flash_attention(q, k, v, causal=True, window=250, sinks=9, out=out) is out and torch.equal(out, want[0])
    streams, got = [torch.cuda.Stream() for _ in calls], [[] for _ in calls]
    torch.cuda.synchronize()
    for _ in range(8):
        for s, (_, c), o in zip(streams, calls, got):
            with torch.cuda.stream(s):
                o.append(c())
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for w, o in zip(want, got) for x in o)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = [c() for _, c in calls]
    for factor in (1.0, -0.5):
        for x, _ in calls:
            x.mul_(factor)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c()) for a, (_, c) in zip(kept, calls))
    del graph
