"""The 4-bit cache without a GPU: the goldens against the formulas, the layout of a block, and everything the functions refuse."""
import ctypes
import math

import pytest
import torch

import mm_rs_with_catlass_b200 as catcoc
from mm_rs_with_catlass_b200 import _native as N
from mm_rs_with_catlass_b200.ops import kv4


def test_a_block_and_the_library_agree():
    for d in (64, 128):
        assert N.lib().catcoc_kv4_block_bytes(d) == 72 * d == catcoc.kv4_cache(1, 1, d, device="cpu").shape[2]
    assert N.lib().catcoc_kv4_block_bytes(96) == -1
    with pytest.raises(ValueError):
        catcoc.kv4_cache(1, 1, 96, device="cpu")
    with pytest.raises(ValueError):
        catcoc.kv4_cache(0, 1, 64, device="cpu")


@pytest.mark.parametrize("d", [64, 128])
def test_words_of_a_row(d):
    """Word G w + g holds the channels 64 g + 8 w + n in its bits 4 n."""
    groups = d // 64
    x = torch.zeros(d)
    for g in range(groups):
        x[64 * g:64 * g + 64] = torch.arange(64) % 16          # codes 0..15: scale 1, zero 0
    codes, params = kv4.quantise_reference(x)
    words = codes.view(torch.int32)
    for w in range(8):
        for g in range(groups):
            for n in range(8):
                assert (int(words[groups * w + g]) >> (4 * n)) & 15 == int(x[64 * g + 8 * w + n])
    assert torch.equal(kv4.dequantise_reference(codes, params), x.double())
    assert params.view(torch.bfloat16).tolist() == [1.0, 0.0] * groups


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_values_are_half_a_step_away(dtype):
    torch.manual_seed(1)
    for gain, offset in ((1.0, 0.0), (1e-3, 0.0), (3.0, 10.0), (100.0, -50.0)):
        x = (torch.randn(50, 128) * gain + offset).to(dtype)
        codes, params = kv4.quantise_reference(x)
        y = kv4.dequantise_reference(codes, params)
        par = params.view(torch.bfloat16).double().view(50, 2, 2)
        s, z = (par[..., i].repeat_interleave(64, -1) for i in (0, 1))
        # half a step, and at the ends what the roundings of the zero (2^-8 of it, half a step of bf16) and of 15 scales cut off
        off = (y - x.double()).abs()
        assert (off <= 0.5001 * s + z.abs() * 2.0 ** -8 + 15 * s * 2.0 ** -8).all()


def test_odd_groups():
    x = torch.full((4, 64), 3.0)
    x[1, 5], x[2, 6], x[3] = math.nan, math.inf, 0.0
    codes, params = kv4.quantise_reference(x.bfloat16())
    y = kv4.dequantise_reference(codes, params)
    assert (y[0] == 3).all() and y[1].isnan().all() and y[2].isnan().all() and (y[3] == 0).all()
    # ranges from the smallest to past the largest number
    tiny = torch.tensor([2.0 ** -130, 0.0] * 32).bfloat16()
    huge = torch.tensor([3e38, -3e38] * 32).bfloat16()
    assert kv4.dequantise_reference(*kv4.quantise_reference(tiny)).abs().max() <= 2.0 ** -130
    assert kv4.dequantise_reference(*kv4.quantise_reference(huge)).isnan().all()


def _filled(d, lens, width, heads=2, seed=0):
    torch.manual_seed(seed)
    cache = torch.randint(0, 256, (len(lens) * width + 2, heads, 72 * d), dtype=torch.uint8)
    table = torch.randperm(len(lens) * width + 2)[:len(lens) * width].view(len(lens), width).int()
    n = sum(lens)
    k, v = torch.randn(n, heads, d).bfloat16(), torch.randn(n, heads, d).bfloat16()
    kv4.kv4_append_reference(cache, k, v, table, torch.tensor(lens, dtype=torch.int32), ends=torch.tensor(lens).cumsum(0).int())
    return cache, table, torch.tensor(lens, dtype=torch.int32), k, v


def test_goldens_of_attention_against_a_dense_computation():
    lens = [70, 3, 0]
    cache, table, kv_lens, _, _ = _filled(64, lens, 2)
    q = torch.randn(6, 4, 64)
    k, v = kv4.kv4_read_reference(cache, table, kv_lens)
    for window, sinks in ((None, 0), (5, 0), (5, 2), (1, 1), (100, 7)):
        out, sums = kv4.kv4_decode_reference(q, cache, table, kv_lens, q_len=2, window=window, sinks=sinks)
        assert torch.allclose(sums.sum(-1), torch.tensor([4.0, 4.0, 0.0], dtype=torch.float64)[:, None].expand(3, 2))
        for b, n in enumerate(lens):
            for t in range(2):
                for h in range(4):
                    p = n - 2 + t
                    seen = [j for j in range(n) if j <= p and (window is None or p - j < window or j < sinks)]
                    if not seen:
                        assert (out[2 * b + t, h] == 0).all()
                        continue
                    s = k[b, h // 2, seen] @ q[2 * b + t, h].double() / 8.0
                    assert torch.allclose(out[2 * b + t, h], torch.softmax(s, 0) @ v[b, h // 2, seen])


def test_golden_of_eviction():
    cache, table, kv_lens, _, _ = _filled(64, [130, 4], 3)
    k, v = kv4.kv4_read_reference(cache, table, kv_lens)
    w = torch.zeros(2, 2, 192)
    w[0, 0, [5, 50, 129]] = torch.tensor([3.0, 9.0, 1.0])
    kept, lens = kv4.kv4_evict_reference(cache, w, table, kv_lens, 6, recent=2, sinks=1)
    assert lens.tolist() == [6, 4]
    assert kept[0, 0].tolist() == [0, 1, 5, 50, 128, 129]              # two heavy ones, then the first of the weightless
    assert kept[0, 1].tolist() == [0, 1, 2, 3, 128, 129] and kept[1, 0].tolist() == [0, 1, 2, 3, -1, -1]
    k2, v2 = kv4.kv4_read_reference(cache, table, lens)
    for h in range(2):
        at = kept[0, h].long()
        assert torch.equal(k2[0, h, :6], k[0, h, at]) and torch.equal(v2[0, h, :6], v[0, h, at])
    assert w[0, 0, :8].tolist() == [0.0, 0.0, 3.0, 9.0, 0.0, 1.0, 0.0, 0.0] and w[0, 0, 6:].abs().max() == 0


def test_refusals(monkeypatch):
    """Arguments are checked before anything reaches a device: CPU tensors stand in for the GPU's."""
    monkeypatch.setattr(kv4.cm, "require_cuda", lambda *t: torch.device("cpu"))
    cache = catcoc.kv4_cache(4, 2, 64, device="cpu")
    table, lens = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    w = torch.zeros(2, 2, 128)
    refused = [
        (ValueError, lambda: catcoc.kv4_append(cache[:, :, :-1], x, x, table, lens)),
        (ValueError, lambda: catcoc.kv4_append(cache.float(), x, x, table, lens)),
        (ValueError, lambda: catcoc.kv4_append(cache[:, :1], x[:, :1], x[:, :1], table, lens)),      # a part of a cache
        (ValueError, lambda: catcoc.kv4_append(cache, x[:, :1], x[:, :1], table, lens)),             # heads
        (ValueError, lambda: catcoc.kv4_append(cache, x, x[:1], table, lens)),
        (TypeError, lambda: catcoc.kv4_append(cache, x.float(), x.float(), table, lens)),
        (TypeError, lambda: catcoc.kv4_append(cache, x, x.half(), table, lens)),
        (ValueError, lambda: catcoc.kv4_append(cache, x[:1], x[:1], table, lens)),                   # 1 token for 2 sequences
        (ValueError, lambda: catcoc.kv4_append(cache, x, x, table, lens, ends=lens.long())),
        (ValueError, lambda: catcoc.kv4_append(cache, x, x, table, lens, ends=lens[:1])),
        (TypeError, lambda: catcoc.kv4_append(cache, x, x, table.long(), lens)),
        (ValueError, lambda: catcoc.kv4_append(cache, x, x, table[:1], lens)),
        (ValueError, lambda: catcoc.kv4_append(cache, x, x, table[:, ::2], lens)),
        (ValueError, lambda: catcoc.kv4_append(cache, x, x, table[:, :0], lens)),
        (TypeError, lambda: catcoc.kv4_read(cache, table, lens, dtype=torch.float32)),
        (ValueError, lambda: catcoc.kv4_read(cache, table, lens, count=0)),
        (ValueError, lambda: catcoc.kv4_read(cache, table, lens, start=lens.long())),
        (ValueError, lambda: catcoc.kv4_decode(q[..., :32], cache, table, lens)),
        (TypeError, lambda: catcoc.kv4_decode(q.float(), cache, table, lens)),
        (ValueError, lambda: catcoc.kv4_decode(q[:, :3], cache, table, lens)),                       # 3 heads over 2
        (ValueError, lambda: catcoc.kv4_decode(q[:, :0], cache, table, lens)),
        (ValueError, lambda: catcoc.kv4_decode(q, cache, table, lens, q_len=2)),
        (ValueError, lambda: catcoc.kv4_decode(q, cache, table, lens, q_len=0)),
        (ValueError, lambda: catcoc.kv4_decode(q, cache, table, lens, window=0)),
        (ValueError, lambda: catcoc.kv4_decode(q, cache, table, lens, sinks=1)),
        (ValueError, lambda: catcoc.kv4_decode(q, cache, table, lens, window=4, sinks=-1)),
        (ValueError, lambda: catcoc.kv4_decode(q, cache, table, lens, scale=0.0)),
        (ValueError, lambda: catcoc.kv4_decode(q, cache, table, lens, out=q[:1])),
        (ValueError, lambda: catcoc.kv4_decode(q, cache, table, lens, weights=w[:, :, :127])),
        (ValueError, lambda: catcoc.kv4_decode(q, cache, table, lens, weights=w.double())),
        (ValueError, lambda: catcoc.kv4_evict(cache, w, table, lens, 0)),
        (ValueError, lambda: catcoc.kv4_evict(cache, w, table, lens, 4, recent=3, sinks=2)),
        (ValueError, lambda: catcoc.kv4_evict(cache, w, table, lens, 4, recent=-1)),
        (ValueError, lambda: catcoc.kv4_evict(cache, w[:1], table, lens, 4)),
        (ValueError, lambda: catcoc.kv4_evict(cache, w, table, lens, 100, out_table=table[:, :1].contiguous())),
        (ValueError, lambda: catcoc.kv4_evict(cache, w, table, lens, 4, out_table=table.long())),
        (ValueError, lambda: catcoc.kv4_evict(cache, w, table, lens, 4, out_weights=w[:, :, :3].contiguous())),
    ]
    for i, (error, call) in enumerate(refused):
        with pytest.raises(error):
            call()
            pytest.fail("call %d was not refused" % i)


def test_the_library_refuses_too():
    """The C entries check what they are given before any launch (no GPU here: a call that passed would fail otherwise)."""
    lib, one = N.lib(), 16

    def call(**changes):
        numbers = dict(B=2, Hk=1, D=64, pages=4, max_pages=2, fmt=N.FMT_BF16, T=2, count=1, keep=4, recent=2, sinks=2, out_pages=2, S=128, S_out=128,
                       Hq=4, q_len=1, window=0, scale=1.0, k_token=64, k_head=64, v_token=64, v_head=64)
        return N.Kv4Call(**{**numbers, **changes})

    def run(entry, pointers, null=None, odd=None, **changes):
        c = call(**changes)
        args = [None if i == null else 8 if i == odd else one for i in range(pointers)]
        tail = (0, None) if entry is lib.catcoc_kv4_decode else (None,)
        return entry(ctypes.addressof(c), *args, *tail)

    append, read, evict, decode = lib.catcoc_kv4_append, lib.catcoc_kv4_read, lib.catcoc_kv4_evict, lib.catcoc_kv4_decode

    def space(**changes):
        c = call(**changes)
        return lib.catcoc_kv4_decode_workspace_bytes(ctypes.addressof(c), 1)
    for entry, pointers in ((append, 7), (read, 7), (evict, 9), (decode, 8)):
        for bad in (dict(B=0), dict(Hk=0), dict(pages=0), dict(max_pages=0)):
            assert run(entry, pointers, **bad) == N.E_BAD_ARG
        assert run(entry, pointers, null=0) == N.E_BAD_ARG and run(entry, pointers, null=pointers - 1) == N.E_BAD_ARG
        assert entry(None, *[one] * pointers, *((0, None) if entry is decode else (None,))) == N.E_BAD_ARG
    assert run(append, 7, T=0) == N.E_BAD_ARG and run(append, 7, null=5, T=3) == N.E_BAD_ARG and run(append, 7, null=4) == N.E_BAD_ARG
    assert run(append, 7, D=96) == N.E_UNSUPPORTED and run(append, 7, fmt=N.FMT_F32) == N.E_UNSUPPORTED
    assert run(append, 7, k_token=65) == N.E_ALIGNMENT and run(append, 7, odd=2) == N.E_ALIGNMENT and run(append, 7, max_pages=1 << 27) == N.E_TOO_LARGE
    assert run(read, 7, count=0) == N.E_BAD_ARG and run(read, 7, D=65) == N.E_UNSUPPORTED and run(read, 7, odd=4) == N.E_ALIGNMENT
    assert run(read, 7, count=1 << 22) == N.E_TOO_LARGE
    assert run(evict, 9, sinks=3) == N.E_BAD_ARG and run(evict, 9, S=127) == N.E_BAD_ARG and run(evict, 9, keep=0) == N.E_BAD_ARG
    assert run(evict, 9, keep=100, out_pages=1) == N.E_BAD_ARG and run(evict, 9, keep=100, S_out=99) == N.E_BAD_ARG
    assert run(evict, 9, D=32) == N.E_UNSUPPORTED and run(evict, 9, odd=0) == N.E_ALIGNMENT
    for bad in (dict(Hq=3, Hk=2), dict(q_len=65), dict(q_len=0), dict(D=96), dict(B=65537), dict(q_len=64, Hq=128), dict(max_pages=1 << 19), dict(window=-1),
                dict(sinks=-1)):
        assert space(**bad) == -1 and run(decode, 8, **bad) == N.E_BAD_ARG
    assert run(decode, 8, scale=0.0) == N.E_UNSUPPORTED and run(decode, 8, scale=float("nan")) == N.E_UNSUPPORTED
    assert run(decode, 8, S=127) == N.E_BAD_ARG and run(decode, 8, odd=0) == N.E_ALIGNMENT and space() > 0
