"""Outputs of the few-rows attention that are not 16-byte aligned: taken where every sequence is cut over several CTAs, whose merge stores 4 bytes at a time,
refused where a CTA stores whole rows."""
import pytest
import torch

import mm_rs_with_catlass_b200 as catcoc
from mm_rs_with_catlass_b200 import _native as N

AT = 1 << 20


def _decode(out, sk, window):
    """The C entry without a GPU: past its checks it ends with a driver error."""
    lib, tail = N.lib(), (1.0, AT, 0, None)
    if window:
        return lib.catcoc_window_attention(AT, AT, AT, out, AT, 1, 4, 1, 1, sk, 64, N.FMT_BF16, window, 4, *tail)
    return lib.catcoc_flash_decode(AT, AT, AT, out, AT, 1, 4, 1, 1, sk, 64, N.FMT_BF16, 1, *tail)


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up")
@pytest.mark.parametrize("window", [0, 9000])
def test_what_is_refused(window):
    for offset in (2, 4, 8, 12):
        assert _decode(AT + offset, 200, window) == N.E_ALIGNMENT               # two blocks: one CTA
    assert _decode(AT + 2, 16384, window) == N.E_ALIGNMENT
    for offset in (0, 4, 8, 12):
        assert _decode(AT + offset, 16384, window) not in (0, N.E_ALIGNMENT)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [None, 9000])
@pytest.mark.parametrize("d", [64, 128])
def test_cut_sequences_store_anywhere(d, window):
    g = torch.Generator(device="cuda").manual_seed(d)
    for b, hq, hk, sq, sk in ((1, 4, 1, 1, 16384), (2, 8, 2, 3, 16400)):
        q, k, v = (torch.randn(b, h, s, d, device="cuda", generator=g).bfloat16() for h, s in ((hq, sq), (hk, sk), (hk, sk)))
        args = dict(causal=True) if window is None else dict(causal=True, window=window, sinks=9)
        want = catcoc.flash_attention(q, k, v, **args)
        for offset in (2, 4, 6):                                                # elements
            room = torch.full((q.numel() + 16,), 7.0, dtype=q.dtype, device="cuda")
            out = room[offset:offset + q.numel()].view(q.shape)
            assert catcoc.flash_attention(q, k, v, out=out, **args) is out and torch.equal(out, want)
            assert (room[:offset] == 7).all() and (room[offset + q.numel():] == 7).all()
        with pytest.raises(RuntimeError):
            catcoc.flash_attention(q, k, v, out=room[1:1 + q.numel()].view(q.shape), **args)
        with pytest.raises(RuntimeError):                                        # a sequence of one CTA
            few = tuple(x[:, :, :min(x.shape[2], 200)].contiguous() for x in (q, k, v))
            catcoc.flash_attention(*few, out=room[2:2 + q.numel()].view(q.shape), **(args if window is None else dict(args, window=100)))
    torch.cuda.synchronize()
