"""A paged key / value cache in 4 bits and the attention over it (``csrc/kernels/kv4_cache.cu``, ``kv4_decode.cu``).

The cache is one uint8 tensor ``[pages, Hk, 72 * D]`` from :func:`kv4_cache`: a page holds 64 tokens, of every head a
block of 4-bit codes and of bf16 scales and zeros per 64 channels of a token (4.5 bits a value, 3.6 times less than 16).
As for :func:`mla_decode`, ``block_table`` ``[B, max_pages]`` (int32) names the pages of every sequence and ``kv_lens``
``[B]`` (int32) its length; both stay on the device. A serving step is

    kv4_append(cache, k, v, block_table, kv_lens)                  # the new tokens, kv_lens counts them already
    out = kv4_decode(q, cache, block_table, kv_lens, weights=sums) # ... attend; `sums` gathers what was attended to
    kept, kv_lens = kv4_evict(cache, sums, block_table, kv_lens, keep, recent=..., sinks=...)   # now and then

and :func:`kv4_read` gives tokens back in 16 bits. A page that is not in the cache is left out, and noted in the device's status
block (``ops._common.raise_on_status``), as a wait that ran out of time is. A length that the table's row cannot hold is noted too:
:func:`kv4_append` leaves out the tokens whose positions lie outside of the row, the other functions take as many tokens as the row holds
(none for a negative length).
Every value of a group that holds an infinity or a NaN reads as NaN; what pages hold behind a sequence's
length, or in front of its window, does not reach a result.

The reference keeps no such cache; its decode example over pages is 3rdparty/catlass/examples/19_mla/mla_kernel.cpp.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Tuple

import torch

from .. import _native as N
from . import _common as cm

PAGE = 64
GROUP = 64
_MOST = 0x7fffffff                    # the library's numbers have 32 bits
_FMT = {torch.float16: N.FMT_F16, torch.bfloat16: N.FMT_BF16}


def kv4_cache(pages: int, kv_heads: int, head_dim: int, device=None) -> torch.Tensor:
    """An empty cache of ``pages`` pages of 64 tokens: uint8 ``[pages, kv_heads, 72 * head_dim]``, ``head_dim`` 64 or 128."""
    if head_dim not in (64, 128):
        raise ValueError("head dimension %d: 64 and 128 are built" % head_dim)
    if pages < 1 or kv_heads < 1:
        raise ValueError("a cache has at least one page and one head")
    return torch.zeros((pages, kv_heads, 72 * head_dim), dtype=torch.uint8, device=device if device is not None else "cuda")


def _cache_dims(cache: torch.Tensor) -> Tuple[int, int, int]:
    """(pages, heads, head dimension) of a cache."""
    if cache.dim() != 3 or cache.dtype != torch.uint8 or cache.shape[2] not in (72 * 64, 72 * 128) or not cache.is_contiguous():
        raise ValueError("the cache must be a contiguous uint8 tensor [pages, heads, 72 * D] from kv4_cache(), D = 64 or 128")
    if not cache.shape[0] or not cache.shape[1]:
        raise ValueError("a cache has at least one page and one head")
    return cache.shape[0], cache.shape[1], cache.shape[2] // 72


def _sequences(block_table: torch.Tensor, kv_lens: torch.Tensor) -> Tuple[int, int]:
    """(sequences, pages in a row of the table)."""
    if block_table.dtype != torch.int32 or kv_lens.dtype != torch.int32 or block_table.dim() != 2 or kv_lens.dim() != 1:
        raise TypeError("block_table [B, max_pages] and kv_lens [B] must be int32")
    batch, width = block_table.shape
    if kv_lens.shape[0] != batch:
        raise ValueError("block_table and kv_lens must have one row per sequence (%d and %d)" % (batch, kv_lens.shape[0]))
    if not batch or not width:
        raise ValueError("block_table must name at least one page of at least one sequence")
    if not block_table.is_contiguous() or not kv_lens.is_contiguous():
        raise ValueError("block_table and kv_lens must be contiguous")
    return batch, width


def _device_ints(t: Optional[torch.Tensor], name: str, batch: int) -> None:
    if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != (batch,) or not t.is_contiguous()):
        raise ValueError("%s must be a contiguous int32 tensor [%d]" % (name, batch))


def _weights(weights: torch.Tensor, batch: int, heads: int, tokens: int, what: str = "weights") -> None:
    if weights.dtype != torch.float32 or weights.dim() != 3 or tuple(weights.shape[:2]) != (batch, heads) or not weights.is_contiguous():
        raise ValueError("%s must be a contiguous fp32 tensor [%d, %d, tokens]" % (what, batch, heads))
    if weights.shape[2] > _MOST:
        raise ValueError("%s: %d tokens a head are more than the kernels count" % (what, weights.shape[2]))
    if weights.shape[2] < tokens:
        raise ValueError("%s must have room for %d tokens, as the block table has (got %d)" % (what, tokens, weights.shape[2]))


# What a call has been found to be, by the layouts of its tensors and its numbers: checks are made and the numbers laid out once (a
# decode step of one short sequence 20 -> 13 us a call). Addresses are no part of it.
_plans: dict = {}


class _Plan:
    __slots__ = ("call", "at", "device", "status", "fresh", "copy")

    def __init__(self, device, copy=(), fresh=None, **numbers):
        self.call = N.Kv4Call(**numbers)
        self.at = C.addressof(self.call)
        self.device, self.status = device, cm.local_status(device).data_ptr()
        self.copy, self.fresh = copy, fresh        # which operands are copied first; what results or scratch are made like


def _keep(key, plan: _Plan) -> _Plan:
    if len(_plans) >= 1024:
        _plans.clear()
    _plans[key] = plan
    return plan


def _run(plan: _Plan, entry, *args) -> None:
    device = plan.device
    if cm.on_device(device):
        N.check(entry(plan.at, *args, cm.stream_of(device)))
    else:
        with torch.cuda.device(device):
            N.check(entry(plan.at, *args, cm.stream_of(device)))


def _dense(x: torch.Tensor, copy: bool) -> torch.Tensor:
    """``x``, or a copy of it where its rows do not begin at 16-byte boundaries (``copy``: by its strides)."""
    return x.clone(memory_format=torch.contiguous_format) if copy or x.data_ptr() & 15 else x


def _pitched(x: torch.Tensor) -> bool:
    """Whether the rows of ``x [T, H, D]`` begin at 16-byte boundaries when ``x`` does."""
    s = x.stride()
    return s[2] == 1 and s[0] % 8 == 0 and s[1] % 8 == 0


def kv4_append(cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, *,
               ends: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Writes new tokens into the cache (in place) and returns it.

    ``k`` and ``v`` are ``[T, Hk, D]`` (fp16 / bf16; parts of a fused projection's rows are read where they are). Without
    ``ends`` every sequence has ``T / B`` of them, one after the other; ``ends`` ``[B]`` (int32, on the device) gives the
    first token behind each sequence instead, and tokens from ``ends[-1]`` on are left out. ``kv_lens`` already counts the
    new tokens: the last one of sequence ``b`` goes to position ``kv_lens[b] - 1``.

    A group of 64 channels gets ``s = bf16((max - min) / 15)``, ``z = bf16(min)`` and the codes ``rint((x - z) / s)``, at most
    15, taken with ``1 / s`` in fp32; it stands for ``s * code + z``.
    """
    lay = cm.layout
    key = (0, lay(cache), lay(k), lay(v), lay(block_table), lay(kv_lens), lay(ends))
    plan = _plans.get(key)
    if plan is None:
        dev = cm.require_cuda(cache, k, v, block_table, kv_lens, ends)
        pages, heads, d = _cache_dims(cache)
        batch, width = _sequences(block_table, kv_lens)
        if k.dim() != 3 or k.shape != v.shape or k.shape[1] != heads or k.shape[2] != d:
            raise ValueError("k and v must be [T, %d, %d] for this cache, got %s and %s" % (heads, d, tuple(k.shape), tuple(v.shape)))
        if k.dtype not in _FMT or v.dtype != k.dtype:
            raise TypeError("kv4_append takes fp16 / bf16 keys and values of one dtype")
        if ends is None and k.shape[0] % batch:
            raise ValueError("%d tokens do not divide over %d sequences; give ends" % (k.shape[0], batch))
        _device_ints(ends, "ends", batch)
        copy = (not _pitched(k), not _pitched(v))
        rows = (heads * d, d)
        (kt, kh), (vt, vh) = (rows if c else x.stride()[:2] for x, c in ((k, copy[0]), (v, copy[1])))
        plan = _keep(key, _Plan(dev, copy, B=batch, Hk=heads, D=d, pages=pages, max_pages=width, fmt=_FMT[k.dtype], T=k.shape[0],
                                k_token=kt, k_head=kh, v_token=vt, v_head=vh))
    if not plan.call.T:
        return cache
    if plan.copy[0] or plan.copy[1] or (k.data_ptr() | v.data_ptr()) & 15:
        # (a base between two boundaries: the rows of the copy are dense, which is another call)
        return kv4_append(cache, _dense(k, plan.copy[0]), _dense(v, plan.copy[1]), block_table, kv_lens, ends=ends)
    _run(plan, N.lib().catcoc_kv4_append, cache.data_ptr(), k.data_ptr(), v.data_ptr(), block_table.data_ptr(), kv_lens.data_ptr(),
         ends.data_ptr() if ends is not None else None, plan.status)
    return cache


def kv4_read(cache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, *, start: Optional[torch.Tensor] = None,
             count: Optional[int] = None, dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(k, v)``, each ``[B, Hk, count, D]`` in fp16 / bf16: the values of the cache's tokens at the positions ``start[b]`` to
    ``start[b] + count - 1`` (``start`` ``[B]``, int32; from the beginning without it; ``count``: as many as the table's
    row can hold), zero where a sequence has no token."""
    lay = cm.layout
    count = None if count is None else cm.whole(count)
    key = (1, lay(cache), lay(block_table), lay(kv_lens), lay(start), count, dtype)
    plan = _plans.get(key)
    if plan is None:
        dev = cm.require_cuda(cache, block_table, kv_lens, start)
        pages, heads, d = _cache_dims(cache)
        batch, width = _sequences(block_table, kv_lens)
        if dtype not in _FMT:
            raise TypeError("kv4_read gives fp16 / bf16")
        _device_ints(start, "start", batch)
        n = width * PAGE if count is None else count
        if n < 1:
            raise ValueError("count must be positive")
        plan = _keep(key, _Plan(dev, fresh=cm.like((batch, heads, n, d), dtype, dev), B=batch, Hk=heads, D=d, pages=pages, max_pages=width,
                                fmt=_FMT[dtype], count=n))
    k, v = cm.fresh(plan.fresh), cm.fresh(plan.fresh)
    _run(plan, N.lib().catcoc_kv4_read, cache.data_ptr(), block_table.data_ptr(), kv_lens.data_ptr(), start.data_ptr() if start is not None else None,
         k.data_ptr(), v.data_ptr(), plan.status)
    return k, v


def kv4_decode(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, *, q_len: int = 1,
               window: Optional[int] = None, sinks: int = 0, weights: Optional[torch.Tensor] = None, scale: Optional[float] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the newest tokens over the cache.

    ``q`` is ``[T, Hq, D]`` (fp16 / bf16, ``Hq`` a multiple of the cache's heads): the last ``q_len`` (1 to 64) tokens of each
    of the ``B = T / q_len`` sequences, whose keys and values are in the cache already. Token ``t`` stands at position
    ``p = kv_lens[b] - q_len + t`` and sees the keys ``j <= p``, with a ``window`` those of them with ``p - j < window`` or
    ``j < sinks``. With ``weights`` (fp32 ``[B, Hk, S]``, ``S`` at least ``64 * max_pages``) the probabilities of all rows of a KV head
    are added to it, position by position: what :func:`kv4_evict` goes by. Returns ``[T, Hq, D]``; a token that sees nothing
    gives zeros.
    """
    lay = cm.layout
    q_len, sinks, window, scale = cm.whole(q_len), cm.whole(sinks), None if window is None else cm.whole(window), None if scale is None else float(scale)
    key = (2, lay(q), lay(cache), lay(block_table), lay(kv_lens), lay(weights), lay(out), q_len, window, sinks, scale)
    plan = _plans.get(key)
    if plan is None:
        plan = _keep(key, _decode_plan(q, cache, block_table, kv_lens, q_len, window, sinks, weights, scale, out))
    q = _dense(q, plan.copy)
    if out is None:
        out = torch.empty_like(q)
    # scratch of the caching allocator: calls on several streams never share one
    ws = cm.fresh(plan.fresh)
    _run(plan, N.lib().catcoc_kv4_decode, q.data_ptr(), cache.data_ptr(), block_table.data_ptr(), kv_lens.data_ptr(), out.data_ptr(),
         weights.data_ptr() if weights is not None else None, ws.data_ptr(), plan.status, cm.timeout_ns())
    return out


def _decode_plan(q, cache, block_table, kv_lens, q_len, window, sinks, weights, scale, out) -> _Plan:
    dev = cm.require_cuda(q, cache, block_table, kv_lens, weights, out)
    pages, heads, d = _cache_dims(cache)
    batch, width = _sequences(block_table, kv_lens)
    if q.dim() != 3 or q.shape[2] != d:
        raise ValueError("q must be [T, Hq, %d] for this cache, got %s" % (d, tuple(q.shape)))
    if q.dtype not in _FMT:
        raise TypeError("kv4_decode takes fp16 / bf16 queries")
    tokens, hq = q.shape[0], q.shape[1]
    if not 1 <= q_len <= 64 or tokens != batch * q_len:
        raise ValueError("q must hold q_len (1 to 64) tokens for each of the %d sequences, got %d for q_len=%d" % (batch, tokens, q_len))
    if not hq or hq % heads:
        raise ValueError("%d query heads do not divide over %d key / value heads" % (hq, heads))
    if window is None:
        if sinks:
            raise ValueError("sinks belong to a window")
        window = 0
    elif window < 1:
        raise ValueError("the window must be at least 1")
    if sinks < 0:
        raise ValueError("sinks must not be negative")
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if not scale > 0.0:
        raise ValueError("the softmax scale must be positive")
    if weights is not None:
        _weights(weights, batch, heads, width * PAGE)
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous()):
        raise ValueError("out must be a contiguous tensor shaped like q")
    plan = _Plan(dev, not q.is_contiguous(), B=batch, Hk=heads, D=d, pages=pages, max_pages=width, fmt=_FMT[q.dtype], Hq=hq, q_len=q_len,
                 window=min(window, 1 << 30), sinks=min(sinks, 1 << 30), scale=scale, S=weights.shape[2] if weights is not None else 0)
    with cm.guard(dev):
        need = int(N.lib().catcoc_kv4_decode_workspace_bytes(plan.at, int(weights is not None)))
    if need < 0:
        raise ValueError("kv4_decode: %d sequences of %d pages with %d rows a head are more than the kernel takes" % (batch, width, hq // heads * q_len))
    plan.fresh = cm.like((need,), torch.uint8, dev)
    return plan


def kv4_evict(cache: torch.Tensor, weights: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, keep: int, *, recent: int = 0,
              sinks: int = 0, out_table: Optional[torch.Tensor] = None,
              out_weights: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Cuts every sequence to ``keep`` tokens: its first ``sinks``, its last ``recent`` and, of the others, those with the largest
    ``weights`` (fp32 ``[B, Hk, S]`` from :func:`kv4_decode`; of equal ones the first, a NaN last), each KV head by its own.

    The kept tokens move to the positions 0, 1, ... in their order, in the sequence's own pages or, with ``out_table``
    ``[B, max_pages']``, to those (which must hold no token of these sequences), and their weights to the same positions of ``weights`` or
    ``out_weights`` ``[B, Hk, S']``, with zeros behind them. In place, no two sequences may share a page. Returns ``(kept, lens)``:
    int32 ``[B, Hk, keep]``, the positions that the tokens had (-1 behind the last), and the new lengths
    ``min(kv_lens, keep)`` as a new int32 tensor. ``block_table`` and ``kv_lens`` are not changed.
    """
    lay = cm.layout
    keep, recent, sinks = cm.whole(keep), cm.whole(recent), cm.whole(sinks)
    key = (3, lay(cache), lay(weights), lay(block_table), lay(kv_lens), lay(out_table), lay(out_weights), keep, recent, sinks)
    plan = _plans.get(key)
    if plan is None:
        dev = cm.require_cuda(cache, weights, block_table, kv_lens, out_table, out_weights)
        pages, heads, d = _cache_dims(cache)
        batch, width = _sequences(block_table, kv_lens)
        if keep > 1 << 30:
            raise ValueError("keep=%d is more than the kernels count (2^30)" % keep)
        if keep < 1 or recent < 0 or sinks < 0 or recent + sinks > keep:
            raise ValueError("keep=%d must be positive and hold the %d first and %d last tokens" % (keep, sinks, recent))
        _weights(weights, batch, heads, width * PAGE)
        most = min(keep, width * PAGE)
        if out_table is not None:
            if out_table.dtype != torch.int32 or out_table.dim() != 2 or out_table.shape[0] != batch or not out_table.is_contiguous():
                raise ValueError("out_table must be a contiguous int32 tensor [%d, max_pages]" % batch)
            if out_table.shape[1] * PAGE < most:
                raise ValueError("out_table must name pages for %d tokens" % most)
        if out_weights is not None:
            _weights(out_weights, batch, heads, most, "out_weights")
        plan = _keep(key, _Plan(dev, fresh=cm.like((batch, heads, keep), torch.int32, dev), B=batch, Hk=heads, D=d, pages=pages, max_pages=width,
                                S=weights.shape[2], keep=keep, recent=recent, sinks=sinks,
                                S_out=(weights if out_weights is None else out_weights).shape[2],
                                out_pages=(block_table if out_table is None else out_table).shape[1]))
    kept, lens = cm.fresh(plan.fresh), torch.empty_like(kv_lens)
    _run(plan, N.lib().catcoc_kv4_evict, cache.data_ptr(), weights.data_ptr(), (weights if out_weights is None else out_weights).data_ptr(),
         block_table.data_ptr(), (block_table if out_table is None else out_table).data_ptr(), kv_lens.data_ptr(), kept.data_ptr(), lens.data_ptr(),
         plan.status)
    return kept, lens


# ---------------------------------------------------------------------------------------
# The same functions in plain PyTorch, sequence by sequence (goldens for the tests, any device)
# ---------------------------------------------------------------------------------------

def _parts(cache: torch.Tensor):
    """Views ``[pages, heads, 64, bytes]`` of the cache: codes and parameters of K, codes and parameters of V."""
    d = cache.shape[2] // 72
    return [x.unflatten(2, (PAGE, -1)) for x in cache.split([32 * d, 4 * d, 32 * d, 4 * d], dim=2)]


def quantise_reference(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x [..., D]`` -> the bytes of its codes ``[..., D / 2]`` and of its scales and zeros ``[..., D / 16]``, step by step in fp32."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    s = ((hi - lo) * (1.0 / 15.0)).bfloat16()
    z = lo.bfloat16()
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    s = torch.where(torch.isfinite(g).all(-1) & torch.isfinite(s.float()), s, torch.full_like(s, math.nan))
    r = torch.where(s > 0, 1.0 / s.float(), torch.zeros_like(lo))
    codes = torch.nan_to_num(((g - z.float()[..., None]) * r[..., None]).round(), nan=0.0).clamp(0, 15).to(torch.uint8)
    # word 2 w + g (w with one group): channels 64 g + 8 w + n in bits 4 n
    n = codes.unflatten(-1, (8, 4, 2)).movedim(-4, -3)
    return (n[..., 0] | (n[..., 1] << 4)).flatten(-3), torch.stack((s, z), -1).flatten(-2).view(torch.uint8)


def dequantise_reference(codes: torch.Tensor, params: torch.Tensor, dtype: torch.dtype = torch.float64) -> torch.Tensor:
    """Bytes as :func:`quantise_reference` gives them -> values ``[..., D]``."""
    par = params.contiguous().view(torch.bfloat16).to(dtype).unflatten(-1, (-1, 2))
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).unflatten(-1, (8, -1, 8)).movedim(-3, -2).flatten(-2).to(dtype)
    return (c * par[..., :1] + par[..., 1:]).flatten(-2)


def kv4_append_reference(cache, k, v, block_table, kv_lens, *, ends=None):
    tokens, batch = k.shape[0], block_table.shape[0]
    last = [(b + 1) * (tokens // batch) for b in range(batch)] if ends is None else ends.tolist()
    parts, first = _parts(cache), 0
    for b, end in enumerate(last):
        for t in range(first, end):
            pos = int(kv_lens[b]) - (end - t)
            page = int(block_table[b, pos // PAGE])
            for x, at in ((k[t], 0), (v[t], 2)):
                codes, params = quantise_reference(x)
                parts[at][page, :, pos % PAGE], parts[at + 1][page, :, pos % PAGE] = codes, params
        first = end
    return cache


def kv4_read_reference(cache, block_table, kv_lens, *, start=None, count=None, dtype=torch.float64):
    heads, d = cache.shape[1], cache.shape[2] // 72
    count = block_table.shape[1] * PAGE if count is None else count
    out = [torch.zeros(block_table.shape[0], heads, count, d, dtype=dtype, device=cache.device) for _ in range(2)]
    parts = _parts(cache)
    for b in range(block_table.shape[0]):
        n, s = int(kv_lens[b]), 0 if start is None else int(start[b])
        lo, hi = max(s, 0), min(s + count, n)
        if hi <= lo:
            continue
        pages = block_table[b, :(hi + PAGE - 1) // PAGE].long()
        for i in (0, 1):
            codes, params = (p[pages].transpose(1, 2).flatten(0, 1)[lo:hi].transpose(0, 1) for p in parts[2 * i:2 * i + 2])
            out[i][b, :, lo - s:hi - s] = dequantise_reference(codes, params).to(dtype)
    return tuple(out)


def kv4_decode_reference(q, cache, block_table, kv_lens, *, q_len=1, window=None, sinks=0, weights=None, scale=None):
    """In fp64; returns ``(out, weights)`` with the probabilities added to a copy of ``weights`` (or to zeros)."""
    tokens, hq, d = q.shape
    heads, batch = cache.shape[1], tokens // q_len
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    room = block_table.shape[1] * PAGE
    sums = torch.zeros(batch, heads, room, dtype=torch.float64, device=q.device) if weights is None else weights.double()
    out = torch.zeros(tokens, hq, d, dtype=torch.float64, device=q.device)
    for b in range(batch):
        n = int(kv_lens[b])
        if n <= 0:
            continue
        k, v = (x[0, :, :n] for x in kv4_read_reference(cache, block_table[b:b + 1], kv_lens[b:b + 1]))
        j = torch.arange(n, device=q.device)
        for t in range(q_len):
            p = n - q_len + t
            seen = j <= p
            if window is not None:
                seen = seen & ((p - j < window) | (j < sinks))
            if not bool(seen.any()):
                continue
            x = q[b * q_len + t].double().view(heads, hq // heads, d)
            prob = torch.zeros(heads, hq // heads, n, dtype=torch.float64, device=q.device)
            prob[..., seen] = torch.softmax(torch.einsum("hgd,hnd->hgn", x, k[:, seen]) * scale, -1)
            out[b * q_len + t] = torch.einsum("hgn,hnd->hgd", prob[..., seen], v[:, seen]).reshape(hq, d)
            sums[b, :, :n] += prob.sum(1)
    return out, sums


def kv4_evict_reference(cache, weights, block_table, kv_lens, keep, *, recent=0, sinks=0, out_table=None, out_weights=None):
    batch, heads = block_table.shape[0], cache.shape[1]
    out_table = block_table if out_table is None else out_table
    target = weights if out_weights is None else out_weights
    parts = _parts(cache)
    kept = torch.full((batch, heads, keep), -1, dtype=torch.int32, device=cache.device)
    lens = kv_lens.clamp(max=keep).to(torch.int32)
    old_parts, old_weights = [p.clone() for p in parts], weights.clone()
    for b in range(batch):
        n = int(kv_lens[b])
        for h in range(heads):
            stay = list(range(n))
            if n > keep:
                rest = range(sinks, n - recent)
                w = old_weights[b, h].tolist()
                heavy = sorted(rest, key=lambda i: (w[i] != w[i], -w[i] if w[i] == w[i] else 0.0, i))[:keep - sinks - recent]
                stay = sorted(list(range(sinks)) + heavy + list(range(n - recent, n)))
            for i, s in enumerate(stay):
                kept[b, h, i] = s
                for p, old in zip(parts, old_parts):
                    p[int(out_table[b, i // PAGE]), h, i % PAGE] = old[int(block_table[b, s // PAGE]), h, s % PAGE]
            target[b, h, :len(stay)] = old_weights[b, h, stay]
            target[b, h, len(stay):] = 0.0
    return kept, lens
