"""The operators of long-context serving as cases that can be timed and compared: attention with a sliding window and visible first
tokens (sinks), a paged key / value cache held in 4 bits (append, read, attention over it), and eviction from that cache by
accumulated attention weight.

``run`` computes them in plain torch operations, in 32 bits, or, where ``own`` is true, calls the library. Kinds of case:

``window``  causal attention with a window and sinks over dense keys and values (prefill, a chunk over a cache, a decode step)
``fill``    new tokens are quantised into the cache, and the values that the cache now holds for them are read back
``decode``  one decode step over the 4-bit cache, with or without a window and accumulated weights
``evict``   the cache is cut to its heaviest, first and last tokens, into new pages, and read back

The 4-bit cache. ``cache`` is uint8 ``[pages, heads, 72 * D]``: 64 tokens of one head. A group of 64 channels of a token has codes
``c`` of 4 bits and a bf16 scale ``s`` and zero ``z`` and stands for ``s * c + z``. A block holds the codes of K (64 rows of D / 2
bytes), the (s, z) pairs of K (64 rows of D / 64 pairs), then the same of V. A row's 32-bit word ``2 w + g`` (``w`` at D = 64) holds
the channels ``64 g + 8 w + n``, n = 0..7, in its bits ``4 n .. 4 n + 3``.
"""
import math

import torch

own = False
DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
PAGE, GROUP = 64, 64


def listed():
    return [
        # prompt of a long chat through a layer with a window: the repository's prefill benchmark, one sequence of it
        dict(name="window_prefill", kind="window", b=1, hq=32, hk=8, sq=8192, sk=8192, d=128, window=1024, sinks=4, dtype="bf16"),
        # ragged prompts behind a cached prefix, small heads
        dict(name="window_ragged", kind="window", b=3, hq=12, hk=4, sq=1003, sk=2777, d=64, window=300, sinks=17, dtype="fp16"),
        # a chunk of a long prompt over what is already there
        dict(name="window_chunk", kind="window", b=1, hq=16, hk=4, sq=512, sk=16384, d=128, window=4096, sinks=64, dtype="bf16"),
        # the decode benchmark with a window: one token each
        dict(name="window_step", kind="window", b=16, hq=32, hk=8, sq=1, sk=4096, d=128, window=1024, sinks=4, dtype="bf16"),
        # two prompts enter the cache
        dict(name="fill_prompt", kind="fill", b=2, hq=32, hk=8, s=8192, new=8192, ragged=True, d=128, dtype="bf16"),
        # one token each of a decode batch enters it: latency
        dict(name="fill_step", kind="fill", b=32, hq=16, hk=4, s=700, new=1, ragged=True, d=64, dtype="fp16"),
        # the decode benchmark over 4 bits
        dict(name="decode_batch", kind="decode", b=16, hq=32, hk=8, s=4096, q_len=1, ragged=False, d=128, window=0, sinks=0, weights=False, dtype="bf16"),
        # a small call: one short sequence
        dict(name="decode_small", kind="decode", b=1, hq=8, hk=2, s=501, q_len=1, ragged=False, d=64, window=0, sinks=0, weights=False, dtype="fp16"),
        # one very long sequence, two tokens at once
        dict(name="decode_long", kind="decode", b=1, hq=32, hk=8, s=131072, q_len=2, ragged=False, d=128, window=0, sinks=0, weights=False, dtype="bf16"),
        # a ragged batch that notes what its tokens attend to
        dict(name="decode_weights", kind="decode", b=12, hq=24, hk=8, s=6001, q_len=1, ragged=True, d=128, window=0, sinks=0, weights=True, dtype="bf16"),
        # a batch is cut to half of its tokens
        dict(name="evict_batch", kind="evict", b=16, hk=8, s=4096, keep=2048, recent=256, sinks=4, ragged=True, d=128, dtype="bf16"),
        # one short sequence is cut
        dict(name="evict_small", kind="evict", b=1, hk=4, s=1111, keep=500, recent=64, sinks=1, ragged=False, d=64, dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["window", "window", "fill", "decode", "decode", "evict"])
    d, dtype = rng.choice([64, 128]), rng.choice(["bf16", "bf16", "fp16"])
    hk, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8, 16])
    b = _log(rng, 1, 32)
    if kind == "window":
        sk = _log(rng, 1, 16384)
        sq = min(sk, rng.choice([1, rng.randint(1, 8), _log(rng, 1, 8192), sk]))
        hq = hk * group
        while b * hq * sq * sk > 32 * 8192 * 8192:
            b, sq = max(1, b // 2), sq if b > 1 else max(1, sq // 2)
        while b * hk * sk > 1 << 19 and b > 1:
            b //= 2
        return dict(kind=kind, b=b, hq=hq, hk=hk, sq=sq, sk=sk, d=d, window=_log(rng, 1, 8192), sinks=rng.choice([0, 1, 4, rng.randint(5, 300)]), dtype=dtype)
    if kind == "fill":
        s = _log(rng, 1, 16384)
        new = min(s, rng.choice([1, rng.randint(1, 8), s, rng.randint(1, s)]))
        while b * hk * s > 1 << 18 and b > 1:
            b //= 2
        return dict(kind=kind, b=b, hq=hk * group, hk=hk, s=s, new=new, ragged=rng.random() < 0.7, d=d, dtype=dtype)
    s = _log(rng, 8, 65536)
    while b * hk * s > 1 << 19 and b > 1:
        b //= 2
    ragged = rng.random() < 0.7
    if kind == "decode":
        window = rng.choice([0, 0, _log(rng, 1, 8192)])
        sinks = rng.choice([0, 4, rng.randint(1, 200)]) if window else 0
        return dict(kind=kind, b=b, hq=hk * group, hk=hk, s=s, q_len=rng.choice([1, 1, 1, 2, 3, 4]), ragged=ragged, d=d, window=window, sinks=sinks,
                    weights=rng.random() < 0.4, dtype=dtype)
    keep = rng.randint(1, s)
    recent = rng.randint(0, keep)
    return dict(kind=kind, b=b, hk=hk, s=s, keep=keep, recent=recent, sinks=rng.randint(0, min(8, keep - recent)), ragged=ragged, d=d, dtype=dtype)


def _lens(c):
    """Lengths of the sequences: the longest is ``s``, a ragged batch goes down to a third of it."""
    b, s = c["b"], c["s"]
    return [s - (2 * s * i) // (3 * b) if c["ragged"] else s for i in range(b)]


def _news(c):
    """New tokens of each sequence of a ``fill``."""
    return [min(c["new"], n) if c["new"] < c["s"] else n for n in _lens(c)]


def work(c):
    d, elt = c["d"], 2
    row = c["hk"] * 2 * (d // 2 + 4 * d // GROUP)              # a token of the 4-bit cache, keys and values of all heads
    if c["kind"] == "window":
        off, w, n = c["sk"] - c["sq"], c["window"], c["sinks"]
        pairs = sum(min(p + 1, w + min(n, max(0, p + 1 - w))) for p in range(off, c["sk"]))
        first = max(0, off - w + 1)
        keys = c["sk"] - first + min(n, first)
        return dict(bytes=elt * d * c["b"] * (2 * c["hq"] * c["sq"] + 2 * c["hk"] * keys), flops=4.0 * d * c["b"] * c["hq"] * pairs)
    if c["kind"] == "fill":
        tokens = sum(_news(c))
        # read the new tokens, write them in 4 bits, read those, write their values
        return dict(bytes=tokens * (4 * c["hk"] * d * elt + 2 * row), flops=8.0 * tokens * c["hk"] * d)
    if c["kind"] == "decode":
        total, pairs = 0, 0
        for n in _lens(c):
            w = c["window"] or n
            first = max(0, n - c["q_len"] - w + 1)
            total += n - first + min(c["sinks"], first)
            for p in range(n - c["q_len"], n):
                if p >= 0:
                    pairs += min(p + 1, w + min(c["sinks"], max(0, p + 1 - w)))
        heads = c["b"] * c["q_len"] * c["hq"]
        return dict(bytes=total * row + 2 * heads * d * elt + (8 * total * c["hk"] if c["weights"] else 0), flops=4.0 * d * c["hq"] * pairs)
    lens = _lens(c)
    kept = sum(min(n, c["keep"]) for n in lens)
    # weights read, kept tokens read and written in 4 bits with their weights, then read again and their values written
    return dict(bytes=sum(lens) * c["hk"] * 4 + kept * (3 * row + 8 * c["hk"] + 2 * c["hk"] * d * elt), flops=2.0 * kept * c["hk"] * d * 2)


# ------------------------------------------------------------- the plain form -------------------------------------------------------------

def _quantise(x):
    """``x [..., D]`` -> codes (32-bit floats 0..15) ``[..., D/64, 64]``, scales and zeros ``[..., D/64]`` as the cache holds them."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    s = ((hi - lo) * (1.0 / 15.0)).bfloat16().float()
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    z = lo.bfloat16().float()
    r = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
    codes = ((g - z[..., None]) * r[..., None]).round().clamp(0, 15)
    return codes, s, z


def _pack(codes):
    """Codes ``[..., D/64, 64]`` -> bytes of a row ``[..., D/2]``."""
    c = codes.to(torch.uint8).unflatten(-1, (8, 4, 2))                  # [.., g, w, byte, nibble]
    return (c[..., 0] | (c[..., 1] << 4)).movedim(-3, -2).flatten(-3)   # [.., w, g, byte]


def _views(cache, d):
    """Views of the cache: K codes, K parameters, V codes, V parameters, each [pages, heads, 64, ...]."""
    nc, np_ = PAGE * d // 2, PAGE * d // GROUP * 4
    cuts = cache.split([nc, np_, nc, np_], dim=2)
    return [x.unflatten(2, (PAGE, -1)) for x in cuts]


def _rows(x, scales, zeros):
    """Bytes of codes ``[..., D/2]`` and parameters ``[..., D/64]`` -> values ``[..., D]``."""
    c = torch.stack((x & 15, x >> 4), -1).flatten(-2).unflatten(-1, (8, -1, 8)).movedim(-2, -3).flatten(-2).float()
    return (c * scales[..., None] + zeros[..., None]).flatten(-2)


def _params(bytes_):
    p = bytes_.contiguous().view(torch.bfloat16).float().unflatten(-1, (-1, 2))
    return p[..., 0], p[..., 1]


def _read(st, table, positions, live):
    """Values of K and V ``[B, Hk, n, D]`` at ``positions [B, n]``, zero where not ``live [B, n]``."""
    page = table.gather(1, (positions // PAGE).clamp(0, table.shape[1] - 1).long()).long()
    slot = (positions % PAGE).long()
    out = []
    parts = [v.transpose(1, 2)[page, slot].transpose(1, 2) for v in _views(st["cache"], st["case"]["d"])]     # [B, Hk, n, bytes]
    for codes, params in (parts[:2], parts[2:]):
        out.append(_rows(codes, *_params(params)).masked_fill_(~live[:, None, :, None], 0.0))
    return out


def _attend(q, k, v, visible, scale):
    """q [B, Hk, R, D], k / v [B, Hk, S, D], visible broadcast over [B, Hk, R, S]: (out, probabilities) in 32 bits; a row that sees
    nothing is zero."""
    s = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).masked_fill_(~visible, -math.inf)
    m = s.amax(-1, keepdim=True)
    s.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    total = s.sum(-1, keepdim=True)
    s.div_(torch.where(total > 0, total, torch.ones_like(total)))
    return torch.matmul(s, v), s


def _seen(query_pos, key_pos, window, sinks):
    """Which keys a query sees: none behind it, of those the last ``window`` (0: all) and the first ``sinks``."""
    seen = key_pos <= query_pos
    if window:
        seen = seen & ((query_pos - key_pos < window) | (key_pos < sinks))
    return seen & (key_pos >= 0)


def _plain_window(st):
    c, q, k, v = st["case"], st["q"].float(), st["k"].float(), st["v"].float()
    i = torch.arange(c["sk"] - c["sq"], c["sk"], device=q.device)
    seen = _seen(i[:, None], torch.arange(c["sk"], device=q.device)[None], c["window"], c["sinks"])
    g = c["hq"] // c["hk"]
    rows = q.view(c["b"], c["hk"], g * c["sq"], c["d"])
    out, _ = _attend(rows, k, v, seen.repeat(g, 1), 1.0 / math.sqrt(c["d"]))
    return out.view_as(q).to(st["q"].dtype)


def _plain_fill(st):
    ends, lens, table = st["ends"].long(), st["lens"].long(), st["table"]
    tokens = torch.arange(st["k"].shape[0], device=ends.device)
    seq = torch.searchsorted(ends, tokens, right=True)
    pos = lens[seq] - (ends[seq] - tokens)
    page, slot = table[seq, pos // PAGE].long(), pos % PAGE
    views = _views(st["cache"], st["case"]["d"])
    for x, codes_at, params_at in ((st["k"], *views[:2]), (st["v"], *views[2:])):
        codes, s, z = _quantise(x)
        params = torch.stack((s, z), -1).bfloat16().flatten(-2).view(torch.uint8)
        codes_at.transpose(1, 2)[page, slot] = _pack(codes)
        params_at.transpose(1, 2)[page, slot] = params
    count = st["count"]
    at = st["start"].long()[:, None] + torch.arange(count, device=ends.device)[None]
    return [x.to(st["k"].dtype) for x in _read(st, table, at, at < lens[:, None])]


def _plain_decode(st):
    c, lens = st["case"], st["lens"].long()
    b, hk, t, g = c["b"], c["hk"], c["q_len"], c["hq"] // c["hk"]
    at = torch.arange(st["table"].shape[1] * PAGE, device=lens.device)[None].expand(b, -1)
    k, v = _read(st, st["table"], at, at < lens[:, None])
    q = st["q"].float().view(b, t, hk, g, c["d"]).permute(0, 2, 1, 3, 4).reshape(b, hk, t * g, c["d"])
    pos = lens[:, None] - t + torch.arange(t, device=lens.device)[None]                                    # [B, T]
    seen = _seen(pos[:, :, None], at[:, None], c["window"], c["sinks"])                                       # [B, T, S]
    out, p = _attend(q, k, v, seen.repeat_interleave(g, 1)[:, None], 1.0 / math.sqrt(c["d"]))
    out = out.view(b, hk, t, g, c["d"]).permute(0, 2, 1, 3, 4).reshape(b * t, c["hq"], c["d"]).to(st["q"].dtype)
    if not c["weights"]:
        return {"out": out}
    return {"out": out, "weights": st["weights"].add_(p.sum(2))}


def _plain_evict(st):
    c, lens, w, table = st["case"], st["lens"].long(), st["weights"], st["table"]
    pos = torch.arange(w.shape[2], device=w.device)[None, None]
    n = lens[:, None, None]
    forced = (pos < c["sinks"]) | (pos >= n - c["recent"])
    key = torch.where(pos < n, torch.where(forced, torch.full_like(w, math.inf), w), torch.full_like(w, -math.inf))
    kept = key.sort(dim=-1, descending=True, stable=True).indices[..., :c["keep"]]
    kept = torch.where(kept < n, kept, w.shape[2]).sort(dim=-1).values
    live = kept < n
    new = lens.clamp(max=c["keep"])
    src = torch.where(live, kept, 0)
    heads = torch.arange(c["hk"], device=w.device)[None, :, None]
    page = table[:, None].expand(-1, c["hk"], -1).gather(2, src // PAGE).long()
    slot = src % PAGE
    to = torch.arange(c["keep"], device=w.device)
    to_page, to_slot = st["out_table"][:, to // PAGE].long()[:, None], (to % PAGE)[None, None]
    for view in _views(st["cache"], c["d"]):
        view[to_page, heads, to_slot] = torch.where(live[..., None], view[page, heads, slot], view[to_page, heads, to_slot])
    out_w = st["out_weights"]
    out_w.zero_()
    out_w[..., :c["keep"]] = torch.where(live, w.gather(2, src), torch.zeros((), device=w.device))
    at = to[None].expand(c["b"], -1)
    k, v = _read(st, st["out_table"], at, at < new[:, None])
    return {"kept": torch.where(live, kept, -1).int(), "lens": new.int(), "weights": out_w, "k": k.to(st["dtype"]), "v": v.to(st["dtype"])}


# ------------------------------------------------------------- cases -------------------------------------------------------------

def _cache(c, gen, pages, lens, table):
    """A cache whose pages hold whatever was there before, and the tokens of all sequences."""
    cache = torch.randint(0, 256, (pages, c["hk"], 72 * c["d"]), dtype=torch.uint8, device=DEVICE, generator=gen)
    views = _views(cache, c["d"])
    for i, n in enumerate(lens):
        used = table[i, :(n + PAGE - 1) // PAGE].long()
        for at in (0, 2):
            # channels of unequal size, as keys have them
            x = torch.randn(c["hk"], n, c["d"], device=DEVICE, generator=gen) * (0.5 + torch.rand(c["hk"], 1, c["d"], device=DEVICE, generator=gen))
            codes, s, z = _quantise(x)
            pad = len(used) * PAGE - n
            for view, rows in ((views[at], _pack(codes)), (views[at + 1], torch.stack((s, z), -1).bfloat16().flatten(-2).view(torch.uint8))):
                full = view[used].transpose(0, 1).flatten(1, 2)
                full[:, :n] = rows
                view[used] = full.unflatten(1, (-1, PAGE)).transpose(0, 1)
    return cache


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dt = DTYPES[c["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device=DEVICE, generator=gen).to(dt)

    st = {"case": c, "dtype": dt}
    if c["kind"] == "window":
        st.update(q=randn(c["b"], c["hq"], c["sq"], c["d"]), k=randn(c["b"], c["hk"], c["sk"], c["d"]), v=randn(c["b"], c["hk"], c["sk"], c["d"]))
        return st
    lens = _lens(c)
    width = (c["s"] + PAGE - 1) // PAGE
    kept_width = (c["keep"] + PAGE - 1) // PAGE if c["kind"] == "evict" else 0
    pages = c["b"] * (width + kept_width) + 3
    names = torch.randperm(pages, device=DEVICE, generator=gen).int()
    table = names[:c["b"] * width].view(c["b"], width).contiguous()
    st.update(table=table, lens=torch.tensor(lens, dtype=torch.int32, device=DEVICE))
    if c["kind"] == "fill":
        news = _news(c)
        ends = torch.tensor(news, device=DEVICE).cumsum(0).int()
        # keys and values are parts of the rows that a fused projection wrote
        qkv = randn(sum(news), c["hq"] + 2 * c["hk"], c["d"])
        st.update(cache=torch.randint(0, 256, (pages, c["hk"], 72 * c["d"]), dtype=torch.uint8, device=DEVICE, generator=gen),
                  k=qkv[:, c["hq"]:c["hq"] + c["hk"]], v=qkv[:, c["hq"] + c["hk"]:], ends=ends, count=max(news),
                  start=st["lens"] - torch.tensor(news, dtype=torch.int32, device=DEVICE))
        return st
    st["cache"] = _cache(c, gen, pages, lens, table)
    if c["kind"] == "decode":
        st["q"] = randn(c["b"] * c["q_len"], c["hq"], c["d"])
        if c["weights"]:
            st["weights"] = torch.rand(c["b"], c["hk"], width * PAGE, device=DEVICE, generator=gen)
        return st
    # weights as they accumulate: few heavy tokens, and some that nothing looked at
    w = torch.randn(c["b"], c["hk"], width * PAGE, device=DEVICE, generator=gen).mul_(2).exp_()
    w[torch.rand(w.shape, device=DEVICE, generator=gen) < 0.1] = 0
    st.update(weights=w, out_table=names[c["b"] * width:c["b"] * (width + kept_width)].view(c["b"], kept_width).contiguous(),
              out_weights=torch.empty(c["b"], c["hk"], kept_width * PAGE, device=DEVICE))
    return st


def _own(st):
    import mm_rs_with_catlass_b200 as catcoc
    c = st["case"]
    if c["kind"] == "window":
        return catcoc.flash_attention(st["q"], st["k"], st["v"], causal=True, window=c["window"], sinks=c["sinks"])
    if c["kind"] == "fill":
        catcoc.kv4_append(st["cache"], st["k"], st["v"], st["table"], st["lens"], ends=st["ends"])
        return list(catcoc.kv4_read(st["cache"], st["table"], st["lens"], start=st["start"], count=st["count"], dtype=st["dtype"]))
    if c["kind"] == "decode":
        w = st.get("weights")
        out = catcoc.kv4_decode(st["q"], st["cache"], st["table"], st["lens"], q_len=c["q_len"], window=c["window"] or None, sinks=c["sinks"], weights=w)
        return {"out": out} if w is None else {"out": out, "weights": w}
    kept, new = catcoc.kv4_evict(st["cache"], st["weights"], st["table"], st["lens"], c["keep"], recent=c["recent"], sinks=c["sinks"],
                                 out_table=st["out_table"], out_weights=st["out_weights"])
    k, v = catcoc.kv4_read(st["cache"], st["out_table"], new, count=c["keep"], dtype=st["dtype"])
    return {"kept": kept, "lens": new, "weights": st["out_weights"], "k": k, "v": v}


PLAIN = {"window": _plain_window, "fill": _plain_fill, "decode": _plain_decode, "evict": _plain_evict}


def run(state):
    return _own(state) if own else PLAIN[state["case"]["kind"]](state)


# ------------------------------------------------------------- 64 bits, written apart -------------------------------------------------------------

def _exact_values(cache, d, h, pages, n):
    """Values of one head's first ``n`` tokens on ``pages``: (K, V), each [n, D] in 64 bits, word by word."""
    words = 64 * d // 8
    out = []
    for part in (0, 1):
        base = part * 36 * d
        blocks = cache[pages, h]
        codes = blocks[:, base:base + 32 * d].contiguous().view(torch.int32).view(-1, d // 8)[:n].long()
        par = blocks[:, base + 32 * d:base + 36 * d].contiguous().view(torch.bfloat16).view(-1, d // 64, 2)[:n].double()
        assert codes.shape[1] * 64 == words
        x = torch.empty(n, d, dtype=torch.float64, device=cache.device)
        groups = d // 64
        for word in range(d // 8):
            w, g = word // groups, word % groups
            for nib in range(8):
                x[:, 64 * g + 8 * w + nib] = ((codes[:, word] >> (4 * nib)) & 15).double() * par[:, g, 0] + par[:, g, 1]
        out.append(x)
    return out


def _exact_rows(q, k, v, lo_pos, window, sinks, scale):
    """q [R, D] at positions lo_pos [R]; k, v [n, D]: (out [R, D], probabilities [R, n]) in 64 bits."""
    j = torch.arange(k.shape[0], device=k.device)[None]
    p = lo_pos[:, None]
    hidden = j > p
    if window:
        hidden = hidden | ((j <= p - window) & (j >= sinks))
    s = (q @ k.t() * scale).masked_fill(hidden, -math.inf)
    prob = torch.softmax(s, -1).nan_to_num(0.0)
    return prob @ v, prob


def exact(case, seed):
    c = dict(case)
    st = prepare(c, seed)
    scale = c["d"] ** -0.5
    if c["kind"] == "window":
        if c["b"] * c["hq"] * c["sq"] > 1 << 20:
            return None
        g, out = c["hq"] // c["hk"], torch.empty(st["q"].shape, dtype=torch.float64, device=DEVICE)
        step = max(1, (1 << 27) // c["sk"])
        for b in range(c["b"]):
            for h in range(c["hq"]):
                k, v = st["k"][b, h // g].double(), st["v"][b, h // g].double()
                for r in range(0, c["sq"], step):
                    q = st["q"][b, h, r:r + step].double()
                    at = torch.arange(r, r + q.shape[0], device=DEVICE) + (c["sk"] - c["sq"])
                    out[b, h, r:r + step] = _exact_rows(q, k, v, at, c["window"], c["sinks"], scale)[0]
        return out
    lens = _lens(c)
    if c["kind"] == "fill":
        news, out, first = _news(c), [], 0
        for x in (st["k"], st["v"]):
            # the value that the nearest of the sixteen levels has
            g = x.double().reshape(x.shape[0], c["hk"], c["d"] // 64, 64)
            low, high = g.min(-1).values, g.max(-1).values
            s, z = ((high - low) / 15).float().bfloat16().double(), low.float().bfloat16().double()
            level = torch.round((g - z[..., None]) / s.clamp(min=1e-300)[..., None]).clamp(0, 15)
            val = (z[..., None] + level * s[..., None]).reshape(x.shape)
            y = torch.zeros(c["b"], c["hk"], st["count"], c["d"], dtype=torch.float64, device=DEVICE)
            first = 0
            for b, n in enumerate(news):
                y[b, :, :n] = val[first:first + n].transpose(0, 1)
                first += n
            out.append(y)
        return out
    if c["kind"] == "decode":
        g, t = c["hq"] // c["hk"], c["q_len"]
        out = torch.empty(st["q"].shape, dtype=torch.float64, device=DEVICE)
        weights = st["weights"].double() if c["weights"] else None
        for b, n in enumerate(lens):
            pages = st["table"][b, :(n + 63) // 64].long()
            for h in range(c["hk"]):
                k, v = _exact_values(st["cache"], c["d"], h, pages, n)
                for i in range(t):
                    at = torch.full((g,), n - t + i, device=DEVICE)
                    o, p = _exact_rows(st["q"][b * t + i, h * g:(h + 1) * g].double(), k, v, at, c["window"], c["sinks"], scale)
                    out[b * t + i, h * g:(h + 1) * g] = o
                    if weights is not None:
                        weights[b, h, :n] += p.sum(0)
        return {"out": out} if weights is None else {"out": out, "weights": weights}
    if c["b"] * c["hk"] > 256:
        return None
    k_out = torch.zeros(c["b"], c["hk"], c["keep"], c["d"], dtype=torch.float64, device=DEVICE)
    v_out, w_out = torch.zeros_like(k_out), torch.zeros_like(st["out_weights"], dtype=torch.float64)
    for b, n in enumerate(lens):
        pages = st["table"][b, :(n + 63) // 64].long()
        for h in range(c["hk"]):
            w = st["weights"][b, h, :n]
            k, v = _exact_values(st["cache"], c["d"], h, pages, n)
            keep = torch.zeros(n, dtype=torch.bool, device=DEVICE)
            if n <= c["keep"]:
                keep[:] = True
            else:
                keep[:c["sinks"]] = True
                keep[n - c["recent"]:] = True
                rest = (~keep).nonzero()[:, 0]
                free = c["keep"] - c["sinks"] - c["recent"]
                keep[rest[torch.argsort(-w[rest], stable=True)[:free]]] = True
            at = keep.nonzero()[:, 0]
            k_out[b, h, :len(at)], v_out[b, h, :len(at)], w_out[b, h, :len(at)] = k[at], v[at], w[at].double()
    return {"kept": None, "lens": None, "weights": w_out, "k": k_out, "v": v_out}
