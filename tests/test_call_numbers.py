"""Calls that are kept by their layouts and numbers (the 4-bit cache, windowed attention): a number given as a 0-dim tensor counts for what it holds at the call,
not for what it held at the first one."""
import pytest
import torch

from mm_rs_with_catlass_b200 import _native as N
from mm_rs_with_catlass_b200.ops import attention, kv4


class _Entries:
    """Stands in for the library: the numbers of each call, by name."""

    def __init__(self):
        self.seen = []

    def __getattr__(self, name):
        if name == "catcoc_kv4_decode_workspace_bytes":
            return lambda call, weights: 256
        if name == "catcoc_window_route":
            return lambda *numbers: 0

        def entry(*args):
            if name == "catcoc_window_attention":
                self.seen.append(dict(window=args[12], sinks=args[13], scale=args[14]))
            else:
                call = N.Kv4Call.from_address(args[0])
                self.seen.append({field: getattr(call, field) for field, _ in N.Kv4Call._fields_})
            return 0
        return entry


@pytest.fixture
def entries(monkeypatch):
    """CPU tensors in place of the GPU's, and the entries that a call would reach."""
    fake = _Entries()
    monkeypatch.setattr(kv4.cm, "require_cuda", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(kv4.cm, "on_device", lambda device: True)
    monkeypatch.setattr(kv4.cm, "stream_of", lambda device: 0)
    monkeypatch.setattr(kv4.N, "lib", lambda: fake)
    monkeypatch.setattr(kv4, "_plans", {})
    monkeypatch.setattr(attention, "_windows", {})
    return fake


def _calls():
    cache, table, lens = torch.zeros(4, 2, 72 * 64, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    q, w = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 2, 128)
    x = torch.zeros(1, 2, 8, 64, dtype=torch.bfloat16)
    return {
        "decode": lambda **n: kv4.kv4_decode(q, cache, table, lens, **n),
        "read": lambda **n: kv4.kv4_read(cache, table, lens, **n),
        "evict": lambda keep=20, **n: kv4.kv4_evict(cache, w, table, lens, keep, **n),
        "window": lambda **n: attention.flash_attention(x, x, x, causal=True, **n),
    }


@pytest.mark.parametrize("op,number,first,second,more", [
    ("decode", "scale", 0.5, 0.25, {}), ("decode", "window", 3, 7, {}), ("decode", "sinks", 2, 5, dict(window=4)),
    ("read", "count", 3, 9, {}), ("evict", "keep", 20, 30, {}), ("evict", "recent", 3, 4, {}), ("evict", "sinks", 1, 2, {}),
    ("window", "scale", 0.5, 0.25, dict(window=4)), ("window", "window", 3, 7, {}), ("window", "sinks", 1, 5, dict(window=4)),
])
def test_a_tensor_is_read_at_every_call(entries, op, number, first, second, more):
    call, x = _calls()[op], torch.tensor(first)
    call(**{number: x}, **more)
    x.fill_(second)
    call(**{number: x}, **more)
    call(**{number: first}, **more)
    assert [n[number] for n in entries.seen] == [first, second, first]


def test_the_number_of_tokens_and_causal_are_read_too(entries):
    calls, one = _calls(), torch.tensor(1)
    calls["decode"](q_len=one)
    with pytest.raises(ValueError):
        calls["decode"](q_len=one.fill_(2))                    # two tokens for two sequences
    x, causal = torch.zeros(1, 2, 8, 64, dtype=torch.bfloat16), torch.tensor(True)
    attention.flash_attention(x, x, x, causal=causal, window=3)
    with pytest.raises(ValueError):
        attention.flash_attention(x, x, x, causal=causal.fill_(False), window=3)


def test_fractions_are_refused(entries):
    calls = _calls()
    for op, n in (("decode", dict(window=2.5)), ("decode", dict(q_len=1.5)), ("read", dict(count=1.5)), ("evict", dict(keep=2.5)), ("window", dict(window=1.5))):
        with pytest.raises(TypeError):
            calls[op](**n)
    calls["decode"](window=2.0)
    assert entries.seen[-1]["window"] == 2




def test_numbers_of_more_than_32_bits_are_refused(entries):
    """The library's numbers have 32 bits: 2^32 + 5 would arrive as 5."""
    from types import SimpleNamespace
    with pytest.raises(ValueError):
        _calls()["evict"](keep=(1 << 32) + 5)
    assert not entries.seen
    long = SimpleNamespace(dtype=torch.float32, dim=lambda: 3, shape=(1, 1, (1 << 32) + 64), is_contiguous=lambda: True)
    with pytest.raises(ValueError):
        kv4._weights(long, 1, 1, 64)


def test_the_library_refuses_what_its_loops_cannot_count():
    """Eviction steps over places and weights in int: past 2^30 of them it is refused, before any launch."""
    import ctypes
    numbers = dict(B=1, Hk=1, D=64, pages=4, max_pages=2, fmt=N.FMT_BF16, keep=100, recent=2, sinks=2, out_pages=2, S=128, S_out=128)

    def evict(**changes):
        call = N.Kv4Call(**{**numbers, **changes})
        return N.lib().catcoc_kv4_evict(ctypes.addressof(call), *[16] * 9, None)
    assert evict(keep=(1 << 30) + 1) == N.E_TOO_LARGE and evict(keep=0x7fffffff) == N.E_TOO_LARGE
    assert evict(S_out=0x7fffffff) == N.E_TOO_LARGE
    assert evict(max_pages=(1 << 24) + 1, S=0x7fffffff) == N.E_TOO_LARGE
