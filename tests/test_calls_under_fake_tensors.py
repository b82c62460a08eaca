"""A call under ``FakeTensorMode`` is refused and leaves nothing behind: what the process keeps of calls (what results are made like, the status block) is
memory of its own, so that later calls of the same layouts run."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from mm_rs_with_catlass_b200.ops import _common as cm
from mm_rs_with_catlass_b200.ops import attention, kv4


class _Entries:
    """Stands in for the library: every call passes that brings addresses of real memory."""

    def __getattr__(self, name):
        if name == "catcoc_kv4_decode_workspace_bytes":
            return lambda call, weights: 256
        if name == "catcoc_window_route":
            return lambda *numbers: 512

        def entry(*args):
            assert args[:5].count(0) == 0 and args[-1] == 0
            return 0
        return entry


@pytest.fixture
def no_gpu(monkeypatch):
    monkeypatch.setattr(cm, "require_cuda", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(cm, "on_device", lambda device: True)
    monkeypatch.setattr(cm, "stream_of", lambda device: 0)
    monkeypatch.setattr(kv4.N, "lib", lambda: _Entries())
    monkeypatch.setattr(cm, "_status_cache", {})
    monkeypatch.setattr(kv4, "_plans", {})
    monkeypatch.setattr(attention, "_windows", {})


def _inputs():
    return dict(cache=torch.zeros(4, 2, 72 * 64, dtype=torch.uint8), table=torch.zeros(2, 2, dtype=torch.int32), lens=torch.ones(2, dtype=torch.int32),
                q=torch.zeros(2, 4, 64, dtype=torch.bfloat16), kv=torch.zeros(2, 2, 64, dtype=torch.bfloat16), w=torch.zeros(2, 2, 128),
                x=torch.zeros(1, 2, 8, 64, dtype=torch.bfloat16))


CALLS = {
    "append": lambda i: kv4.kv4_append(i["cache"], i["kv"], i["kv"], i["table"], i["lens"]),
    "read": lambda i: kv4.kv4_read(i["cache"], i["table"], i["lens"]),
    "decode": lambda i: kv4.kv4_decode(i["q"], i["cache"], i["table"], i["lens"], weights=i["w"]),
    "evict": lambda i: kv4.kv4_evict(i["cache"], i["w"], i["table"], i["lens"], 7),
    "window": lambda i: attention.flash_attention(i["x"], i["x"], i["x"], causal=True, window=4),
}


@pytest.mark.parametrize("status", [False, True])
@pytest.mark.parametrize("real_inputs", [False, True])
@pytest.mark.parametrize("op", CALLS)
def test_a_refused_call_leaves_nothing_behind(no_gpu, op, real_inputs, status):
    if status:
        cm.local_status(torch.device("cpu"))                 # the process has run other calls before
    real = _inputs()
    with FakeTensorMode(allow_non_fake_inputs=True):
        if not (real_inputs and status and op == "append"):  # (which makes no tensor: it runs)
            with pytest.raises((RuntimeError, AssertionError)):
                CALLS[op](real if real_inputs else _inputs())
    got = CALLS[op](real)
    assert all(type(t) is torch.Tensor and t.data_ptr() for t in (got if isinstance(got, tuple) else (got,)))


def test_the_status_block_is_real(no_gpu):
    with FakeTensorMode(), pytest.raises(RuntimeError):
        cm.local_status(torch.device("cpu"))
    assert type(cm.local_status(torch.device("cpu"))) is torch.Tensor
