"""A device's status block serves calls inside and outside of ``torch.inference_mode``, wherever it was first made."""
import pytest
import torch

from mm_rs_with_catlass_b200.ops import _common as cm


@pytest.mark.parametrize("made_inside", [False, True])
@pytest.mark.parametrize("read_inside", [False, True])
def test_inference_mode(monkeypatch, made_inside, read_inside):
    monkeypatch.setattr(cm, "_status_cache", {})
    with torch.inference_mode(made_inside):
        status = cm.local_status(torch.device("cpu"))
    status.numpy()[:] = [3, 0, 401, 5, 9, 0, 0, 0]             # as a kernel writes it
    with torch.inference_mode(read_inside):
        with pytest.raises(cm.StatusError):
            cm.raise_on_status(cm.local_status(torch.device("cpu")), "call")
        cm.raise_on_status(cm.local_status(torch.device("cpu")), "call")
    assert status.tolist() == [0] * 8
