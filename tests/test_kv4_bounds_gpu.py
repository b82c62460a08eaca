"""The 4-bit cache at the ends of what its tables name: lengths that a row cannot hold, and pages that are not in the cache."""
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
