"""One group of few rows is launched for its rows, as a projection of as many rows is, and
not for twice as many."""
import re

import pytest

torch = pytest.importorskip("torch")


def _kernel(call):
    from torch.profiler import ProfilerActivity, profile
    call()
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CPU, ProfilerActivity.CUDA]) as p:
        call()
        torch.cuda.synchronize()
    # the name but for its last argument, which says whether there are adapters; 16-bit types
    # are not spelled out in it, but the ring's stages tell the rows apart
    found = [re.sub(r"(true|false)>\(.*", "", e.key) for e in p.key_averages()
             if "few_rows_product" in e.key]
    assert len(found) == 1, [e.key for e in p.key_averages()]
    return found[0]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,K", [(16, 4096), (32, 4096)])
def test_one_group_is_launched_as_a_projection(S, rows, K):
    x = torch.randn(rows, K, device="cuda").bfloat16()
    w = torch.randn(1, 4096, K, device="cuda").bfloat16()
    offsets = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    a, b = torch.zeros(1, 8, K, device="cuda").bfloat16(), torch.zeros(1, 4096, 8, device="cuda").bfloat16()
    ids = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    one = _kernel(lambda: S.grouped_mm(x, w, offsets))
    assert one == _kernel(lambda: S.adapter_mm(x, w[0], a, b, ids))
