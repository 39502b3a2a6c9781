"""Adapters of many rows (`adapters_tiles.cuh`): what the short prompts of test_adapters_gpu.py do not reach."""
import pytest
import torch

from test_adapters_gpu import K, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width,features,rank", [(65, 64, 13), (65, 65, 16), (64, 129, 8), (64, 64, 12), (64, 64, 8)])
@pytest.mark.parametrize("n", [1, 3])
def test_copies_are_launches_too(width, features, rank, n):
    """x, A or B off 16 bytes are copied first, by a kernel that counts; both ways of a call."""
    from torch.profiler import ProfilerActivity, profile
    s = make(400, width, features, n, rank, torch.bfloat16, [t % n for t in range(400)])
    out = torch.empty_like(s["y"])
    for kw in ({}, {"out": out}):
        call = lambda: K().add_adapters(s["y"], s["x"], s["a"], s["b"], s["index"], s["scales"], **kw)         # noqa: E731
        call()
        before = K().launch_count
        with profile(activities=[ProfilerActivity.CUDA]) as p:
            call()
            torch.cuda.synchronize()
        ran = sum(e.count for e in p.key_averages() if "adapter_" in e.key)
        assert K().launch_count - before == ran == 1 + (n > 1) + (width % 8 != 0 or rank % 8 != 0)
