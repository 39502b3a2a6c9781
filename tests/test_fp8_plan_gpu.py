"""The cache plan beside 8-bit feed-forward weights: what they free is there for pages."""
import gc

import pytest
import torch

from tiny import TINY, make_model_dir

pytestmark = pytest.mark.gpu


def test_8_bit_weights_leave_more_pages(tmp_path):
    """Two layers whose feed-forwards hold 200 MB in 16 bits, and a plan that takes what memory there is."""
    from logssms_b200.cache.manager import CacheManager
    from logssms_b200.engine import Engine
    inter, hidden = 256 * 1024, 64
    raw = {**TINY["A"], "intermediate_size": inter}
    model_dir = make_model_dir(tmp_path / "m", raw, seed=1, dtype=torch.bfloat16)
    held = 3 * raw["num_hidden_layers"] * inter * hidden * 2
    gc.collect()
    torch.cuda.empty_cache()                               # (what tests before this one have left behind)
    free, total = torch.cuda.mem_get_info()
    ratio = 1 - (free - (1 << 30)) / total                 # about 1 GB for the engine, whatever the device holds besides
    pages = {}
    for choice in ("model", "float8"):
        gc.collect()
        torch.cuda.empty_cache()
        engine = Engine(model_dir, "bfloat16", max_requests=64, max_seq_len=1 << 18, memory_ratio=ratio, use_graphs=False,
                        feed_forward_weights=choice)
        per_page = CacheManager.bytes_per_page(engine.model.cache_needs(), 64, torch.bfloat16)
        pages[choice] = engine.cache.groups[0].pool.count
        del engine
    assert pages["float8"] < 1 << 18                       # not what the requests could use at most
    # half of the weights' bytes, less the segments that the allocator fills up (2 MB each) and what other parts hold in them
    assert (pages["float8"] - pages["model"]) * per_page >= held // 2 - (32 << 20)
