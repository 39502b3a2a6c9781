"""Attention over a shared prefix where there is nothing to read: a pool without pages, a table without columns or requests."""
import pytest
import torch

from test_shared_attention_gpu import FORMS, K, call, ints, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,hd,page,dtype", [FORMS[0], FORMS[2], FORMS[4], FORMS[6], FORMS[8]])
@pytest.mark.parametrize("what", ["pages", "columns", "requests", "keys"])
def test_nothing_to_read_is_zeros(heads, kv_heads, hd, page, dtype, what):
    s = make([(2 * page, [3, page, 2]), (0, [5])], heads, kv_heads, hd, page, dtype, stale=0.0)
    if what == "pages":
        s["k_cache"], s["v_cache"] = s["k_cache"][:0], s["v_cache"][:0]
    elif what == "columns":
        s["block_table"] = s["block_table"][:, :0].contiguous()
    elif what == "requests":
        s["block_table"] = s["block_table"][:0]
    else:
        s["positions"].fill_(-1)
    out = torch.full_like(s["q"], 7.0)
    for got in (call(s, max_prefix=2 * page, max_context=4 * page), call(s, out=out, max_prefix=2 * page, max_context=4 * page)):
        assert bool((got == 0).all())
    s["group_start"], s["prefix_lens"] = ints([1, 2]), ints([page])               # rows of no group stay as they are
    out.fill_(7.0)
    call(s, out=out, max_prefix=2 * page, max_context=4 * page)
    assert bool((out[1] == 0).all()) and bool((out[0] == 7).all()) and bool((out[2:] == 7).all())
    torch.cuda.synchronize()
    K().check_kernel_errors()
