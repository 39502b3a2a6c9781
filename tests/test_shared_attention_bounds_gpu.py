"""Attention over a shared prefix, each type to its own bound: views, rows of no group, requests that are not there, replays, positions
at the end of 32 bits."""
import pytest
import torch

from serving_util import shared_attention, shared_attention_error
from test_shared_attention_gpu import FORMS, K, call, ints, make

pytestmark = pytest.mark.gpu
SOME = [FORMS[0], FORMS[2], FORMS[4], FORMS[8], FORMS[9], FORMS[10]]


def agree(got, s, rows=slice(None)):
    """`rows` of `got` against 64 bits."""
    hd = s["q"].shape[2]
    want, size, reach = shared_attention(*(s[n].cpu() for n in ("q", "k_cache", "v_cache", "block_table", "token_req", "positions")), hd ** -0.5)
    error = shared_attention_error(want, size, reach, hd, got.dtype)
    assert bool(((got.cpu().double() - want).abs() <= error)[rows].all())
    K().check_kernel_errors()


@pytest.mark.parametrize("heads,kv_heads,hd,page,dtype", SOME)
def test_queries_of_any_stride(heads, kv_heads, hd, page, dtype):
    s = make([(600, [3, 70, 21, 300]), (100, [2])], heads, kv_heads, hd, page, dtype)
    for more in (1, 2, 3, 8):
        wide = torch.zeros((5, heads * hd + more), dtype=dtype, device="cuda")
        wide[:, more:] = s["q"].view(5, -1)
        agree(call({**s, "q": wide[:, more:].view(5, heads, hd)}), s)


@pytest.mark.parametrize("heads,kv_heads,hd,page,dtype", SOME)
def test_rows_of_a_group_beside_rows_of_none(heads, kv_heads, hd, page, dtype):
    s = make([(100, [3, 70, 21, 9, 5])], heads, kv_heads, hd, page, dtype)
    s["group_start"], s["prefix_lens"] = ints([1, 1, 3]), ints([64, 100])
    out = torch.full_like(s["q"], 7.0)
    agree(call(s, out=out), s, slice(1, 3))
    assert bool((out[0] == 7).all()) and bool((out[3:] == 7).all())


@pytest.mark.parametrize("heads,kv_heads,hd,page,dtype", SOME)
def test_a_request_that_is_not_there_sees_the_prefix(heads, kv_heads, hd, page, dtype):
    s = make([(2 * page + 3, [3, page, 2])], heads, kv_heads, hd, page, dtype, stale=0.0)
    s["token_req"][2] = 99
    got = call(s)
    s["token_req"][2], s["positions"][2] = 0, 2 * page + 2
    agree(got, s)


@pytest.mark.parametrize("heads,kv_heads,hd,page,dtype", SOME)
def test_a_replay_reads_the_present_state(heads, kv_heads, hd, page, dtype):
    s = make([(600, [3, 70, 21, 300]), (100, [2])], heads, kv_heads, hd, page, dtype)
    call(s)
    graph, out = torch.cuda.CUDAGraph(), torch.zeros_like(s["q"])
    with torch.cuda.graph(graph):
        call(s, out=out, max_prefix=600, max_context=900)
    for prefix in (600, 511, 64, 0):
        s["prefix_lens"].copy_(ints([prefix, min(prefix, 100)]))
        graph.replay()
        agree(out, s)
        s["positions"].sub_(1)
        s["q"].mul_(-0.75)


@pytest.mark.parametrize("heads,kv_heads,hd,page,dtype", SOME)
def test_positions_behind_the_table(heads, kv_heads, hd, page, dtype):
    """They see what the table has, whatever the longest context is said to be."""
    s = make([(page, [2 * page, page])], heads, kv_heads, hd, page, dtype, stale=0.0)
    s["block_table"] = s["block_table"][:, :2].contiguous()
    for position in (2 * page - 1, 2 * page, 0x7ffffffe, 0x7fffffff):
        for max_context in (2 * page, 3 * page, 1):
            s["positions"].fill_(position)
            got = call(s, max_prefix=page, max_context=max_context)
            s["positions"].fill_(2 * page - 1)
            agree(got, s)


@pytest.mark.parametrize("heads,kv_heads,hd,page", [(12, 2, 128, 64), (8, 2, 64, 64), (16, 1, 96, 64), (8, 2, 64, 5)])
@pytest.mark.parametrize("prefix,own", [(3000, 1), (900, 700), (1, 1500), (0, 1500)])
def test_bfloat16_is_off_by_the_rounding_of_the_output(heads, kv_heads, hd, page, prefix, own):
    """The mean square of the errors.  A rounding is off by up to half a step, evenly spread: a twelfth of the step's square.  The scores,
    the weights and their sums are held in more bits than that, and so is what goes into the product with the values: all of it is to
    leave a tenth at most (12,000 numbers or more, whose mean square is known within a hundredth).  Weights rounded to bfloat16 would
    leave as much again as the output's rounding."""
    s = make([(prefix, [own + 3 * i for i in range(24)])], heads, kv_heads, hd, page, torch.bfloat16)
    want, _, _ = shared_attention(*(s[n].cpu() for n in ("q", "k_cache", "v_cache", "block_table", "token_req", "positions")), hd ** -0.5)
    step = 2.0 ** (torch.floor(torch.log2(want.abs().clamp(min=2.0 ** -40))) - 7)
    off = (call(s).cpu().double() - want).square().mean()
    assert float(off) <= 1.1 * float(step.square().mean()) / 12
