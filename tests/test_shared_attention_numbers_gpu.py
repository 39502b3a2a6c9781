"""Infinities and NaN among the values of a shared prefix (`attention_shared.cu`): those that a row sees are its result at no cost; those
that it does not see cost a walk over its own keys and leave no trace."""
import pytest
import torch

from serving_util import shared_attention, shared_attention_error
from test_shared_attention_gpu import FORMS, K, call, ints, make

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def inside(heads, kv_heads, hd, page, dtype, prefix=20000):
    """Eight tokens that stand inside of a long prefix."""
    s = make([(prefix, [4] * 8)], heads, kv_heads, hd, page, dtype, stale=0.0)
    s["positions"].copy_(ints([prefix - 1000 + 100 * i for i in range(8)]))
    return s


def put(s, key, column, value):
    page = s["k_cache"].shape[1]
    s["v_cache"][int(s["block_table"][0, key // page]), key % page, 0, column] = value


def least_ms(f, n=5):
    f()
    torch.cuda.synchronize()
    took = []
    for _ in range(n):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        took.append(a.elapsed_time(b))
    return min(took)


@pytest.mark.parametrize("heads,kv_heads,hd,page,dtype", [FORMS[2], FORMS[9]])
@pytest.mark.parametrize("value", [INF, -INF, NAN])
def test_what_a_row_sees_costs_nothing(heads, kv_heads, hd, page, dtype, value):
    """Each head of the key/value head has this value in its column 3, and every other column as it was."""
    s = inside(heads, kv_heads, hd, page, dtype)
    run = lambda: call(s, max_prefix=20000, max_context=20004)          # noqa: E731
    want, clean = run(), least_ms(run)
    put(s, 5, 3, value)
    got = run()
    G = heads // kv_heads
    assert bool((got[:, :G, 3].isnan() if value != value else got[:, :G, 3] == value).all())
    got[:, :G, 3] = want[:, :G, 3]
    assert torch.equal(got, want)
    assert least_ms(run) < 4 * clean + 0.1          # (a walk over 19,000 keys, one at a time, takes 100 times as long)
    s["q"][0, 0, 0] = NAN
    assert bool(run()[0, 0].isnan().all()) and least_ms(run) < 4 * clean + 0.1


@pytest.mark.parametrize("heads,kv_heads,hd,page,dtype", [FORMS[0], FORMS[2], FORMS[4], FORMS[6], FORMS[8], FORMS[11], FORMS[13]])
def test_what_a_row_does_not_see_leaves_no_trace_in_a_long_prefix(heads, kv_heads, hd, page, dtype):
    """Infinities right behind each token, so that every row's last tile of keys holds some that are not its own; one token sees an
    infinity and a NaN as well, in columns of their own."""
    prefix = 2000
    s = make([(prefix, [4] * 8)], heads, kv_heads, hd, page, dtype, stale=0.0)
    s["positions"].copy_(ints([1000 + 100 * i for i in range(8)]))
    for i in range(8):
        put(s, 1001 + 100 * i, i % hd, (INF, -INF, NAN)[i % 3])
    want, size, reach = shared_attention(*(s[n].cpu() for n in ("q", "k_cache", "v_cache", "block_table", "token_req", "positions")), hd ** -0.5)
    got = call(s).cpu().double()
    fine = want.isfinite() & size.isfinite()
    assert int((~fine).sum()) > 0 and bool(fine[0].all())
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    assert torch.equal(got[want.isinf()], want[want.isinf()])
    error = shared_attention_error(want, size, reach, hd, dtype)
    assert bool(((got - want).abs() <= error)[fine].all())
    K().check_kernel_errors()
