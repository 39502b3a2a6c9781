"""Attention over a shared prefix (`attention_shared*.cu`) against 64 bits, token by token."""
import pytest
import torch

from serving_util import shared_attention, shared_attention_error

pytestmark = pytest.mark.gpu


def K():
    from logssms_b200.ops import kernels
    return kernels


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def make(groups, heads, kv_heads, hd, page, dtype, seed=0, stale=float("nan"), per=1, q_size=1.0):
    """`groups`: (prefix, [own keys of each request]) per group.  Every place that no key was written to holds `stale`."""
    g = torch.Generator().manual_seed(seed + hd + page)
    requests = sum(len(own) for _, own in groups)
    columns = max(-(-(p + max(own, default=0)) // page) for p, own in groups) + 1
    pages = sum(-(-p // page) + sum(-(-(p + n) // page) - p // page for n in own) for p, own in groups) + 3
    free = torch.randperm(pages, generator=g).tolist()
    k = torch.full((pages, page, kv_heads, hd), stale)
    v = k.clone()
    table = torch.full((requests, columns), pages + 7, dtype=torch.int32)       # places without a page name none
    positions, token_req, starts, r = [], [], [0], 0
    for p, own in groups:
        keys, values = (torch.randn((p, kv_heads, hd), generator=g) for _ in range(2))
        shared = [free.pop() for _ in range(p // page)]
        for i, pg in enumerate(shared):
            k[pg], v[pg] = keys[i * page:(i + 1) * page], values[i * page:(i + 1) * page]
        for n in own:
            mine = [free.pop() for _ in range(-(-(p + n) // page) - len(shared))]
            row = shared + mine
            table[r, :len(row)] = torch.tensor(row, dtype=torch.int32)
            rest_k = torch.cat([keys[len(shared) * page:], torch.randn((n, kv_heads, hd), generator=g)])
            rest_v = torch.cat([values[len(shared) * page:], torch.randn((n, kv_heads, hd), generator=g)])
            for i, pg in enumerate(mine):
                part = rest_k[i * page:(i + 1) * page]
                k[pg, :len(part)], v[pg, :len(part)] = part, rest_v[i * page:(i + 1) * page]
            for i in range(per):
                positions.append(max(p + n - per + i, -1))
                token_req.append(r)
            r += 1
        starts.append(starts[-1] + len(own) * per)
    q = torch.randn((len(positions), heads, hd), generator=g) * q_size
    return {"q": q.to(dtype).cuda(), "k_cache": k.to(dtype).cuda(), "v_cache": v.to(dtype).cuda(), "block_table": table.cuda(),
            "token_req": ints(token_req), "positions": ints(positions), "group_start": ints(starts),
            "prefix_lens": ints([p for p, _ in groups])}


def call(s, out=None, max_prefix=None, max_context=None, scale=None):
    scale = s["q"].shape[2] ** -0.5 if scale is None else scale
    if max_prefix is None:
        max_prefix = int(s["prefix_lens"].max()) if s["prefix_lens"].numel() else 0
    if max_context is None:
        max_context = int(s["positions"].max()) + 1
    return K().attention_decode_shared(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["token_req"], s["positions"],
                                       s["group_start"], s["prefix_lens"], scale, max_prefix=max_prefix, max_context=max_context, out=out)


def check(s, **kw):
    hd = s["q"].shape[2]
    want, size, reach = shared_attention(*(s[n].cpu() for n in ("q", "k_cache", "v_cache", "block_table", "token_req", "positions")), hd ** -0.5)
    got = call(s, **kw)
    assert got.dtype == s["q"].dtype and got.shape == s["q"].shape
    error = shared_attention_error(want, size, reach, hd, got.dtype)
    assert bool(((got.cpu().double() - want).abs() <= error).all())
    K().check_kernel_errors()
    return got


FORMS = [(8, 2, 64, 64, torch.bfloat16), (6, 2, 128, 64, torch.bfloat16), (12, 2, 128, 128, torch.bfloat16), (4, 4, 64, 16, torch.bfloat16),
         (16, 1, 96, 64, torch.bfloat16), (20, 1, 128, 64, torch.bfloat16), (3, 1, 8, 5, torch.bfloat16), (4, 2, 256, 32, torch.bfloat16),
         (8, 2, 64, 64, torch.float32), (6, 2, 128, 48, torch.float32), (5, 1, 24, 7, torch.float32), (2, 1, 256, 64, torch.float32),
         (16, 1, 96, 16, torch.bfloat16), (6, 2, 128, 16, torch.bfloat16), (4, 2, 96, 48, torch.bfloat16), (8, 2, 64, 32, torch.bfloat16),
         (34, 2, 128, 64, torch.bfloat16), (6, 2, 128, 24, torch.bfloat16)]


@pytest.mark.parametrize("heads,kv_heads,hd,page,dtype", FORMS)
def test_groups_of_every_kind(heads, kv_heads, hd, page, dtype):
    """A single token, an empty group, no prefix, prefixes that end inside of a page and on its end, own parts of nothing to many."""
    check(make([(1, [1])], heads, kv_heads, hd, page, dtype))
    check(make([(300, [1, 5, 64, 200])], heads, kv_heads, hd, page, dtype))
    check(make([(0, [3, 70]), (128, [1, 2, 1]), (257, []), (63, [130])], heads, kv_heads, hd, page, dtype))
    check(make([(64, [0, 0, 9])], heads, kv_heads, hd, page, dtype))            # tokens that stand on the prefix's last key


@pytest.mark.parametrize("heads,kv_heads,hd,page,dtype", FORMS[:6] + FORMS[8:9] + FORMS[12:16])
@pytest.mark.parametrize("requests", [9, 40, 90])
def test_more_rows_than_a_tile(heads, kv_heads, hd, page, dtype, requests):
    check(make([(700, [1 + (i * 37) % 150 for i in range(requests)])], heads, kv_heads, hd, page, dtype))


@pytest.mark.parametrize("heads,kv_heads,hd,page,dtype", FORMS[:3] + FORMS[8:9] + FORMS[12:14])
def test_a_long_prefix(heads, kv_heads, hd, page, dtype):
    check(make([(5000, [10, 3000, 1, 77])], heads, kv_heads, hd, page, dtype))
    check(make([(5000, [10, 300]), (2500, [4] * 11)], heads, kv_heads, hd, page, dtype, q_size=4.0))


@pytest.mark.parametrize("heads,kv_heads,hd,page,dtype", [FORMS[0], FORMS[2], FORMS[8]])
def test_several_tokens_of_a_request_and_tokens_inside_the_prefix(heads, kv_heads, hd, page, dtype):
    check(make([(200, [4, 60, 130]), (70, [5])], heads, kv_heads, hd, page, dtype, per=4))
    s = make([(200, [4, 60, 130])], heads, kv_heads, hd, page, dtype, stale=0.0)
    s["positions"].copy_(ints([17, 259, -1]))                                   # within the prefix; at the end; nowhere
    got = check(s)
    assert bool((got[2] == 0).all())


@pytest.mark.parametrize("heads,kv_heads,hd,page,dtype", [FORMS[0], FORMS[2], FORMS[4], FORMS[6], FORMS[8], FORMS[13]])
@pytest.mark.parametrize("stale", [float("nan"), float("inf")])
def test_what_a_row_does_not_see_may_be_anything(heads, kv_heads, hd, page, dtype, stale):
    """Tokens inside of the prefix: keys and values behind all of them; behind some of them (those that see it are no numbers)."""
    s = make([(200, [4, 60, 130]), (150, [9])], heads, kv_heads, hd, page, dtype, stale=0.0, q_size=2.0)
    s["positions"].copy_(ints([17, 99, 98, 158]))
    want = check(s)
    row = s["block_table"][0].long()
    for j in range(100, 200):
        s["k_cache"][row[j // page], j % page] = stale
        s["v_cache"][row[j // page], j % page] = stale
    got = call(s)
    scale_of_values = float(s["v_cache"][s["v_cache"].isfinite()].abs().max())
    close = (2.0 ** -6 if dtype == torch.bfloat16 else 2.0 ** -16) * scale_of_values   # weights in bfloat16 or in 32 bits: 2^-8 of the values, twice
    assert bool(((got.float() - want.float()).abs() <= close).all())
    s["v_cache"][row[99 // page], 99 % page] = stale                            # token 1 sees this one
    again = call(s)
    assert not bool(again[1].isfinite().any())
    keep = [0, 2, 3]
    assert bool(((again[keep].float() - want[keep].float()).abs() <= close).all())
    K().check_kernel_errors()


@pytest.mark.parametrize("heads,kv_heads,hd,page,dtype", [FORMS[0], FORMS[8]])
def test_positions_at_the_end_of_32_bits(heads, kv_heads, hd, page, dtype):
    """A position behind everything sees all that its table has."""
    s = make([(page, [2 * page, page])], heads, kv_heads, hd, page, dtype, stale=0.0)
    s["block_table"] = s["block_table"][:, :2].contiguous()
    s["positions"].copy_(ints([2 * page - 1, 2 * page - 1]))
    want = check(s)
    s["positions"].fill_(0x7fffffff)
    assert torch.equal(call(s, max_context=3 * page), call(s, max_context=3 * page))
    assert bool(((call(s, max_context=2 * page).float() - want.float()).abs() <= 2.0 ** -6).all())


@pytest.mark.parametrize("heads,kv_heads,hd,page,dtype", [FORMS[0], FORMS[2], FORMS[4], FORMS[8]])
def test_cutting_up_changes_no_result(heads, kv_heads, hd, page, dtype):
    s = make([(1500, [5, 900, 40])], heads, kv_heads, hd, page, dtype)
    for max_prefix, max_context in ((1, 1), (1500, 2400), (100000, 200000), (0, 10 ** 9)):
        check(s, max_prefix=max_prefix, max_context=max_context)


@pytest.mark.parametrize("heads,kv_heads,hd,page,dtype", [FORMS[0], FORMS[1], FORMS[4], FORMS[9]])
def test_the_same_as_every_token_by_itself(heads, kv_heads, hd, page, dtype):
    """Against the framework's own attention over the same tables, where that takes the sizes."""
    s = make([(310, [3, 70, 21]), (128, [1, 1])], heads, kv_heads, hd, page, dtype, stale=0.0)
    s["block_table"].clamp_(max=s["k_cache"].shape[0] - 1)
    got = check(s)
    other = K().attention_decode(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["token_req"], s["positions"], hd ** -0.5)
    close = 2.0 ** -6 if dtype == torch.bfloat16 else 2.0 ** -16
    assert bool(((got.float() - other.float()).abs() <= close * (1 + other.float().abs())).all())


@pytest.mark.parametrize("heads,kv_heads,hd,page,dtype", [FORMS[0], FORMS[2], FORMS[4], FORMS[8]])
def test_rows_of_no_group_are_left_alone(heads, kv_heads, hd, page, dtype):
    s = make([(100, [3, 70, 21, 9, 5])], heads, kv_heads, hd, page, dtype)
    whole = check(s)
    s["group_start"], s["prefix_lens"] = ints([1, 1, 3]), ints([64, 100])
    out = torch.full_like(s["q"], 7.0)
    got = call(s, out=out)
    assert got is out and bool((out[0] == 7).all()) and bool((out[3:] == 7).all())
    assert bool(((out[1:3].float() - whole[1:3].float()).abs() <= 2.0 ** -6).all())
    s["group_start"], s["prefix_lens"] = ints([0]), ints([])
    assert bool((call(s, out=torch.full_like(s["q"], 3.0)) == 3).all())


@pytest.mark.parametrize("heads,kv_heads,hd,page,dtype", [FORMS[0], FORMS[2], FORMS[4], FORMS[8], FORMS[13]])
def test_what_is_not_there_has_no_keys(heads, kv_heads, hd, page, dtype):
    """A request that the table does not have, positions past the table's columns, pages outside of the pool: the keys that are
    there are what counts."""
    s = make([(page, [3, page, 2])], heads, kv_heads, hd, page, dtype, stale=0.0)
    want = check(s)
    s["token_req"][2] = 99
    got = call(s)
    # the prefix is read through the first token's row, the own part through a row that is not there
    alone = {**s, "q": s["q"][2:], "token_req": ints([0]), "positions": ints([page - 1]), "group_start": ints([0, 1])}
    assert bool(((got[2:].float() - call(alone).float()).abs() <= 2.0 ** -6).all())
    assert bool(((got[:2].float() - want[:2].float()).abs() <= 2.0 ** -6).all())
    s["token_req"].copy_(ints([-5, 99, 1 << 30]))
    assert bool((call(s) == 0).all())
    s["token_req"].copy_(ints([0, 1, 2]))
    s["block_table"].fill_(-1)
    assert bool((call(s) == 0).all())
    s["block_table"].fill_(1 << 30)
    assert bool((call(s) == 0).all())


@pytest.mark.parametrize("heads,kv_heads,hd,page,dtype", [FORMS[0], FORMS[2], FORMS[4], FORMS[8]])
def test_groups_that_are_no_groups(heads, kv_heads, hd, page, dtype):
    """Starts that descend or lie outside of the batch, prefixes longer than the table: nothing is read or written elsewhere."""
    s = make([(page, [3, page, 2])], heads, kv_heads, hd, page, dtype, stale=0.0)
    guard = torch.full((5, *s["q"].shape[1:]), 9.0, dtype=dtype, device="cuda")
    for starts, prefixes in (([3, 0, 2], [page, page]), ([-100, 100], [1 << 30]), ([0, 1 << 30], [-7]), ([2, 1, 0, 3], [5, 5, 5])):
        s["group_start"], s["prefix_lens"] = ints(starts), ints(prefixes)
        call(s, out=guard[1:4], max_prefix=page, max_context=4 * page)
        assert bool((guard[0] == 9).all()) and bool((guard[4] == 9).all())
    torch.cuda.synchronize()
    K().check_kernel_errors()


def test_nan_in_a_query_or_a_key_stays_with_its_rows():
    for heads, kv_heads, hd, page, dtype in (FORMS[0], FORMS[8]):
        s = make([(200, [3, 70, 21])], heads, kv_heads, hd, page, dtype, stale=0.0)
        want = call(s)
        s["q"][1, 2] = float("nan")
        got = call(s)
        assert bool(got[1, 2].isnan().all())
        got[1, 2] = want[1, 2]
        assert torch.equal(got, want)


@pytest.mark.parametrize("heads,kv_heads,hd,page,dtype", [FORMS[0], FORMS[2], FORMS[8]])
def test_row_strides_streams_and_graphs(heads, kv_heads, hd, page, dtype):
    s = make([(600, [3, 70, 21, 300]), (100, [2])], heads, kv_heads, hd, page, dtype)
    want = check(s)
    for more in (8, 3):                                                          # queries as a view of a wider projection
        wide = torch.zeros((5, heads * hd + more), dtype=dtype, device="cuda")
        wide[:, more:] = s["q"].view(5, -1)
        t = {**s, "q": wide[:, more:].view(5, heads, hd)}
        assert bool(((call(t).float() - want.float()).abs() <= 2.0 ** -6).all())
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append(call(s, max_prefix=600, max_context=900))
    for st in streams:
        torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(got[0], want) and torch.equal(got[1], want)
    graph, out = torch.cuda.CUDAGraph(), torch.zeros_like(s["q"])
    with torch.cuda.graph(graph):
        call(s, out=out, max_prefix=600, max_context=900)
    graph.replay()
    assert torch.equal(out, want)
    s["positions"].sub_(1)                                                        # a step back: the graph reads the present state
    s["prefix_lens"].copy_(ints([511, 100]))
    graph.replay()
    torch.cuda.synchronize()
    assert bool(((out.float() - check(s).float()).abs() <= 2.0 ** -6).all())


@pytest.mark.parametrize("heads,kv_heads,hd,page,dtype", [FORMS[0], FORMS[2], FORMS[8], FORMS[13]])
def test_one_page_of_the_prefix_is_not_there(heads, kv_heads, hd, page, dtype):
    """Keys of a page outside of the pool are left out, its neighbours within a tile are not."""
    s = make([(5 * page, [3, 70])], heads, kv_heads, hd, page, dtype, stale=0.0)
    s["block_table"][:, 2] = s["k_cache"].shape[0]
    got = call(s)
    # the same without that page: a table that skips it, positions a page earlier
    t = {**s, "block_table": torch.cat([s["block_table"][:, :2], s["block_table"][:, 3:]], 1).contiguous(),
         "positions": s["positions"] - page, "prefix_lens": s["prefix_lens"] - page}
    want, size, reach = shared_attention(*(t[n].cpu() for n in ("q", "k_cache", "v_cache", "block_table", "token_req", "positions")), hd ** -0.5)
    assert bool(((got.cpu().double() - want).abs() <= shared_attention_error(want, size, reach, hd, dtype)).all())
    K().check_kernel_errors()


@pytest.mark.parametrize("groups", [33, 70])
def test_many_groups(groups):
    """More groups than a warp has lanes, some of them empty."""
    heads, kv_heads, hd, page, dtype = FORMS[0]
    check(make([((37 * i) % 150, [1 + (i + r) % 5 for r in range(i % 3)]) for i in range(groups)], heads, kv_heads, hd, page, dtype))


def test_the_binding_and_the_ordinary_way_are_the_same_call():
    k = K()
    for heads, kv_heads, hd, page, dtype in (FORMS[0], FORMS[8]):
        s = make([(300, [1, 5, 64, 200]), (0, [7])], heads, kv_heads, hd, page, dtype)
        launched = k.launch_count
        got = call(s)
        assert k.launch_count == launched + 3
        again = call(s, out=torch.empty_like(s["q"]))                             # (an output of the caller's goes the ordinary way)
        assert torch.equal(again, got) and k.launch_count == launched + 6
