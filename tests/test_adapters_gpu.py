"""What the adapters of many requests add to a shared projection (`adapters.cu`) against 64 bits."""
import pytest
import torch

from serving_util import adapters, adapters_error

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]


def K():
    from logssms_b200.ops import kernels
    return kernels


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def make(rows, width, features, n, rank, dtype, index, seed=0):
    g = torch.Generator().manual_seed(seed + rows * 7 + width)
    r = lambda *s: torch.randn(s, generator=g)          # noqa: E731
    return {"y": r(rows, features).to(dtype).cuda(), "x": r(rows, width).to(dtype).cuda(),
            "a": (r(n, rank, width) * max(width, 1) ** -0.5).to(dtype).cuda(), "b": r(n, features, rank).to(dtype).cuda(),
            "index": ints(index), "scales": (torch.rand(n, generator=g) * 2 - 0.7).cuda()}


def check(s, ranks=None, **kw):
    want, size = adapters(*(s[k].cpu() for k in ("y", "x", "a", "b", "index", "scales")), None if ranks is None else ranks.cpu())
    error = adapters_error(s["y"].cpu(), want, size, s["x"].shape[1], s["a"].shape[1], s["y"].dtype)
    got = K().add_adapters(s["y"], s["x"], s["a"], s["b"], s["index"], s["scales"], ranks=ranks, **kw)
    assert got.dtype == s["y"].dtype and got.shape == s["y"].shape
    assert bool(((got.cpu().double() - want).abs() <= error).all())
    without = [t for t, i in enumerate(s["index"].tolist()) if not 0 <= i < s["a"].shape[0]]
    if without:
        assert torch.equal(got[without], s["y"][without])
    K().check_kernel_errors()
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width,features,rank", [(1, 64, 64, 8), (1, 1024, 4096, 16), (2, 8, 8, 1), (3, 1, 5, 3), (5, 130, 70, 13),
                                                      (7, 512, 264, 64), (9, 1003, 97, 24), (4, 2048, 1280, 128), (2, 96, 40, 200)])
def test_few_rows_each_with_its_own(dtype, rows, width, features, rank):
    check(make(rows, width, features, rows + 1, rank, dtype, [(3 * t) % (rows + 1) for t in range(rows)]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [8, 16, 17, 33, 64, 127, 129, 200, 300])
def test_decoding_rows_in_any_order_some_without_an_adapter(dtype, rows):
    g = torch.Generator().manual_seed(rows)
    index = torch.randint(-2, 9, (rows,), generator=g).tolist()          # 8 is none of the adapters either
    check(make(rows, 320, 200, 8, 16, dtype, index))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width,features,rank", [(700, 256, 384, 16), (1500, 192, 136, 64), (1025, 512, 128, 40), (640, 72, 1000, 8),
                                                      (600, 200, 264, 128), (700, 250, 333, 13), (900, 328, 1032, 72), (520, 64, 128, 200),
                                                      (1100, 131, 1001, 96), (400, 65, 129, 64), (2100, 1003, 515, 5)])
def test_prompts_one_behind_the_other(dtype, rows, width, features, rank):
    """Portions whose ends lie within tiles, one of a single token, one without an adapter."""
    cuts = [0, rows // 5, rows // 5 + 1, rows // 2 + 3, rows - 130, rows]
    index = [0] * rows
    for i, (lo, hi) in enumerate(zip(cuts, cuts[1:])):
        index[lo:hi] = [(2, 0, -1, 3, 1)[i]] * (hi - lo)
    check(make(rows, width, features, 4, rank, dtype, index))


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_step_with_decoding_rows_and_a_prompt(dtype):
    g = torch.Generator().manual_seed(5)
    index = torch.randint(-1, 40, (70,), generator=g).tolist() + [7] * 530 + [11] * 100
    check(make(700, 256, 320, 40, 16, dtype, index))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [6, 600])
def test_ranks_that_differ_and_what_lies_behind_them(dtype, rows):
    s = make(rows, 160, 144, 5, 24, dtype, [t * 5 // rows for t in range(rows)])
    ranks = ints([24, 8, 0, 5, 99])
    for i, r in enumerate([24, 8, 0, 5, 24]):                           # padding may hold anything
        s["a"][i, r:], s["b"][i, :, r:] = float("nan"), float("inf")
    clean = {**s, "a": s["a"].nan_to_num(0.0), "b": s["b"].nan_to_num(0.0, posinf=0.0)}
    got = check(clean, ranks)
    again = K().add_adapters(s["y"], s["x"], s["a"], s["b"], s["index"], s["scales"], ranks=ranks)
    assert torch.equal(again, got)


@pytest.mark.parametrize("rows", [4, 400])
@pytest.mark.parametrize("dtype", DTYPES)
def test_one_rows_nan_is_its_own(dtype, rows):
    """NaN and infinities in one row, in one adapter and in a row without an adapter reach nobody else."""
    s = make(rows, 128, 96, 3, 16, dtype, [t % 2 if t % 4 != 3 else -1 for t in range(rows)])
    fine = K().add_adapters(s["y"], s["x"], s["a"], s["b"], s["index"], s["scales"])
    s["x"][3], s["x"][2], s["a"][2], s["b"][2] = float("nan"), float("inf"), float("nan"), float("nan")
    got = K().add_adapters(s["y"], s["x"], s["a"], s["b"], s["index"], s["scales"])
    keep = [t for t in range(rows) if t != 2]
    assert torch.equal(got[keep], fine[keep])
    assert not bool(got[2].isfinite().any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [3, 300])
def test_strides_views_in_place_and_odd_places(dtype, rows):
    base = make(rows, 264, 104, 3, 16, dtype, [t % 4 - 1 for t in range(rows)])
    want = check(base)
    wide = torch.zeros((rows, 400), dtype=dtype, device="cuda")
    s = dict(base)
    for shift in (0, 1, 8):
        s["y"] = wide[:, shift:shift + 104]                              # a part of a wider product's columns
        s["y"].copy_(base["y"])
        x = torch.zeros((rows, 300), dtype=dtype, device="cuda")[:, shift:shift + 264]
        x.copy_(base["x"])
        a = torch.zeros((3, 20, 280), dtype=dtype, device="cuda")[:, 2:18, shift:shift + 264]
        a.copy_(base["a"])
        b = torch.zeros((3, 110, 32), dtype=dtype, device="cuda")[:, 3:107, shift:shift + 16]
        b.copy_(base["b"])
        s.update(x=x, a=a, b=b)
        check(s)
        before = wide.clone()
        got = K().add_adapters(s["y"], x, a, b, s["index"], s["scales"], out=s["y"])
        assert got is s["y"]
        error = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -16     # (another order of the sums may round the other way)
        assert bool(((got.float() - want.float()).abs() <= error * (1 + want.float().abs())).all())
        before[:, shift:shift + 104] = got
        assert torch.equal(wide, before)


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_same_call_gives_the_same_bits(dtype):
    for rows in (5, 500):
        s = make(rows, 512, 256, 4, 16, dtype, [t % 4 for t in range(rows)])
        first = K().add_adapters(s["y"], s["x"], s["a"], s["b"], s["index"], s["scales"])
        for _ in range(5):
            assert torch.equal(K().add_adapters(s["y"], s["x"], s["a"], s["b"], s["index"], s["scales"]), first)


@pytest.mark.parametrize("rows", [5, 500])
def test_streams_and_graphs(rows):
    s = make(rows, 512, 256, 4, 16, torch.bfloat16, [t % 4 for t in range(rows)])
    want = check(s)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for st in streams:                                                   # two calls at once
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append(K().add_adapters(s["y"], s["x"], s["a"], s["b"], s["index"], s["scales"]))
    for st in streams:
        torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(got[0], want) and torch.equal(got[1], want)
    graph, out = torch.cuda.CUDAGraph(), torch.zeros_like(s["y"])
    with torch.cuda.graph(graph):
        K().add_adapters(s["y"], s["x"], s["a"], s["b"], s["index"], s["scales"], out=out)
    graph.replay()
    assert torch.equal(out, want)
    s["index"].copy_(s["index"].flip(0) - 1)                             # other requests in the same places
    graph.replay()
    assert torch.equal(out, check(s))


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty_sizes(dtype):
    assert check(make(4, 0, 24, 2, 8, dtype, [0, 1, 0, -1])).shape == (4, 24)
    assert check(make(4, 16, 24, 2, 0, dtype, [0, 1, 0, -1])).shape == (4, 24)
    assert check(make(4, 16, 24, 0, 8, dtype, [0, 1, 0, -1])).shape == (4, 24)
    assert check(make(0, 16, 24, 2, 8, dtype, [])).shape == (0, 24)
    assert check(make(4, 16, 0, 2, 8, dtype, [0, 1, 0, -1])).shape == (4, 0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ranks_past_what_the_tensor_core_forms_take(dtype):
    check(make(6, 96, 80, 3, 300, dtype, [0, 1, 2, -1, 1, 0]))
    check(make(450, 64, 40, 2, 264, dtype, [0] * 200 + [1] * 250))


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_keep_their_sign(dtype):
    """A short sum that is infinite has no remainder to add: y becomes that infinity and no NaN."""
    for rows in (3, 400):
        s = make(rows, 64, 48, 1, 16, dtype, [0] * rows)
        s["x"][1] = 0.0
        s["x"][1, 0] = float("inf")
        s["a"][0, :, 0], s["b"][0] = 1.0, s["b"][0].abs() + 0.5
        s["scales"][0] = 1.0
        got = K().add_adapters(s["y"], s["x"], s["a"], s["b"], s["index"], s["scales"])
        assert bool((got[1] == float("inf")).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [5, 500])
def test_the_binding_and_the_ordinary_way_are_the_same_call(dtype, rows):
    s = make(rows, 256, 136, 4, 16, dtype, [t % 5 - 1 for t in range(rows)])
    got = K().add_adapters(s["y"], s["x"], s["a"], s["b"], s["index"], s["scales"])
    again = K().add_adapters(s["y"], s["x"], s["a"], s["b"], s["index"], s["scales"], out=torch.empty_like(s["y"]))
    assert torch.equal(got, again)


def test_without_scales_and_ranks_and_a_single_adapter():
    for rows in (2, 400):
        s = make(rows, 64, 64, 1, 8, torch.bfloat16, [0] * rows)
        s["scales"].fill_(1.0)
        got = check(s)
        assert torch.equal(got, K().add_adapters(s["y"], s["x"], s["a"], s["b"], s["index"]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width,features,n,rank", [(64, 96, 72, 7, 16), (390, 256, 200, 9, 16), (777, 131, 97, 30, 24), (1500, 264, 328, 5, 64),
                                                        (900, 328, 130, 700, 40), (1300, 128, 264, 8, 128), (400, 64, 80, 5000, 8), (500, 72, 66, 6, 260)])
def test_many_rows_in_any_order(dtype, rows, width, features, n, rank):
    """Rows in random order; the same in two captures of a graph; a part of a wider matrix, in place; the same bits every time."""
    g = torch.Generator().manual_seed(rows)
    index = torch.randint(-1, n, (rows,), generator=g).tolist()
    if rows == 1500:
        index[256:640] = [3] * 384                                       # some rows as they come in between
    s = make(rows, width, features, n, rank, dtype, index)
    ranks = torch.randint(0, rank + 1, (n,), generator=g).to(torch.int32).cuda()
    want = check(s, ranks)
    call = lambda out=None: K().add_adapters(s["y"], s["x"], s["a"], s["b"], s["index"], s["scales"], ranks=ranks, out=out)       # noqa: E731
    assert torch.equal(call(), want)
    wide = torch.full((rows, features + 24), 7.0, dtype=dtype, device="cuda")
    base = s["y"]
    s["y"] = wide[:, 8:8 + features]
    s["y"].copy_(base)
    call(s["y"])
    assert torch.equal(s["y"], want) or bool(((s["y"].double() - want.double()).abs() <= 2.0 ** -7 * (1 + want.double().abs())).all())
    assert bool((wide[:, :8] == 7).all()) and bool((wide[:, 8 + features:] == 7).all())
    s["y"] = base
    graph, out = torch.cuda.CUDAGraph(), torch.zeros_like(base)
    with torch.cuda.graph(graph):
        call(out)
    graph.replay()
    assert torch.equal(out, want)
    s["index"].copy_(s["index"].flip(0))
    graph.replay()
    assert torch.equal(out, check(s, ranks))


def test_launches_are_counted_as_they_are():
    from torch.profiler import ProfilerActivity, profile
    for rows, n, rank, dtype in ((4, 3, 8, torch.bfloat16), (400, 3, 8, torch.bfloat16), (400, 1, 8, torch.bfloat16), (70, 3, 8, torch.float32),
                                 (12, 9, 8, torch.float32), (12, 8, 8, torch.float32), (5, 2, 264, torch.bfloat16)):
        s = make(rows, 64, 64, n, rank, dtype, [t % n for t in range(rows)])
        call = lambda: K().add_adapters(s["y"], s["x"], s["a"], s["b"], s["index"], s["scales"])         # noqa: E731
        call()
        before = K().launch_count
        with profile(activities=[ProfilerActivity.CUDA]) as p:
            call()
            torch.cuda.synchronize()
        ran = sum(e.count for e in p.key_averages() if "adapter_" in e.key)
        assert K().launch_count - before == ran
