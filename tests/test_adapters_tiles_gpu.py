"""Adapters of many rows (`adapters_tiles.cuh`): what the short prompts of test_adapters_gpu.py do not reach."""
import pytest
import torch

from serving_util import adapters_error
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


# ------------------------------------------------------------------ tiles of 128 rows by clusters of 4, of 2 and by single CTAs
def in_64_bits(s, ranks):
    """(out, sum of the sizes of all products), adapter by adapter on the GPU."""
    out, size = s["y"].double().clone(), torch.zeros(s["y"].shape, dtype=torch.float64, device="cuda")
    for i in range(s["a"].shape[0]):
        rows = (s["index"] == i).nonzero()[:, 0]
        r = s["a"].shape[1] if ranks is None else max(0, min(int(ranks[i]), s["a"].shape[1]))
        x, a, b, scale = s["x"][rows].double(), s["a"][i, :r].double(), s["b"][i, :, :r].double(), float(s["scales"][i])
        out[rows] += scale * ((x @ a.t()) @ b.t())
        size[rows] = abs(scale) * ((x.abs() @ a.abs().t()) @ b.abs().t())
    return out, size


def check(s, ranks=None, out=None):
    want, size = in_64_bits(s, ranks)
    error = adapters_error(s["y"], want, size, s["x"].shape[1], s["a"].shape[1], s["y"].dtype)
    got = K().add_adapters(s["y"], s["x"], s["a"], s["b"], s["index"], s["scales"], ranks=ranks, out=out)
    assert bool(((got.double() - want).abs() <= error).all())
    K().check_kernel_errors()
    return got


def indices(rows, n, order):
    if order == "random":
        return torch.randint(-1, n, (rows,), generator=torch.Generator().manual_seed(rows)).tolist()
    index, cuts = [0] * rows, [0, 1, rows // 7, rows // 3 + 5, rows // 3 + 6, rows // 2 + 77, rows - 129, rows]
    for i, (lo, hi) in enumerate(zip(cuts, cuts[1:])):
        index[lo:hi] = [(2, 0, -1, 3, 1, 4, 2)[i]] * (hi - lo)
    return index


# Rows that make 19, 38 and 76 tiles, the last one in part: 8 CTAs have a tile up to 18 tiles, 4 up to 37, 2 up to 74, one from then on.
@pytest.mark.parametrize("rows", [2401, 4801, 9613])
@pytest.mark.parametrize("order", ["portions", "random"])
@pytest.mark.parametrize("width,features,rank", [(136, 264, 24), (64, 520, 64), (200, 136, 100), (131, 257, 24), (77, 391, 61), (2048, 1544, 64),
                                                 (1536, 648, 128), (1003, 1431, 13)])
def test_every_size_of_a_tiles_cluster(rows, order, width, features, rank):
    s = make(rows, width, features, 9, rank, torch.bfloat16, indices(rows, 9, order))
    ranks = torch.tensor([rank, 1, rank - 1, rank // 2, rank, 0, rank, 5, rank], dtype=torch.int32, device="cuda")
    got = check(s, ranks)
    assert torch.equal(check(s, ranks), got)
    check(s)
    y = s["y"].clone()                                   # in place
    assert torch.equal(K().add_adapters(y, s["x"], s["a"], s["b"], s["index"], s["scales"], ranks=ranks, out=y), got) and torch.equal(y, got)
    graph, held = torch.cuda.CUDAGraph(), torch.zeros_like(s["y"])
    with torch.cuda.graph(graph):
        K().add_adapters(s["y"], s["x"], s["a"], s["b"], s["index"], s["scales"], ranks=ranks, out=held)
    s["index"].copy_(s["index"].flip(0))
    graph.replay()
    assert torch.equal(held, check(s, ranks))


@pytest.mark.parametrize("rows", [2401, 4801, 9613])
@pytest.mark.parametrize("features,rank", [(264, 24), (257, 24), (264, 100)])
def test_numbers_behind_a_rank_and_of_other_rows_in_every_cluster(rows, features, rank):
    s = make(rows, 136, features, 5, rank, torch.bfloat16, indices(rows, 5, "portions"))
    ranks = torch.tensor([rank, 7, rank - 3, 0, 16], dtype=torch.int32, device="cuda")
    fine = check(s, ranks)
    for i, r in enumerate(ranks.tolist()):
        s["a"][i, r:], s["b"][i, :, r:] = float("nan"), float("inf")
    s["x"][rows // 7 + 3] = float("nan")                 # a row without an adapter
    assert torch.equal(K().add_adapters(s["y"], s["x"], s["a"], s["b"], s["index"], s["scales"], ranks=ranks), fine)
    bad = rows // 2
    s["x"][bad] = float("nan")
    got = K().add_adapters(s["y"], s["x"], s["a"], s["b"], s["index"], s["scales"], ranks=ranks)
    assert not bool(got[bad].isfinite().any())
    got[bad] = fine[bad]
    assert torch.equal(got, fine)


@pytest.mark.parametrize("rows", [3, 60, 300, 700])
def test_a_part_of_a_wider_matrix_in_float32_to_its_own_bound(rows):
    for shift in (0, 1, 8):
        s = make(rows, 264, 104, 3, 16, torch.float32, [t % 4 - 1 for t in range(rows)])
        wide = torch.full((rows, 400), 7.0, device="cuda")
        kept = s["y"]
        s["y"] = wide[:, shift:shift + 104]
        s["y"].copy_(kept)
        want, size = in_64_bits({**s, "y": kept}, None)
        got = K().add_adapters(s["y"], s["x"], s["a"], s["b"], s["index"], s["scales"], out=s["y"])
        assert got is s["y"] and bool(((got.double() - want).abs() <= adapters_error(kept, want, size, 264, 16, torch.float32)).all())
        assert bool((wide[:, :shift] == 7).all()) and bool((wide[:, shift + 104:] == 7).all())
