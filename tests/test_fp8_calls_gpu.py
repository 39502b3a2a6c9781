"""How the 8-bit operators are called: through the binding and past it, what they allocate and
what they refuse."""
from ctypes import c_float, c_int, c_long, c_void_p
from types import SimpleNamespace

import pytest
import torch

from fp8_util import make_rows, make_weight
from test_fp8_linear_gpu import check_linear, check_swiglu
from tiny import TINY, make_model_dir

pytestmark = pytest.mark.gpu


def K():
    from logssms_b200.ops import kernels
    return kernels


def operands(m, n, k, seed=0):
    g = torch.Generator().manual_seed(1000 * m + n + k + seed)
    kk = K()
    return kk.Fp8Rows(*make_rows(m, k, g)), kk.Fp8Weight(*make_weight(n, k, g), settled=True), kk.Fp8Weight(*make_weight(n, k, g), settled=True)


def same(a, b):
    return a.shape == b.shape and a.stride() == b.stride() and a.dtype == b.dtype and torch.equal(
        a.view(torch.uint8) if a.dtype == torch.float8_e4m3fn else a, b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b)


@pytest.fixture
def past_the_binding(monkeypatch):
    """A context in which every call goes the ordinary way, as a profiled engine's do."""
    k = K()

    def switch():
        none = lambda *args: None     # noqa: E731
        monkeypatch.setattr(k, "_fp8_binding", SimpleNamespace(norm=none, quantize=none, linear=none, swiglu=none, error_word=none))
    return switch


@pytest.mark.parametrize("width", [1, 100, 128, 500, 1003])
def test_whole_rows_are_allocated(width, past_the_binding):
    """The gated product writes 16 bytes at a time: what fills up the last row belongs to the tensor as well."""
    k = K()
    x, w, u = operands(3, width, 256)
    source = torch.randn(3, width, device="cuda")
    for way in range(2):
        if way:
            past_the_binding()
        for got in (k.linear_swiglu_fp8(x, w, u), k.quantize_rows_fp8(source), k.quantize_weight_fp8(source),
                    k.add_rmsnorm_fp8(source, torch.ones(width, device="cuda"), 1e-5)[0]):
            pitch = (width + 15) // 16 * 16
            assert got.values.shape == (3, width) and got.values.stride() == (pitch, 1)
            assert got.values.untyped_storage().nbytes() >= 3 * pitch


@pytest.fixture
def no_words(monkeypatch):
    """As before the first product of the process: no device has an error word, and the binding knows of none."""
    k = K()
    here = torch.cuda.current_device()
    k._fp8_calls().error_word(here, 0)
    with monkeypatch.context() as m:
        m.setattr(k, "_gemm_error", {})
        yield here
    k._fp8_calls().error_word(here, k.error_word(torch.device("cuda", here)).data_ptr())


def test_only_the_device_in_use_gets_an_error_word(no_words, monkeypatch):
    k = K()
    asked, make = [], k.error_word

    def spy(device):
        asked.append(torch.device(device).index)
        assert asked[-1] == no_words, "a device that the caller does not use"
        return make(device)
    monkeypatch.setattr(k, "error_word", spy)
    monkeypatch.setattr(k, "_fp8_binding", None)
    monkeypatch.setattr(torch.cuda, "device_count", lambda: 3)
    x = torch.randn(4, 256, device="cuda")
    rows = k.quantize_rows_fp8(x)
    k.add_rmsnorm_fp8(x, torch.ones(256, device="cuda"), 1e-5)
    assert asked == []                                     # nothing of these waits
    w = k.quantize_weight_fp8(x)
    first = k.linear_fp8(rows, w)
    assert set(asked) == {no_words} and list(k._gemm_error) == [torch.device("cuda", no_words)]
    count = len(asked)
    assert torch.equal(k.linear_fp8(rows, w), first) and k.linear_swiglu_fp8(rows, w, w).shape == (4, 4)
    assert len(asked) == count                             # from then on the binding has it
    k.check_kernel_errors()


def test_a_first_product_inside_a_capture_is_refused(no_words):
    """Its error word would be cleared by every replay."""
    k = K()
    x = torch.randn(4, 256, device="cuda")
    rows, w = k.quantize_rows_fp8(x), k.quantize_weight_fp8(x)
    torch.cuda.synchronize()
    kept = torch.zeros(1, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept.add_(1)
        for call in (lambda: k.linear_fp8(rows, w), lambda: k.linear_swiglu_fp8(rows, w, w)):
            with pytest.raises(k.KernelError, match="before a capture"):
                call()
    assert k._gemm_error == {}
    want = k.linear_fp8(rows, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = k.linear_fp8(rows, w)
    graph.replay()
    assert torch.equal(got, want)
    k.check_kernel_errors()


@pytest.mark.parametrize("yes,no", [(1, 0), ("yes", ""), ([0], None)])
def test_what_is_true_counts_as_true(yes, no, past_the_binding):
    """Flags of any type, through the binding as past it."""
    k = K()
    x, r = torch.randn(4, 64, device="cuda"), torch.randn(4, 64, device="cuda")
    weight = torch.ones(64, device="cuda")
    xq, w, u = operands(4, 64, 256)
    for way in range(2):
        if way:
            past_the_binding()
        kept = r.clone()
        assert k.add_rmsnorm_fp8(x, weight, 1e-5, kept, want_residual=yes, in_place=yes)[1] is kept
        assert torch.equal(kept, r + x)
        kept = r.clone()
        new = k.add_rmsnorm_fp8(x, weight, 1e-5, kept, want_residual=yes, in_place=no)[1]
        assert new is not kept and torch.equal(kept, r) and torch.equal(new, r + x)
        assert k.add_rmsnorm_fp8(x, weight, 1e-5, kept, want_residual=no)[1] is None and torch.equal(kept, r)
        for settled in (yes, no):
            a, b = k.Fp8Weight(w.values, w.scales, settled), k.Fp8Weight(u.values, u.scales, settled)
            check_linear(xq, a)
            check_swiglu(xq, a, b, 1.0)


def test_sizes_near_the_end_of_32_bits_are_refused():
    """By the launchers, before anything is launched: within 2^16 of 2^31 the kernels' own places would leave 32 bits."""
    from logssms_b200.ops import build
    p, l, i, f = c_void_p, c_long, c_int, c_float                     # noqa: E741
    at, big, pitch = 1 << 20, (1 << 31) - 100, (1 << 31) - (1 << 16)
    linear = build.load("fp8_linear").lb_linear_fp8
    linear.argtypes = [p, l, p, l, l, p, l, p, l, l, p, p, l, i, i, i, f, i, i, i, p, p]
    swiglu = build.load("fp8_linear").lb_linear_swiglu_fp8
    swiglu.argtypes = [p, l, p, l, l, p, p, l, p, p, l, l, p, l, p, l, l, i, i, i, f, i, i, p, p]
    for sizes in ((big, 16, 16), (16, big, 16), (16, 16, big)):
        for form in range(4):
            assert linear(at, pitch, at, 1, 1, at, pitch, at, 1, 1, None, at, 16, *sizes, 1.0, 0, 0, form, None, None) == -3
            assert swiglu(at, pitch, at, 1, 1, at, at, pitch, at, at, 1, 1, at, pitch, at, 1, 1, *sizes, 1.0, 0, form, None, None) == -3
    quantize = build.load("fp8_rows").lb_quantize_fp8
    quantize.argtypes = [p, l, p, l, p, l, l, l, i, i, i, p]
    for block_rows in (1, 128):
        for width in (big, big + 4):                       # by values, by pieces of 8
            assert quantize(at, 1 << 31, at, 1 << 31, at, 1, 1, 1, width, block_rows, 0, None) == -3
    norm = build.load("fp8_rows").lb_add_rmsnorm_fp8
    norm.argtypes = [p, l, p, l, p, l, p, l, p, p, l, p, l, l, i, i, f, f, f, f, i, p]
    assert norm(at, 1 << 31, None, 0, None, 0, None, 0, at, at, 1 << 31, at, 1, 1, 1, big, 1e-5, 1.0, 1.0, 1.0, 0, None) == -3


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,width", [(1, 40), (5, 301), (130, 1024)])
def test_both_ways_give_the_same_bytes(rows, width, dtype, past_the_binding):
    k = K()
    g = torch.Generator().manual_seed(rows)
    x, o, r = (torch.randn(rows, width, generator=g).to(dtype).cuda() for _ in range(3))
    weight = torch.rand(width, generator=g).cuda()
    xq, w, u = operands(rows, 200, width)
    bias = torch.randn(200, generator=g).cuda()

    def everything():
        outs = []
        for kw in ({}, {"other": o, "in_scales": (0.5, 0.25)}, {"other": o, "want_residual": False}, {"in_place": False, "out_scale": 2.0}):
            kept = r.clone()
            made, new = k.add_rmsnorm_fp8(x, weight, 1e-5, kept, **kw)
            outs += [made.values, made.scales, kept, kept if new is None else new]
        made, new = k.add_rmsnorm_fp8(x, weight, 1e-5)
        outs += [made.values, made.scales, new]
        for made in (k.quantize_rows_fp8(x), k.quantize_weight_fp8(x), k.linear_swiglu_fp8(xq, w, u, 0.9)):
            outs += [made.values, made.scales]
        return outs + [k.linear_fp8(xq, w), k.linear_fp8(xq, w, bias, out_scale=1.5, out_dtype=torch.float32)]
    first = everything()
    past_the_binding()
    before = k.launch_count
    second = everything()
    assert k.launch_count - before == 10
    assert all(same(a, b) for a, b in zip(first, second, strict=True))
    k.check_kernel_errors()


def test_a_profiled_engine_gives_the_same_logits(tmp_path):
    from logssms_b200.engine import Engine, StepEntry
    from logssms_b200.ops.profiler import PROFILER
    model_dir = make_model_dir(tmp_path / "m", TINY["A"], seed=4, dtype=torch.bfloat16)
    ids = torch.randint(0, 256, (60,), generator=torch.Generator().manual_seed(1)).tolist()
    got = []
    try:
        for profile in (False, True):
            engine = Engine(model_dir, "bfloat16", max_requests=2, max_seq_len=64, num_pages=4, use_graphs=False, profile=profile,
                            feed_forward_weights="float8")
            r = engine.new_request()
            got.append([engine.step([StepEntry(r, part, list(range(len(part))))]).clone() for part in (ids[:59], ids[59:])])
            if profile:
                names = " ".join(PROFILER.report()["kernels"])
                assert "lb_add_rmsnorm_fp8" in names and "lb_linear_fp8" in names and "lb_linear_swiglu_fp8" in names
    finally:
        PROFILER.disable()
    assert all(torch.equal(a, b) for a, b in zip(*got, strict=True))


@pytest.mark.parametrize("split", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("m", [1, 6, 17, 33, 64, 150])
def test_no_split_is_refused(m, split):
    """All of these fit an SM's shared memory, the plain product and the gated one."""
    k = K()
    k._FP8_FORMS["split"] = (1 if m <= 64 else 2) + 256 * split
    k.FP8_FORM = "split"
    try:
        for n, kd in ((200, 128 * 9), (257, 128 * 8 * 3 - 5), (128, 128 * 40), (300, 100)):
            x, w, u = operands(m, n, kd)
            check_linear(x, w)
            check_swiglu(x, w, u, 0.8)
    finally:
        k.FP8_FORM = "auto"
        del k._FP8_FORMS["split"]
