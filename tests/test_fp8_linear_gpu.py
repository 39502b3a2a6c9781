"""Products of 8-bit operands (`fp8_linear.cu`) against 64 bits: both ways round, split and whole, every edge of a tile."""
import pytest
import torch

from fp8_util import holds, make_rows, make_weight, product, product_error

pytestmark = pytest.mark.gpu


def K():
    from logssms_b200.ops import kernels
    return kernels


@pytest.fixture(params=["auto", "rows", "tiles", "pair"])
def form(request):
    """The form of the kernel that runs, whatever the rule would choose."""
    k = K()
    k.FP8_FORM = request.param
    yield request.param
    k.FP8_FORM = "auto"


def operands(m, n, k, seed=0, row_major=False):
    g = torch.Generator().manual_seed(1000 * m + n + k + seed)
    kk = K()
    return kk.Fp8Rows(*make_rows(m, k, g, row_major)), kk.Fp8Weight(*make_weight(n, k, g), settled=bool(seed % 2))


def check_linear(x, w, bias=None, out_scale=1.0):
    k = K()
    y, size = product(x.values, x.scales, w.values, w.scales)
    error = product_error(size, x.shape[1])
    if bias is not None:
        y, error = y + bias.double(), error + (y + bias.double()).abs() * 2.0 ** -24
    y, error = y * out_scale, (error * abs(out_scale) + (y * out_scale).abs() * 2.0 ** -24)
    got = k.linear_fp8(x, w, bias, out_scale=out_scale, out_dtype=torch.float32)
    assert got.dtype == torch.float32 and got.shape == y.shape
    assert bool(((got.double() - y).abs() <= error + y.abs() * 2.0 ** -24).all())
    half = k.linear_fp8(x, w, bias, out_scale=out_scale)
    assert half.dtype == torch.bfloat16 and torch.equal(half, got.to(torch.bfloat16))      # the same sums, rounded once
    k.check_kernel_errors()


def check_swiglu(x, gate, up, act_scale):
    k = K()
    g, g_size = product(x.values, x.scales, gate.values, gate.scales)
    u, u_size = product(x.values, x.scales, up.values, up.scales)
    g_error, u_error = product_error(g_size, x.shape[1]), product_error(u_size, x.shape[1])
    g = g * act_scale
    h = g * torch.sigmoid(g) * u
    # silu's slope is at most 1.1; its own exponential and division and the last product: 2^-24 x (the exponent's size + 6)
    error = 1.1 * act_scale * g_error * u.abs() + (g * torch.sigmoid(g)).abs() * u_error + 1.1 * act_scale * g_error * u_error \
        + h.abs() * (g.abs() + 8) * 2.0 ** -24
    got = k.linear_swiglu_fp8(x, gate, up, act_scale)
    assert got.values.stride(0) % 16 == 0
    holds(got.values, got.scales, h, error)
    k.check_kernel_errors()


# rows: one, the edges of the padded sizes 16 / 32 / 64, tiles of 128 and their remainders
ROWS = [1, 15, 16, 17, 32, 33, 64, 65, 128, 129, 300]
# features: one, a short tile, a whole one, remainders, many tiles; columns: one, less than a block, blocks, remainders, a ring that
# goes round, splits of K
SIZES = [(1, 16), (40, 100), (128, 128), (130, 1), (257, 640), (1003, 1431), (128, 4096), (3352, 330), (20000, 264)]


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("n,k", SIZES)
def test_linear(m, n, k, form):
    x, w = operands(m, n, k, seed=m % 2, row_major=m % 3 == 0)
    check_linear(x, w)
    check_linear(x, w, torch.randn(n, generator=torch.Generator().manual_seed(n)).cuda(), 0.7)


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("n,k", SIZES)
def test_swiglu(m, n, k, form):
    x, gate = operands(m, n, k, seed=m % 2, row_major=m % 3 == 0)
    _, up = operands(m, n, k, seed=m % 2 + 2)
    check_swiglu(x, gate, up, 0.9)


# a K whose scales do not fit beside the ring, long sums, prompts
@pytest.mark.parametrize("m,n,k", [(64, 70000, 3000), (64, 256, 70000), (16, 128, 140000), (700, 640, 2500), (2100, 1300, 1100)])
def test_large(m, n, k, form):
    if form == "rows" and k > 60000:
        pytest.skip("the scales of so many columns do not fit beside the ring; the rule takes another form")
    x, w = operands(m, n, k)
    check_linear(x, w)
    if n * k < 1 << 26:
        check_swiglu(x, w, operands(m, n, k, 2)[1], 1.0)


@pytest.mark.parametrize("split", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("m", [1, 6, 17, 33, 64, 150])
def test_every_split(m, split):
    """A tile's blocks over so many CTAs, whatever the rule would choose: few blocks and many each, rings that go round and rings
    that do not, shares of rows that are empty."""
    k = K()
    k._FP8_FORMS["split"] = (1 if m <= 64 else 2) + 256 * split
    k.FP8_FORM = "split"
    try:
        for n, kd in ((200, 128 * 9), (257, 128 * 8 * 3 - 5), (128, 128 * 40), (300, 100)):
            x, w = operands(m, n, kd)
            try:
                check_linear(x, w)
                check_swiglu(x, w, operands(m, n, kd, 2)[1], 0.8)
            except k.KernelError as e:
                assert "beyond the kernel's limit" in str(e)      # a ring that does not fit: the rule takes another form then
    finally:
        k.FP8_FORM = "auto"
        del k._FP8_FORMS["split"]


@pytest.mark.parametrize("parts", [2, 4])
@pytest.mark.parametrize("m,n,k", [(1, 256, 128), (300, 200, 100), (129, 257, 128 * 3), (256, 256, 128 * 4 + 5), (700, 640, 128 * 33),
                                   (257, 1003, 5001), (513, 130, 128 * 60), (4900, 1000, 128 * 9), (18900, 64, 1100)])
def test_pairs_share_a_tile(m, n, k, parts):
    """A tile's blocks over so many pairs: fewer blocks than pairs, uneven ranges, rings that go round, whole rounds of tiles in
    front, ragged rows and features."""
    kk = K()
    kk._FP8_FORMS["parts"] = 3 + 256 * parts
    kk.FP8_FORM = "parts"
    try:
        x, w = operands(m, n, k, seed=m % 2)
        check_linear(x, w)
        check_linear(x, w, torch.randn(n, generator=torch.Generator().manual_seed(n)).cuda(), 0.7)
        first = kk.linear_fp8(x, w, out_dtype=torch.float32)
        for _ in range(5):
            assert torch.equal(kk.linear_fp8(x, w, out_dtype=torch.float32), first)
    finally:
        kk.FP8_FORM = "auto"
        del kk._FP8_FORMS["parts"]


def test_every_block_has_its_own_scales(form):
    """Blocks of very different size: a scale that met a neighbour's block would be off by its factor."""
    k = K()
    g = torch.Generator().manual_seed(5)
    for m in (5, 40, 200):
        x, w = torch.randn(m, 700, generator=g), torch.randn(500, 700, generator=g)
        for b in range(6):
            x[:, 128 * b:128 * (b + 1)] *= 10.0 ** (b - 3) * torch.exp(torch.randn(m, 1, generator=g))
            w[:, 128 * b:128 * (b + 1)] *= 10.0 ** (2 - b)
        for r in range(4):
            w[128 * r:128 * (r + 1)] *= 5.0 ** r
        xq, wq = k.quantize_rows_fp8(x.cuda()), k.quantize_weight_fp8(w.cuda())
        torch.cuda.synchronize()
        check_linear(xq, wq)
        check_swiglu(xq, wq, wq, 1e-3)


def test_the_order_of_sums_is_fixed(form):
    k = K()
    x, w = operands(24, 640, 4096)
    first = k.linear_fp8(x, w, out_dtype=torch.float32)
    for _ in range(20):
        assert torch.equal(k.linear_fp8(x, w, out_dtype=torch.float32), first)


@pytest.mark.parametrize("m", [3, 100])
def test_zeros_infinities_nan_and_extreme_scales(m):
    k = K()
    x, w = operands(m, 200, 300)
    xs = x.scales.clone()
    xs[0, 1], xs[1, 0], xs[2, 2] = float("nan"), 0.0, float("inf")
    got = k.linear_fp8(k.Fp8Rows(x.values, xs), w, out_dtype=torch.float32)
    assert bool(torch.isnan(got[0]).all()) and bool(torch.isfinite(got[1]).all())
    assert bool((~torch.isfinite(got[2])).all())           # infinite, or NaN where infinities of both signs meet
    if m > 3:
        assert torch.equal(got[3:], k.linear_fp8(x, w, out_dtype=torch.float32)[3:])
    # scales whose product is beyond 32 bits over values that are zero: the sum is zero, not NaN
    zeros = torch.zeros_like(x.values.view(torch.uint8)).contiguous()
    pad = torch.zeros(m, 304, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :300]
    assert zeros.shape == pad.shape
    big = k.Fp8Weight(w.values, torch.full_like(w.scales, 1e30))
    got = k.linear_fp8(k.Fp8Rows(pad, torch.full_like(x.scales, 1e30)), big, out_dtype=torch.float32)
    assert bool((got == 0).all())


def test_empty_strided_and_other_streams():
    k = K()
    x, w = operands(20, 96, 256)
    assert k.linear_fp8(k.Fp8Rows(x.values[:0], x.scales[:0]), w).shape == (0, 96)
    assert k.linear_swiglu_fp8(k.Fp8Rows(x.values[:0], x.scales[:0]), w, w).shape == (0, 96)
    none = k.linear_fp8(x, k.Fp8Weight(w.values[:0], w.scales[:0]))
    assert none.shape == (20, 0)
    # every second row, and the second block of columns on its own
    check_linear(k.Fp8Rows(x.values[::2], x.scales[::2]), w)
    check_linear(k.Fp8Rows(x.values[:, 128:], x.scales[:, 1:]), k.Fp8Weight(w.values[:, 128:], w.scales[:, 1:]))
    want = k.linear_fp8(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = k.linear_fp8(x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_a_weight_that_is_not_settled_waits_for_what_writes_it():
    """Quantised and used at once, behind a long row of kernels: the product reads what the last of them wrote."""
    k = K()
    g = torch.Generator().manual_seed(3)
    x, _ = operands(8, 16, 1024)
    src = [torch.randn(512, 1024, generator=g).cuda() for _ in range(4)]
    want = []
    for s in src:
        w = k.quantize_weight_fp8(s)
        torch.cuda.synchronize()
        want.append(k.linear_fp8(x, w))
    torch.cuda.synchronize()
    got = [k.linear_fp8(x, k.quantize_weight_fp8(s)) for s in src for _ in range(3)]
    for i, y in enumerate(got):
        assert torch.equal(y, want[i // 3])


def test_refusals():
    k = K()
    x, w = operands(4, 64, 256)
    raises = lambda match: pytest.raises(k.KernelError, match=match)     # noqa: E731
    with raises("must be `Fp8Rows`"):
        k.linear_fp8(x.values, w)
    with raises("must be `Fp8Weight`"):
        k.linear_fp8(x, x)
    with raises("no CPU path"):
        k.linear_fp8(k.Fp8Rows(x.values.cpu(), x.scales), w)
    with raises("multiples of 16 bytes"):
        odd = torch.zeros(4, 250, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        k.linear_fp8(k.Fp8Rows(odd, x.scales), w)
    with raises("one scale for each row"):
        k.linear_fp8(k.Fp8Rows(x.values, x.scales[:, :1]), w)
    with raises("one scale for each 128 rows"):
        k.linear_fp8(x, k.Fp8Weight(w.values, w.scales.repeat(2, 1)))
    with raises("float8_e4m3fn values"):
        k.linear_fp8(k.Fp8Rows(x.values.view(torch.uint8), x.scales), w)
    with raises("weight must be"):
        k.linear_fp8(x, operands(4, 64, 128)[1])
    with raises("out_dtype"):
        k.linear_fp8(x, w, out_dtype=torch.float16)
    with raises("bias must be"):
        k.linear_fp8(x, w, torch.zeros(64, dtype=torch.bfloat16, device="cuda"))
    with raises("gate and up must both"):
        k.linear_swiglu_fp8(x, w, operands(4, 65, 256)[1])
    with raises("laid out alike"):
        k.linear_swiglu_fp8(x, w, k.Fp8Weight(w.values, torch.empty(2, 4, device="cuda")[:1, ::2]))
