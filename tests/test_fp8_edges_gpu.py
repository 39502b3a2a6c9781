"""8-bit operators where their 32-bit numbers end, whatever form of the kernel runs: scales whose product leaves 32 bits, SiLU far
below zero, quotients beside the boundary between two 8-bit values."""
import pytest
import torch

from fp8_util import holds
from test_fp8_linear_gpu import check_linear, check_swiglu

pytestmark = pytest.mark.gpu

# forms of the products: which kernel, and so many CTAs (pairs) for a tile
FORMS = {"auto": 0, "rows": 1, "rows of 3": 1 + 256 * 3, "tiles": 2, "tiles of 2": 2 + 256 * 2, "pair": 3, "two pairs": 3 + 256 * 2}


def K():
    from logssms_b200.ops import kernels
    return kernels


@pytest.fixture(params=list(FORMS))
def form(request):
    k = K()
    k._FP8_FORMS["asked"] = FORMS[request.param]
    k.FP8_FORM = "asked"
    yield request.param
    k.FP8_FORM = "auto"
    del k._FP8_FORMS["asked"]


def codes(rows, width, low, high, gen):
    """Random e4m3 numbers of either sign from the bytes low .. high, rows at multiples of 16 bytes."""
    q = torch.randint(low, high + 1, (rows, width), generator=gen) | (torch.randint(0, 2, (rows, width), generator=gen) << 7)
    held = torch.full((rows, (width + 15) // 16 * 16), 0x7F, dtype=torch.uint8)
    held[:, :width] = q.to(torch.uint8)
    return held.cuda().view(torch.float8_e4m3fn)[:, :width]


def row_scales(rows, columns, gen):
    """A scale per row and block: the column's own, in some rows a thousandth of it."""
    s = torch.tensor(columns)[None] * torch.where(torch.rand(rows, len(columns), generator=gen) < 0.3, 1e-3, 1.0)
    return s.float().cuda().t().contiguous().t()


def weight_scales(columns):
    return torch.tensor([columns, [0.5 * s for s in columns]]).cuda()


# Sums of the smallest e4m3 numbers' products (up to 0.024 a block) under scales whose product is 2e39; sums of large ones (up to
# 2^24) under products of 1e-40 and below, of which 32 bits hold a few bits or none.  (bytes of the values; scales of x and of the
# weight in three blocks; scales of another weight whose products with x's are ordinary; what makes a gate of the first one's sums)
BEYOND = ((0x00, 0x07), [1e30, 1e38, 1.0], [2e9, 20.0, 1e-20], [1e-27, 1e-35, 1e3], 1e-36)
BELOW = ((0x28, 0x7E), [1e-20, 1e-35, 1e-10], [1e-20, 1e-8, 1e-33], [1e14, 1e29, 1e4], 1e34)


@pytest.mark.parametrize("m", [5, 40, 200, 300])
@pytest.mark.parametrize("case", [BEYOND, BELOW], ids=["beyond 2^128", "below 2^-126"])
def test_scales_whose_product_leaves_32_bits(m, case, form):
    k = K()
    values, x_scales, w_scales, plain_scales, act_scale = case
    g = torch.Generator().manual_seed(m)
    n, width = 200, 300
    x = k.Fp8Rows(codes(m, width, *values, g), row_scales(m, x_scales, g))
    w = k.Fp8Weight(codes(n, width, *values, g), weight_scales(w_scales))
    plain = k.Fp8Weight(codes(n, width, *values, g), weight_scales(plain_scales))
    check_linear(x, w)
    check_swiglu(x, plain, w, 1.0)                         # as the up half of a gated product
    check_swiglu(x, w, plain, act_scale)                   # as the gate half


def one_column(rows, width, columns):
    """e4m3 rows that are zero but for the given {column: values}, on 16 bytes."""
    held = torch.zeros(rows, (width + 15) // 16 * 16, dtype=torch.float8_e4m3fn)
    for c, v in columns.items():
        held[:, c] = torch.as_tensor(v, dtype=torch.float32).to(torch.float8_e4m3fn)
    return held.cuda()[:, :width]


@pytest.mark.parametrize("m", [3, 70, 260])
def test_silu_far_below_zero(m, form):
    """Gates from -80 down to -92 under up values that keep the product a number: SiLU's own size is 1e-33 to 1e-38."""
    k = K()
    width = 520
    gates = torch.arange(80.0, 92.0, 0.25).float() / 448           # a scale for each 128 features
    blocks = len(gates)
    n = 128 * blocks
    g = torch.Generator().manual_seed(m)
    x = k.Fp8Rows(one_column(m, width, {0: 1.0}), torch.ones(m, 5).cuda())
    gate = k.Fp8Weight(one_column(n, width, {0: -448.0}), gates.cuda()[:, None].repeat(1, 5))
    ups = torch.randint(1, 0x7F, (n,), generator=g).to(torch.uint8).view(torch.float8_e4m3fn).float()
    up = k.Fp8Weight(one_column(n, width, {0: ups}), torch.full((blocks, 5), 1e30).cuda())
    a = (-448 * gates.double()).repeat_interleave(128)
    h = (a * torch.sigmoid(a) * ups.double() * float(torch.tensor(1e30))).cuda().expand(m, n)
    # the exponent's constant and its rounding: 1.25 |a|; exponential 4, denominator 1, reciprocal 2, products 5, all 2^-24 of h.
    # Where e^-a is beyond 32 bits (a below -88.7) the denominator is infinite, as in any 32-bit form of it, and SiLU 0.
    error = h.abs() * torch.where(a < -88.7, 1.0, (1.25 * a.abs() + 12) * 2.0 ** -24).cuda()
    got = k.linear_swiglu_fp8(x, gate, up)
    holds(got.values, got.scales, h, error)
    assert bool((got.scales[:, :32] > 2.0 ** -126).all())          # gates down to -87.75: nothing is lost
    k.check_kernel_errors()


@pytest.mark.parametrize("m", [3, 70, 260])
def test_silu_of_large_gates(m, form):
    """Gates up to the largest numbers are their own SiLU, down to the largest negative ones nothing is left of them."""
    k = K()
    width = 520
    sizes = torch.tensor([1e2, 1e10, 1e30, 1e36, 3e38])
    n = 128 * len(sizes)
    sign = torch.where(torch.arange(n) % 2 == 0, 1.0, -1.0)
    x = k.Fp8Rows(one_column(m, width, {0: 1.0}), torch.ones(m, 5).cuda())
    gate = k.Fp8Weight(one_column(n, width, {0: 64 * sign}), (sizes / 64).cuda()[:, None].repeat(1, 5))
    up = k.Fp8Weight(one_column(n, width, {0: torch.full((n,), 0.5)}), torch.full((len(sizes), 5), 0.25).cuda())
    h = torch.where(sign > 0, (64.0 * (sizes / 64)).double().repeat_interleave(128) / 8, 0.0).cuda().expand(m, n)
    got = k.linear_swiglu_fp8(x, gate, up)
    holds(got.values, got.scales, h, h * 2.0 ** -22)
    k.check_kernel_errors()


@pytest.mark.parametrize("m", [4, 20, 60, 200, 300])
def test_a_row_does_not_hang_on_its_neighbours(m, form):
    """Rows of zeros, NaN, extreme scales beside ordinary ones: the ordinary ones' results keep their bits."""
    k = K()
    g = torch.Generator().manual_seed(m)
    n, width = 200, 400
    w, u = (k.Fp8Weight(codes(n, width, 0x10, 0x50, g), 0.01 * torch.rand(2, 4, generator=g).cuda()) for _ in range(2))
    x = codes(m, width, 0x10, 0x50, g)
    scales = torch.rand(m, 4, generator=g).cuda()
    plain, gated = k.linear_fp8(k.Fp8Rows(x, scales), w, out_dtype=torch.float32), k.linear_swiglu_fp8(k.Fp8Rows(x, scales), w, u)
    other = scales.clone()
    other[0, 0], other[1, 1], other[2], other[-1, 3] = 2.0 ** -126, float("nan"), 1e-38, 3e38
    rows = k.Fp8Rows(x, other)
    got, rest = k.linear_fp8(rows, w, out_dtype=torch.float32), slice(3, m - 1)
    assert torch.equal(got[rest], plain[rest])
    again = k.linear_swiglu_fp8(rows, w, u)
    assert torch.equal(again.scales[rest], gated.scales[rest])
    assert torch.equal(again.values.view(torch.uint8)[rest], gated.values.view(torch.uint8)[rest])
    k.check_kernel_errors()


@pytest.mark.parametrize("m", [3, 70, 260])
def test_gated_rows_are_divided_by_their_scale(m, form):
    """A gate of 64 is its own SiLU, and sums of two products are exact: the 8-bit values are the float32 quotients by the scale,
    rounded once, also where a quotient lies on the boundary between two of them or beside it."""
    k = K()
    width, blocks = 520, 60
    n = 128 * blocks
    g = torch.Generator().manual_seed(7)
    first = torch.tensor([256, 288, 320, 352, 384, 416, 128, 144, 160, 176, 192, 208, 224, 240] * 9 + [448, 448]).float().repeat(blocks)
    second = torch.tensor([256, 240, 256, 288, 256, 256, 128, 128, 120, 128, 144, 128, 128, 128] * 9 + [0, 0]).float().repeat(blocks)
    up_scales = torch.exp(4 * torch.randn(blocks, generator=g))
    x = k.Fp8Rows(one_column(m, width, {0: 1.0, 1: 0.0625}), torch.ones(m, 5).cuda())
    gate = k.Fp8Weight(one_column(n, width, {0: 64.0}), torch.ones(blocks, 5).cuda())
    up = k.Fp8Weight(one_column(n, width, {0: first, 1: second}), up_scales[:, None].repeat(1, 5).cuda())
    got = k.linear_swiglu_fp8(x, gate, up)
    h = 64 * ((first + second / 16).view(blocks, 128) * up_scales[:, None])          # float32 on the CPU, one rounding
    scales = (h.amax(1).double() / 448).float()
    want = (h / scales[:, None]).to(torch.float8_e4m3fn).view(torch.uint8).view(-1)
    assert torch.equal(got.scales.cpu(), scales.expand(m, blocks))
    assert torch.equal(got.values.view(torch.uint8).cpu(), want.expand(m, n))
    k.check_kernel_errors()
