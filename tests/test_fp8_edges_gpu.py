"""8-bit operators where their 32-bit numbers end: scales whose product leaves 32 bits, whatever form of the kernel runs."""
import pytest
import torch

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
