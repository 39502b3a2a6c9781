"""Quantisation to 8-bit floating point and the norm that leaves 8-bit rows (`fp8_rows.cu`) against 64 bits."""
import pytest
import torch

from fp8_util import BLOCK, TINY, blocks_top, holds

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]


def K():
    from logssms_b200.ops import kernels
    return kernels


def activations(rows, width, dtype, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width + pad, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))
    return x.to(dtype).cuda()[:, :width]


# widths: one value, less than a piece, pieces, one block, a remainder, odd, several pieces per thread, beyond the pieces
WIDTHS = [1, 5, 8, 120, 128, 136, 1003, 1024, 3072, 5000, 8192, 9000]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 3, 130])
@pytest.mark.parametrize("width", WIDTHS)
def test_quantised_rows(width, rows, dtype):
    for pad in (0, 8, 3):                                  # whole rows, strided rows on 16 bytes, strided rows off them
        x = activations(rows, width, dtype, width + rows, pad)
        got = K().quantize_rows_fp8(x)
        assert got.values.stride(0) % 16 == 0 and got.scales.stride() == (1, rows)
        holds(got.values, got.scales, x.double(), torch.zeros_like(x, dtype=torch.float64))
        # the largest magnitude is exact and its quotient rounded once
        assert torch.equal(got.scales, (blocks_top(x) / 448).float().clamp(min=TINY))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (5, 128), (128, 128), (129, 136), (200, 1003), (640, 384), (1000, 264)])
def test_quantised_weight(rows, width, dtype):
    for pad in (0, 8, 3):
        w = activations(rows, width, dtype, width + rows, pad)
        got = K().quantize_weight_fp8(w)
        assert got.shape == (rows, width) and not got.settled
        holds(got.values, got.scales, w.double(), torch.zeros_like(w, dtype=torch.float64), BLOCK)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("width", WIDTHS)
def test_norm(width, rows, dtype):
    k = K()
    for other, residual, pad in ((True, True, 0), (False, True, 8), (False, False, 0), (True, False, 3)):
        x = activations(rows, width, dtype, width, pad)
        o = activations(rows, width, dtype, width + 1, pad) if other else None
        r = activations(rows, width, dtype, width + 2, pad) if residual else None
        w = (1 + 0.2 * torch.randn(width, generator=torch.Generator().manual_seed(1))).cuda()
        a, b = (0.8, 0.7) if other else (1.3, 1.0)
        keep = None if r is None else r.clone()
        got, new = k.add_rmsnorm_fp8(x, w, 1e-5, r, other=o, in_scales=(a, b), out_scale=1.5, in_place=False)
        terms = [a * x.double()] + ([b * o.double()] if other else []) + ([r.double()] if residual else [])
        total, size = sum(terms), sum(t.abs() for t in terms)
        inv = torch.rsqrt(total.square().mean(1, keepdim=True) + 1e-5) * w.double() * 1.5
        # 32-bit arithmetic in front of the 8 bits: the sum (three roundings of its terms' size), the mean of squares (a thread
        # adds at most 36 values in a row, the CTA ten more; half of it after the root; the sum's own errors once more), four
        # factors: 2^-24 x (3 + 23 + 3 + 8), rounded up
        mean_error = (size * total.abs()).mean(1, keepdim=True) / (total.square().mean(1, keepdim=True) + 1e-5)
        error = (size + total.abs() * (1 + mean_error)) * inv.abs() * 2.0 ** -18
        holds(got.values, got.scales, total * inv, error)
        # the new residual: the 32-bit sum, rounded once
        step = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23
        assert bool(((new.double() - total).abs() <= total.abs() * step + size * 2.0 ** -22).all())
        if residual:
            assert torch.equal(r, keep)
            again, same = k.add_rmsnorm_fp8(x, w, 1e-5, r, other=o, in_scales=(a, b), out_scale=1.5)
            assert same is r and torch.equal(r, new) and torch.equal(again.scales, got.scales)
            assert torch.equal(again.values.view(torch.uint8), got.values.view(torch.uint8))
        none = k.add_rmsnorm_fp8(x, w, 1e-5, keep, other=o, in_scales=(a, b), out_scale=1.5, want_residual=False)
        assert none[1] is None and torch.equal(none[0].scales, got.scales)


@pytest.mark.parametrize("width", [256, 301])
def test_zeros_infinities_and_nan_stay_in_their_blocks(width):
    k = K()
    x = torch.ones(4, width, device="cuda")
    x[0] = 0
    x[1, 130] = float("inf")
    x[2, 5] = float("nan")
    x[3, 140] = 1e-44                                      # a denormal beside ones
    for got, rows in ((k.quantize_rows_fp8(x), 1), (k.quantize_weight_fp8(x), 4)):
        v, s = got.values.float(), got.scales
        if rows == 1:
            assert bool((v[0] == 0).all()) and bool((s[0] == TINY).all())
            assert bool((v[1, :128] == 448).all()) and torch.isinf(s[1, 1]) and torch.isnan(v[1, 130])
            assert bool((v[1, 131:256] == 0).all())
            assert torch.isnan(s[2, 0]) and bool(torch.isnan(v[2, :128]).all()) and bool((v[2, 128:] == 448).all())
            assert v[3, 140] == 0 and v[3, 139] == 448
        else:
            assert bool(torch.isnan(s[0, 0])) and bool(torch.isnan(v[:, :128]).all()) and bool(torch.isinf(s[0, 1]))
            assert bool(torch.isnan(v[1, 130])) and bool((v[0, 128:] == 0).all())
    tiny = torch.full((1, width), 1e-42, device="cuda")    # a block whose quotient would be denormal
    got = k.quantize_rows_fp8(tiny)
    assert bool((got.scales == TINY).all()) and bool((got.values.float() == 0).all())
    normed, new = k.add_rmsnorm_fp8(x, torch.ones(width, device="cuda"), 1e-5)
    v = normed.values.float()
    assert bool((v[0] == 0).all()) and bool((new[0] == 0).all())
    # an infinity: the row's root is infinite, the others become zeros, itself NaN; a NaN takes its whole row
    assert bool((v[1, :128] == 0).all()) and bool(torch.isnan(v[1, 128:256]).all()) and bool(torch.isnan(v[2]).all())
    assert bool((v[3, :128] == 448).all())


def test_empty_and_other_streams():
    k = K()
    empty = k.quantize_rows_fp8(torch.empty(0, 64, device="cuda"))
    assert empty.shape == (0, 64) and empty.scales.shape == (0, 1)
    rows, new = k.add_rmsnorm_fp8(torch.empty(0, 64, device="cuda"), torch.ones(64, device="cuda"), 1e-5)
    assert rows.shape == (0, 64) and new.shape == (0, 64)
    side = torch.cuda.Stream()
    x = torch.randn(500, 640, device="cuda")
    want = k.quantize_rows_fp8(x)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = k.quantize_rows_fp8(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got.scales, want.scales) and torch.equal(got.values.view(torch.uint8), want.values.view(torch.uint8))


def test_refusals():
    k = K()
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    with pytest.raises(k.KernelError, match="no CPU path"):
        k.quantize_rows_fp8(x.cpu())
    with pytest.raises(k.KernelError, match="unit column stride"):
        k.quantize_rows_fp8(x.t())
    with pytest.raises(k.KernelError, match="unsupported dtype"):
        k.quantize_weight_fp8(x.half())
    with pytest.raises(k.KernelError, match="at least one column"):
        k.quantize_rows_fp8(x[:, :0])
    with pytest.raises(k.KernelError, match="norm weight"):
        k.add_rmsnorm_fp8(x, w[:32], 1e-5)
    with pytest.raises(k.KernelError, match="residual must match"):
        k.add_rmsnorm_fp8(x, w, 1e-5, x.bfloat16())
    with pytest.raises(k.KernelError, match="other must match"):
        k.add_rmsnorm_fp8(x, w, 1e-5, other=x[:2])
