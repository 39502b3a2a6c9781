"""8-bit rows and weights in 64 bits, and how far a kernel's may be from them.

e4m3 keeps 3 bits behind the point from 2^-6 up and steps of 2^-9 below: a value rounded to nearest is off by at most 2^-4 of
itself, or by 2^-10.  `HALF_STEP` has a little more (2^-10 of it) for the 32-bit quotient that is rounded: its own two roundings
can carry it over a boundary."""
import torch

BLOCK = 128
TINY = 2.0 ** -126
SLACK = 1.0 + 2.0 ** -10


def blocks_top(v, block_rows=1):
    """Largest magnitude of every block, 64-bit [ceil(rows / block_rows), ceil(width / 128)]."""
    rows, width = v.shape
    v = torch.nn.functional.pad(v.double().abs(), (0, -width % BLOCK, 0, -rows % block_rows))
    return v.view(v.shape[0] // block_rows, block_rows, v.shape[1] // BLOCK, BLOCK).amax((1, 3))


def spread(scales, block_rows, rows, width):
    return scales.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :width]


def half_step(v, each):
    """How far the rounding to 8 bits may take a value `v` of a block whose scale is `each`."""
    return torch.maximum(v.abs() * 2.0 ** -4, each * 2.0 ** -10) * SLACK


def holds(values, scales, v, error, block_rows=1):
    """Asserts that 8-bit rows stand for the 64-bit `v`, which the 32-bit arithmetic in front may have missed by `error` (a
    tensor like v): the scales are those of v up to that, the values within half a step."""
    rows, width = v.shape
    top, top_error = blocks_top(v, block_rows), blocks_top(error, block_rows)
    s = scales.double()
    assert s.shape == top.shape and values.shape == v.shape and values.dtype == torch.float8_e4m3fn
    want = (top / 448).clamp(min=TINY)
    assert bool(((s - want).abs() <= want * 2.0 ** -22 + top_error / 448).all())
    each = spread(s, block_rows, rows, width)
    off = (values.double() * each - v).abs()
    assert bool((off <= half_step(v, each) + error * SLACK).all())


def make_rows(m, k, gen, row_major=False, loud=True):
    """8-bit rows (values, scales) of random activations on the GPU, laid out by elementary operations."""
    x = torch.randn(m, k, generator=gen)
    if loud:
        x *= torch.where(torch.rand(k, generator=gen) < 0.02, 8.0, 1.0)
    x *= torch.exp(torch.randn(m, 1, generator=gen))
    return lay_out(x, 1, row_major)


def make_weight(n, k, gen):
    return lay_out(torch.randn(n, k, generator=gen) * k ** -0.5 * torch.exp(torch.randn(n, 1, generator=gen)), BLOCK, True)


def lay_out(x, block_rows, row_major):
    rows, width = x.shape
    scales = (blocks_top(x, block_rows) / 448).clamp(min=TINY).float()
    q = (x / spread(scales, block_rows, rows, width)).to(torch.float8_e4m3fn)
    pitch = (width + 15) // 16 * 16
    # what lies between the rows must not matter: NaN bytes
    held = torch.full((rows, pitch), 0x7F, dtype=torch.uint8)
    held[:, :width] = q.view(torch.uint8)
    values = held.cuda().view(torch.float8_e4m3fn)[:, :width]
    scales = scales.cuda()
    return values, scales if row_major else scales.t().contiguous().t()


def product(x, xs, w, ws):
    """(x @ w^T, the same of the magnitudes) of 8-bit operands in 64 bits."""
    a = x.double() * spread(xs.double(), 1, *x.shape)
    b = w.double() * spread(ws.double(), BLOCK, *w.shape)
    return a @ b.t(), a.abs() @ b.abs().t()


def product_error(size, k):
    """Bound on the 32-bit sums' error: the products of two e4m3 values are exact; a block's 128 of them are added, at worst one by
    one with the last bit cut off (2^-23 each), then times the joined scales (2^-24 twice) and added over the blocks."""
    return size * (128 + 2 * ((k + 127) // 128) + 4) * 2.0 ** -23
