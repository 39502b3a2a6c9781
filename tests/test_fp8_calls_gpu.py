"""How the 8-bit operators are called: through the binding and past it, and what they allocate."""
from types import SimpleNamespace

import pytest
import torch

from fp8_util import make_rows, make_weight

pytestmark = pytest.mark.gpu


def K():
    from logssms_b200.ops import kernels
    return kernels


def operands(m, n, k, seed=0):
    g = torch.Generator().manual_seed(1000 * m + n + k + seed)
    kk = K()
    return kk.Fp8Rows(*make_rows(m, k, g)), kk.Fp8Weight(*make_weight(n, k, g), settled=True), kk.Fp8Weight(*make_weight(n, k, g), settled=True)


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
