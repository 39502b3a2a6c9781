"""The choice of 8-bit feed-forward weights on the CPU: the command line's option, what the block asks of the norm, and what a
feed-forward refuses."""
from types import SimpleNamespace

import pytest

from logssms_b200.cli import build_parser
from logssms_b200.parts.block import PreNormParallelBlock


def test_the_option_parses():
    assert build_parser().parse_args(["--model", "/m"]).feed_forward_weights == "model"
    assert build_parser().parse_args(["--model", "/m", "--feed-forward-weights", "float8"]).feed_forward_weights == "float8"
    with pytest.raises(SystemExit):
        build_parser().parse_args(["--model", "/m", "--feed-forward-weights", "int8"])


class Norm:
    def __init__(self, can_fp8):
        if can_fp8:
            self.can_fp8 = True
        self.asked = []

    def forward(self, x, residual=None, *, out_scales=(1.0,), **kw):
        self.asked.append(kw)
        return tuple(("normed", x) for _ in out_scales), ("residual", x)


class Mixer:
    def forward(self, x, ctx, cache_layer, writes_cache=True):
        return ("mixed", x)


class FeedForward:
    can_lazy_scale = False

    def __init__(self, takes):
        self.takes_fp8_rows = takes

    def forward(self, x):
        return ("ff", x)


@pytest.mark.parametrize("takes", [False, True])
@pytest.mark.parametrize("can", [False, True])
@pytest.mark.parametrize("mixers", [1, 2])
def test_the_norm_is_asked_for_8_bit_rows_only_where_both_sides_say_so(takes, can, mixers):
    block = object.__new__(PreNormParallelBlock)
    block.spec = SimpleNamespace(mixers=[SimpleNamespace(in_scale=1.0, out_scale=1.0) for _ in range(mixers)])
    block.mixers = [Mixer() for _ in range(mixers)]
    block.mixer_norm, block.ff_norm = Norm(can), Norm(can)
    block.feed_forward = FeedForward(takes)
    out, residual = block.forward("x", "r", SimpleNamespace(extras={"next_norm_takes_scaled": True}), cache_layer=0)
    assert out[0] == "ff" and residual[0] == "residual"
    assert "fp8" not in block.mixer_norm.asked[0]
    assert block.ff_norm.asked[0].get("fp8", False) == (takes and can)


def test_a_feed_forward_knows_two_kinds_of_weights():
    from logssms_b200.parts.mlp import GatedMLP
    part = GatedMLP(SimpleNamespace(hidden_size=8, intermediate_size=16, activation_scale=1.0, output_scale=1.0))
    part.setup(SimpleNamespace(options={}))
    part.setup(SimpleNamespace(options={"feed_forward_weights": "model"}))
    assert part.fp8 is None and not part.takes_fp8_rows and part.takes_normed_rows
    with pytest.raises(ValueError, match="model or float8"):
        part.setup(SimpleNamespace(options={"feed_forward_weights": "int4"}))


def test_a_norm_leaves_one_output_in_8_bits():
    from logssms_b200.parts.norm import RMSNorm
    norm = RMSNorm(SimpleNamespace(size=8, eps=1e-5))
    with pytest.raises(ValueError, match="one output"):
        norm.forward(None, None, out_scales=(1.0, 2.0), fp8=True)
