"""Gated (SwiGLU) feed-forward."""
from __future__ import annotations

import torch

from ..ops import build as kernel_build
from ..ops import kernels as K
from ..registry import FEED_FORWARDS
from .base import MATRIX, ParamSpec, Part


@FEED_FORWARDS.register("gated_mlp")
class GatedMLP(Part):
    """down(silu(gate * s0) * up) * s1.  `gate_proj` and `up_proj` are concatenated at bind time
    (python/logssms/models/weight.py:32-33); flow python/logssms/layers/mlp.py:50-61.

    With 8-bit weights (the engine's `feed_forward_weights`): e4m3 values with a float32 scale per 128 x 128, the rows in 8 bits
    too, and two kernels behind the norm that leaves them: gate, up, SiLU and product in one, whose output is 8-bit rows again, and
    down.  Sums are 32-bit and rounded once."""
    takes_normed_rows = True      # forward() passes its input straight into a product
    joins_residual = True         # forward() takes `join=`: its last product may add the residual in its epilogue
    kernels = ("norm", "linear_skinny", "linear_rows_tc", "gemm_tcgen05")

    def __init__(self, spec, perturb_init: bool = False, shared: dict | None = None):
        self.spec = spec
        self.gate_up = self.down = None
        self.fp8 = None       # (gate, up, down) as `K.Fp8Weight` where the engine's user chose 8-bit feed-forward weights
        self.dtype = None

    def param_specs(self):
        s = self.spec
        return {
            "gate_proj.weight": ParamSpec((s.intermediate_size, s.hidden_size), MATRIX),
            "up_proj.weight": ParamSpec((s.intermediate_size, s.hidden_size), MATRIX),
            "down_proj.weight": ParamSpec((s.hidden_size, s.intermediate_size), MATRIX),
        }

    def bind(self, t):
        self.gate_up = torch.cat([t["gate_proj.weight"], t["up_proj.weight"]], 0).contiguous()
        self.down = t["down_proj.weight"]

    def setup(self, rt) -> None:
        """With `feed_forward_weights` = "float8" the matrices are laid out in 8 bits here, once, and the 16-bit ones given up."""
        choice = rt.options.get("feed_forward_weights", "model")
        if choice not in ("model", "float8"):
            raise ValueError(f"feed_forward_weights must be model or float8, got {choice!r}")
        if choice == "model":
            return
        kernel_build.build_many(("fp8_rows", "fp8_linear"))
        gate, up = self.gate_up.chunk(2)
        self.fp8 = tuple(K.quantize_weight_fp8(w) for w in (gate, up, self.down))
        torch.cuda.synchronize(rt.device)
        for w in self.fp8:
            w.settled = True                  # a product may ask for them while the kernels in front of it still run
        self.gate_up = self.down = None
        self.dtype = rt.dtype
        # what the norm in front and the block do for 16-bit products has no place here: the norm hands over 8-bit rows
        self.takes_fp8_rows, self.takes_normed_rows, self.joins_residual, self.can_lazy_scale = True, False, False, False

    takes_fp8_rows = False    # (8-bit weights) forward() takes `K.Fp8Rows`
    can_lazy_scale = True     # forward() takes `lazy_scale=`: see there

    def forward(self, x: torch.Tensor, join=None, lazy_scale: bool = False):
        """With `join` (a `K.ResidualJoin`) and few rows the down projection adds the residual in its epilogue and
        `K.SummedRows` come back instead of a tensor.  With `lazy_scale` (the norm that reads the output next takes
        `K.ScaledRows`) the output multiplier may be left to that norm."""
        s = self.spec
        if self.fp8 is not None:
            gate, up, down = self.fp8
            if not isinstance(x, K.Fp8Rows):
                x = K.quantize_rows_fp8(x if isinstance(x, torch.Tensor) else x.tensor())
            return K.linear_fp8(K.linear_swiglu_fp8(x, gate, up, s.activation_scale), down, out_scale=s.output_scale, out_dtype=self.dtype)
        h = K.linear_swiglu(x, self.gate_up, s.activation_scale)
        if K.linear_join_ok(h, self.down, None, join):
            return K.linear_join(h, self.down, None, join, out_scale=s.output_scale)
        return K.linear(h, self.down, out_scale=s.output_scale, lazy_scale=lazy_scale)
