"""The engine on 8-bit feed-forward weights: generation against the plain model whose feed-forwards quantise weights and rows the
same way, steps in graphs and without, and what is refused."""
import pytest
import torch

from fp8_util import BLOCK, blocks_top, holds, product, product_error, spread
from tiny import TINY, make_model_dir, plain_logits

pytestmark = pytest.mark.gpu

# The plain model's 8-bit values are the engine's except where rounding in front of them differs: a value of 8 bits then moves by a
# step, 2^-3 of itself, in a few of a hundred columns, which moves a feed-forward's output by about a hundredth and the logits by
# less.  The bound is the one of bfloat16 engines, 2e-2 of the largest logit.
TOL = 2e-2


def through_8_bits(v, block_rows):
    rows, width = v.shape
    each = spread((blocks_top(v, block_rows) / 448).clamp(min=2.0 ** -126).float(), block_rows, rows, width)
    return (v.float() / each).to(torch.float8_e4m3fn).to(v.dtype) * each.to(v.dtype)


@pytest.fixture
def plain_in_8_bits(monkeypatch):
    from plain import falcon_h1_plain

    def gated_mlp(h, w_gate, w_up, w_down, act_scale, out_scale, rnd, linear):
        x = through_8_bits(h, 1)
        gate, up = (x @ through_8_bits(w.to(x.dtype), BLOCK).t() for w in (w_gate, w_up))
        gate = gate * act_scale
        y = through_8_bits(gate * torch.sigmoid(gate) * up, 1) @ through_8_bits(w_down.to(x.dtype), BLOCK).t()
        return rnd(y * out_scale)
    monkeypatch.setattr(falcon_h1_plain, "gated_mlp", gated_mlp)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B"])
def test_greedy_generation(tmp_path, name, dtype, plain_in_8_bits):
    from logssms_b200.engine import LLM
    from logssms_b200.ops import kernels as K
    from logssms_b200.sampling import SamplingParams
    raw = TINY[name]
    model_dir = make_model_dir(tmp_path / "m", raw, seed=21, dtype=torch.float32 if dtype == "float32" else torch.bfloat16)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, raw["vocab_size"], (n,), generator=g).tolist() for n in (1, 5, 70, 33)]
    make = lambda **kw: LLM(model_dir, dtype, max_running_requests=3, max_seq_len_override=128, num_pages=4, max_prefill_tokens=24,   # noqa: E731
                            feed_forward_weights="float8", **kw)
    params = SamplingParams(temperature=0.0, max_tokens=10, ignore_eos=True)
    llm = make()
    for layer in llm.engine.model.layers:
        ff = layer.feed_forward
        assert ff.gate_up is None and ff.down is None and all(w.settled and w.values.dtype == torch.float8_e4m3fn for w in ff.fp8)
        assert ff.fp8[0].shape == (raw["intermediate_size"], raw["hidden_size"])
    before = K.launch_count
    outs = llm.generate(prompts, params)
    assert K.launch_count > before
    exact = total = 0
    for prompt, out in zip(prompts, outs):
        ids = list(prompt)
        for tok in out.token_ids:
            logits = plain_logits(model_dir, ids, dtype)[-1]
            gap = float(logits.max() - logits[tok]) / float(logits.abs().max())
            assert gap <= TOL, f"engine chose {tok}, gap {gap:.3g}"
            exact, total = exact + int(tok == int(logits.argmax())), total + 1
            ids.append(tok)
    assert exact >= 0.8 * total
    K.check_kernel_errors()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_logits_of_portions_and_decoded_tokens(tmp_path, dtype, plain_in_8_bits):
    """A prompt whole, in portions, and its last tokens one by one, kernel by kernel and from graphs: all give the plain logits."""
    from logssms_b200.engine import Engine, StepEntry
    raw = TINY["B"]
    model_dir = make_model_dir(tmp_path / "m", raw, seed=3, dtype=torch.float32 if dtype == "float32" else torch.bfloat16)
    ids = torch.randint(0, raw["vocab_size"], (100,), generator=torch.Generator().manual_seed(1)).tolist()
    want = plain_logits(model_dir, ids, dtype)
    largest = float(want.abs().max())
    for graphs in (False, True):
        engine = Engine(model_dir, dtype, max_requests=4, max_seq_len=128, num_pages=8, use_graphs=graphs, feed_forward_weights="float8")
        for cuts in ([100], [37, 100], [80] + list(range(81, 101))):
            r, at = engine.new_request(), 0
            for end in cuts:
                got = engine.step([StepEntry(r, ids[at:end], list(range(end - at)))]).float().cpu()
                assert float((got - want[at:end].float()).abs().max()) <= TOL * largest
                at = end
            engine.release(r)


def test_the_part_alone_is_its_three_quantised_products():
    from logssms_b200.config import GatedMLPSpec
    from logssms_b200.ops import kernels as K
    from logssms_b200.parts import Runtime
    from logssms_b200.parts.mlp import GatedMLP
    g = torch.Generator().manual_seed(2)
    hidden, inter = 300, 500
    part = GatedMLP(GatedMLPSpec(hidden_size=hidden, intermediate_size=inter, activation_scale=0.9, output_scale=1.1))
    part.bind({n: (torch.randn(s.shape, generator=g) * s.shape[1] ** -0.5).to(torch.bfloat16).cuda() for n, s in part.param_specs().items()})
    part.setup(Runtime(torch.device("cuda:0"), torch.bfloat16, 64, 64, {"feed_forward_weights": "float8"}))
    x = torch.randn(40, hidden, generator=g).to(torch.bfloat16).cuda()
    rows = K.quantize_rows_fp8(x)
    y = part.forward(rows)
    assert y.dtype == torch.bfloat16 and torch.equal(part.forward(x), y)          # plain rows are quantised on the way
    gate, up, down = part.fp8
    h = K.linear_swiglu_fp8(rows, gate, up, 0.9)
    a, a_size = product(rows.values, rows.scales, gate.values, gate.scales)
    b, b_size = product(rows.values, rows.scales, up.values, up.scales)
    a = a * 0.9
    error = 1.1 * 0.9 * product_error(a_size, hidden) * b.abs() + a.abs() * product_error(b_size, hidden) + (a * b).abs() * (a.abs() + 8) * 2.0 ** -24
    holds(h.values, h.scales, a * torch.sigmoid(a) * b, error)
    want, size = product(h.values, h.scales, down.values, down.scales)
    assert bool(((y.double() - 1.1 * want).abs() <= 1.1 * product_error(size, inter) + want.abs() * 2.0 ** -7).all())


def test_refusals(tmp_path):
    from logssms_b200.engine import Engine
    from tiny_dudurax import DUDU_A
    model_dir = make_model_dir(tmp_path / "m", TINY["A"], seed=1)
    with pytest.raises(ValueError, match="model or float8"):
        Engine(model_dir, "bfloat16", max_requests=2, max_seq_len=64, num_pages=2, feed_forward_weights="int8")
    other = make_model_dir(tmp_path / "d", DUDU_A, seed=1)
    with pytest.raises(ValueError, match="no feed-forward of this model"):
        Engine(other, "bfloat16", max_requests=2, max_seq_len=64, num_pages=2, feed_forward_weights="float8")
