"""What the serving operators refuse, on the CPU: tensors that only pretend to be on a device reach every check, and no launch."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from logssms_b200.ops import kernels as K
from logssms_b200.sampling import edit_logits


@pytest.fixture(autouse=True)
def pretended_device(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0)

    class NothingInOrder:
        def __getattr__(self, name):
            return lambda *args: None

    monkeypatch.setattr(K, "_serving_binding", NothingInOrder())

    def launched(lib, name, argtypes):
        raise AssertionError(f"{name} was reached")

    monkeypatch.setattr(K, "_fn", launched)
    with FakeTensorMode(allow_non_fake_inputs=True):
        yield


def on(*shape, dtype=torch.float32, device="cuda:0"):
    return torch.empty(shape, dtype=dtype, device=device)


def i32(*shape, **kw):
    return on(*shape, dtype=torch.int32, **kw)


def refused(call, words):
    with pytest.raises(K.KernelError, match=words):
        call()


# --------------------------------------------------------------------------- attention over a shared prefix
def attention(scale=0.125, **change):
    a = {"q": on(4, 8, 64, dtype=torch.bfloat16), "k_cache": on(10, 64, 2, 64, dtype=torch.bfloat16), "v_cache": on(10, 64, 2, 64, dtype=torch.bfloat16),
         "block_table": i32(3, 5), "token_req": i32(4), "positions": i32(4), "group_start": i32(3), "prefix_lens": i32(2), **change}
    kw = {k: a.pop(k) for k in ("out",) if k in a}
    return K.attention_decode_shared(*a.values(), scale, max_prefix=64, max_context=128, **kw)


def test_attention_in_order_reaches_the_launcher():
    with pytest.raises(AssertionError, match="lb_attention_shared"):
        attention()


@pytest.mark.parametrize("change,words", [
    ({"q": on}, "CUDA tensors only"),
    ({"q": lambda: on(4, 512, dtype=torch.bfloat16)}, r"q must be \[tokens, heads, head_dim\]"),
    ({"q": lambda: on(4, 64, 8, dtype=torch.bfloat16).transpose(1, 2)}, "queries must lie side by side"),
    ({"q": lambda: on(4, 8, 64)}, "q's dtype"),
    ({"q": lambda: on(4, 8, 64, dtype=torch.float16), "k_cache": lambda: on(10, 64, 2, 64, dtype=torch.float16),
      "v_cache": lambda: on(10, 64, 2, 64, dtype=torch.float16)}, "unsupported dtype"),
    ({"q": lambda: on(4, 7, 64, dtype=torch.bfloat16)}, "multiple of key/value heads"),
    ({"q": lambda: on(4, 8, 36, dtype=torch.bfloat16), "k_cache": lambda: on(10, 64, 2, 36, dtype=torch.bfloat16),
      "v_cache": lambda: on(10, 64, 2, 36, dtype=torch.bfloat16)}, "steps of 8 up to 256"),
    ({"v_cache": lambda: on(10, 64, 2, 128, dtype=torch.bfloat16)}, "caches must be contiguous"),
    ({"k_cache": lambda: on(10, 2, 64, 64, dtype=torch.bfloat16).transpose(1, 2)}, "caches must be contiguous"),
    ({"block_table": lambda: on(3, 5)}, "block table"),
    ({"block_table": lambda: i32(5, 3).t()}, "block table"),
    ({"token_req": lambda: i32(3)}, "one entry of token_req"),
    ({"positions": lambda: on(4, dtype=torch.int64)}, "positions must be a contiguous int32"),
    ({"group_start": lambda: i32(2)}, "one entry more than prefix_lens"),
    ({"prefix_lens": lambda: i32(2, device="cuda:1")}, "prefix_lens must be on q's device"),
    ({"out": lambda: on(4, 8, 64)}, "out must be a contiguous tensor like q"),
    ({"out": lambda: on(4, 8, 128, dtype=torch.bfloat16)[:, :, :64]}, "out must be a contiguous tensor like q"),
])
def test_attention_refuses(change, words):
    if words == "CUDA tensors only":
        change = {"q": lambda: on(4, 8, 64, dtype=torch.bfloat16, device="cpu")}
    refused(lambda: attention(**{k: v() for k, v in change.items()}), words)


@pytest.mark.parametrize("scale", [0.0, -0.125, float("nan"), float("inf"), 1e39, 1e-60])
def test_attention_refuses_scales_that_are_no_positive_numbers(scale):
    refused(lambda: attention(scale=scale), "scale must be a positive number")


@pytest.mark.parametrize("which", ["k_cache", "v_cache", "out"])
def test_attention_refuses_places_between_16_bytes(which):
    shape = (4, 8, 64) if which == "out" else (10, 64, 2, 64)
    n = shape[0] * shape[1] * shape[2] * (shape[3] if len(shape) > 3 else 1)
    for off in (1, 4):
        refused(lambda: attention(**{which: on(n + 8, dtype=torch.bfloat16)[off:off + n].view(shape)}), "multiple of 16 bytes")


def test_attention_of_another_device_than_the_current_one(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)
    refused(attention, "current device")


def test_attention_of_nothing_launches_nothing():
    assert attention(q=on(0, 8, 64, dtype=torch.bfloat16), token_req=i32(0), positions=i32(0)).shape == (0, 8, 64)
    assert attention(group_start=i32(1), prefix_lens=i32(0)).shape == (4, 8, 64)


# --------------------------------------------------------------------------- adapters
def adapters(**change):
    a = {"y": on(4, 32), "x": on(4, 16), "a": on(3, 8, 16), "b": on(3, 32, 8), "index": i32(4), "scales": on(3), **change}
    kw = {k: a.pop(k) for k in ("ranks", "out") if k in a}
    return K.add_adapters(*a.values(), **kw)


@pytest.mark.parametrize("change,words", [
    ({"y": lambda: on(4, 32, device="cpu")}, "CUDA tensors only"),
    ({"y": lambda: on(32, 4).t()}, "unit column stride"),
    ({"x": lambda: on(5, 16)}, "x must be"),
    ({"x": lambda: on(4, 16, dtype=torch.bfloat16)}, "one dtype"),
    ({"a": lambda: on(3, 16, 8).transpose(1, 2)}, "columns of a and b must lie side by side"),
    ({"a": lambda: on(8, 16)}, r"a must be \[adapters, rank, width\]"),
    ({"b": lambda: on(3, 32, 9)}, "b must be"),
    ({"index": lambda: i32(5)}, "one index per row"),
    ({"index": lambda: on(4, dtype=torch.int64)}, "index must be a contiguous int32"),
    ({"scales": lambda: on(3, dtype=torch.bfloat16)}, "scales must be"),
    ({"ranks": lambda: i32(2)}, "one rank per adapter"),
    ({"b": lambda: on(3, 32, 8, device="cuda:1")}, "b must be on y's device"),
    ({"out": lambda: on(4, 33)}, "out must match y"),
    ({"out": lambda: on(1, 32).expand(4, 32)}, "its rows must not overlap"),
])
def test_adapters_refuse(change, words):
    refused(lambda: adapters(**{k: v() for k, v in change.items()}), words)


def test_adapters_refuse_types_that_no_kernel_takes():
    half = {k: v.half() for k, v in {"y": on(4, 32), "x": on(4, 16), "a": on(3, 8, 16), "b": on(3, 32, 8)}.items()}
    refused(lambda: adapters(**half), "unsupported dtype")


def test_adapters_of_nothing_launch_nothing():
    assert adapters(y=on(0, 32), x=on(0, 16), index=i32(0)).shape == (0, 32)
    assert adapters(y=on(4, 0), b=on(3, 0, 8)).shape == (4, 0)


# --------------------------------------------------------------------------- rules on logits
@pytest.mark.parametrize("change,words", [
    ({"logits": lambda: on(3, 70, device="cpu")}, "CUDA tensors only"),
    ({"logits": lambda: on(3, 70, dtype=torch.bfloat16)}, "logits must be float32"),
    ({"logits": lambda: on(70, 3).t()}, "unit column stride"),
    ({"lengths": None}, "a history needs lengths"),
    ({"lengths": lambda: i32(4)}, "lengths must be a contiguous"),
    ({"prompt_lengths": lambda: on(3)}, "prompt_lengths must be a contiguous"),
    ({"history": lambda: on(3, 9)}, "history must be a row-major int32 matrix"),
    ({"history": lambda: i32(2, 9)}, "needs a row for every row of logits"),
    ({"history": None, "lengths": None}, "penalties need a history"),
    ({"frequency": lambda: on(3, dtype=torch.float64)}, "frequency must be a contiguous"),
    ({"presence": lambda: on(3, device="cuda:1")}, "presence must be on the logits' device"),
    ({"bias_start": lambda: i32(4)}, "biases need"),
    ({"bias_ids": lambda: i32(4)}, "biases need"),
    ({"bias_start": lambda: i32(3), "bias_ids": lambda: i32(5), "bias_values": lambda: on(5)}, "bias_start must be"),
    ({"bias_start": lambda: i32(4), "bias_ids": lambda: i32(5), "bias_values": lambda: on(6)}, "bias_values must be"),
    ({"allowed": lambda: i32(3, 2)}, "needs 3 words"),
    ({"allowed": lambda: i32(2, 3)}, "a mask for every row"),
    ({"allowed_row": lambda: i32(3)}, "allowed_row needs allowed"),
    ({"out": lambda: on(3, 71)}, "out must match the logits"),
    ({"out": lambda: on(1, 70).expand(3, 70)}, "must not overlap"),
])
def test_rules_refuse(change, words):
    kw = {"logits": lambda: on(3, 70), "history": lambda: i32(3, 9), "lengths": lambda: i32(3), "repetition": lambda: on(3), **change}
    kw = {k: v() for k, v in kw.items() if v is not None}
    refused(lambda: edit_logits(kw.pop("logits"), **kw), words)


def test_rules_on_nothing_launch_nothing():
    assert edit_logits(on(0, 70)).shape == (0, 70) and edit_logits(on(3, 0)).shape == (3, 0)


# --------------------------------------------------------------------------- outputs that share memory with inputs
class At:
    """A tensor's place, for the check of overlaps (a pretended tensor has no address)."""

    def __init__(self, first, shape, strides, size=4):
        self.first, self.shape, self.strides, self.size = first, shape, strides, size

    data_ptr = lambda self: self.first                    # noqa: E731
    stride = lambda self: self.strides                    # noqa: E731
    element_size = lambda self: self.size                 # noqa: E731

    def numel(self):
        return self.shape[0] * self.shape[1]


def test_overlaps():
    a = At(1000, (4, 8), (8, 1))
    K._same_place(a, At(1000, (4, 8), (8, 1)), "out")                     # one and the same
    K._same_place(a, At(1128, (4, 8), (8, 1)), "out")                     # behind it
    K._apart(a, At(872, (4, 8), (8, 1)), "out and x")
    for b in (At(1004, (4, 8), (8, 1)), At(1000, (4, 8), (9, 1)), At(900, (4, 8), (8, 1))):
        refused(lambda b=b: K._same_place(a, b, "out"), "must not share memory")
        refused(lambda b=b: K._apart(a, b, "out and x"), "must not share memory")


def test_scratch_of_adapters_never_wraps_round():
    """More than 2^31 pieces of 256 bytes are asked for as the most there are (which nobody has), not as a few."""
    import ctypes

    from logssms_b200.ops import build
    f = build.load("adapters").lb_adapters_scratch
    p, n, i = ctypes.c_void_p, ctypes.c_long, ctypes.c_int
    f.argtypes = [p, n, p, n, p, n, n, p, n, n, p, n, n, i, i, i, i, i]
    pieces = lambda rows, rank, count, code: f(0, 64, 0, 64, 0, 64 * rank, 64, 0, 64 * rank, rank, 0, 64, rows, 64, 64, rank, count, code)      # noqa: E731
    assert pieces(100, 8, 1, 0) == 4 * 100 * 8 // 256 + 1 and pieces(100, 8, 3, 1) == 0
    assert pieces(1 << 24, 1 << 24, 1, 0) == pieces(1 << 30, 1 << 29, 1, 0) == 0x7fffffff
