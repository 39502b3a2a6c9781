"""Rules on logits (`logit_rules.cu`) against 64 bits: penalties, biases and masks by themselves and together, at every alignment."""
import pytest
import torch

from serving_util import rules

pytestmark = pytest.mark.gpu


def edit(*args, **kw):
    from logssms_b200.sampling import edit_logits
    return edit_logits(*args, **kw)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def floats(values):
    return torch.tensor(values, dtype=torch.float32, device="cuda")


def listed(biases):
    """The flat form of per-row lists."""
    starts = [0]
    for b in biases:
        starts.append(starts[-1] + len(b))
    return {"bias_start": ints(starts), "bias_ids": ints([i for b in biases for i, _ in b]), "bias_values": floats([v for b in biases for _, v in b])}


def agree(got, want, size):
    """Equal infinities and NaN; the others within six roundings of 32 bits of what was added."""
    want = want.to(got.device)
    want = torch.where(want.float().isinf(), want.float().double(), want)          # (past 32 bits' largest number: that infinity)
    fine = want.isfinite()
    assert torch.equal(got.isfinite(), fine) and torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[~fine & ~want.isnan()].double(), want[~fine & ~want.isnan()])
    off = torch.where(fine, (got.double() - want).abs(), 0.0)
    assert bool((off <= 6 * 2.0 ** -24 * size.to(got.device) + 1e-42).all())


def check(logits, biases=None, **kw):
    want, size = rules(logits.cpu(), biases=biases, **{k: v.cpu() for k, v in kw.items()})
    more = listed(biases) if biases is not None else {}
    kept = logits.clone()
    agree(edit(logits, **kw, **more), want, size)
    assert torch.equal(logits.nan_to_num(nan=7.0), kept.nan_to_num(nan=7.0))
    own = logits.clone()
    assert edit(own, **kw, **more, out=own) is own
    agree(own, want, size)


def draw(rows, vocab, capacity, seed=0):
    g = torch.Generator().manual_seed(seed + 1000 * rows + vocab)
    logits = torch.randn((rows, vocab), generator=g) * 3
    history = (vocab * torch.rand((rows, capacity), generator=g) ** 3).int()
    lengths = torch.randint(0, capacity + 1, (rows,), generator=g, dtype=torch.int32)
    prompts = (lengths.float() * torch.rand((rows,), generator=g)).int()
    pen = torch.rand((3, rows), generator=g)
    return logits.cuda(), {"history": history.cuda(), "lengths": lengths.cuda(), "prompt_lengths": prompts.cuda(),
                           "repetition": (0.7 + pen[0]).cuda(), "frequency": (pen[1] - 0.3).cuda(), "presence": (pen[2] - 0.3).cuda()}


@pytest.mark.parametrize("rows,vocab,capacity", [(1, 1, 1), (1, 3, 5), (2, 33, 7), (3, 64, 40), (5, 1003, 130), (2, 4099, 300),
                                                 (17, 2051, 64), (1, 32784, 500), (3, 70001, 900)])
def test_penalties(rows, vocab, capacity):
    logits, kw = draw(rows, vocab, capacity)
    check(logits, **kw)
    check(logits, history=kw["history"], lengths=kw["lengths"], repetition=kw["repetition"])
    check(logits, history=kw["history"], lengths=kw["lengths"], frequency=kw["frequency"])
    check(logits, history=kw["history"], lengths=kw["lengths"], prompt_lengths=kw["prompt_lengths"], presence=kw["presence"])


def test_many_rows_share_long_slices():
    logits, kw = draw(160, 33001, 50)                  # (enough CTAs for slices of 32,768 tokens)
    check(logits, **kw)


def test_counts_past_16_bits():
    """A history whose capacity a 16-bit counter could not hold, and one token that fills it."""
    logits = torch.randn((2, 300), generator=torch.Generator().manual_seed(3)).cuda()
    history = torch.full((2, 70000), 7, dtype=torch.int32, device="cuda")
    history[1, ::2] = 299
    check(logits, history=history, lengths=ints([70000, 69999]), prompt_lengths=ints([1, 30000]), frequency=floats([1e-4, 2e-4]),
          presence=floats([0.5, 0.1]), repetition=floats([1.2, 1.0]))
    full = torch.full((1, 32767), 5, dtype=torch.int32, device="cuda")        # and the most that 16 bits hold
    check(logits[:1], history=full, lengths=ints([32767]), frequency=floats([1e-3]))


def test_history_alignment_strides_slots_and_foreign_ids():
    logits, kw = draw(6, 517, 44)
    wide = torch.randint(0, 517, (9, 61), generator=torch.Generator().manual_seed(1), dtype=torch.int32).cuda()
    wide[:, 3], wide[:, 9], wide[:, 11] = -1, 517, 1 << 30
    for first in range(5):
        kw["history"] = wide[:, first:first + 44]
        check(logits, **kw, slots=ints([8, 0, 0, -1, 9, 3]))


def test_lengths_past_the_capacity_and_below_zero():
    logits, kw = draw(4, 100, 20)
    kw["lengths"], kw["prompt_lengths"] = ints([-5, 1000, 20, 0]), ints([4, -3, 1000, 2])
    check(logits, **kw)


def test_logits_with_infinities_and_nan():
    logits, kw = draw(2, 99, 300)
    logits[0, ::3], logits[0, 1], logits[1, 5], logits[1, 7] = float("-inf"), float("inf"), float("nan"), 0.0
    check(logits, **kw)
    check(logits, **kw, allowed=torch.zeros((2, 4), dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 1001, 5003])
def test_masks(vocab):
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn((6, vocab), generator=g).cuda()
    words = -(-vocab // 32)
    allowed = torch.randint(-2 ** 31, 2 ** 31 - 1, (3, words + 2), generator=g, dtype=torch.int64).int().cuda()
    allowed[1] = 0                                     # allows nothing
    check(logits, allowed=allowed, allowed_row=ints([2, 0, -1, 1, 3, 1]))
    check(logits[:3], allowed=allowed[:, :words])
    assert bool((edit(logits, allowed=allowed, allowed_row=ints([1] * 6)) == float("-inf")).all())


@pytest.mark.parametrize("shift", [0, 1, 2, 3])
def test_rows_that_begin_off_a_16_byte_boundary(shift):
    logits, kw = draw(3, 1003, 60)
    wide = torch.zeros((3, 1016), device="cuda")
    view = wide[:, shift:shift + 1003]
    view.copy_(logits)
    allowed = torch.randint(-2 ** 31, 2 ** 31 - 1, (3, 32), generator=torch.Generator().manual_seed(1), dtype=torch.int64).int().cuda()
    biases = [[(0, 1.0), (1, 2.0), (1002, 3.0)], [], [(5, -4.0), (2, 0.5)]]
    check(view, biases, **kw, allowed=allowed)
    out = torch.full((3, 1024), 5.0, device="cuda")     # in and out differ within 16 bytes
    want, size = rules(logits.cpu(), biases=biases, allowed=allowed.cpu(), **{k: v.cpu() for k, v in kw.items()})
    agree(edit(view, **kw, **listed(biases), allowed=allowed, out=out[:, 8:1011]), want, size)
    assert bool((out[:, :8] == 5).all()) and bool((out[:, 1011:] == 5).all())


def test_biases_of_the_same_token_are_added_in_their_order():
    logits = torch.randn((3, 700), generator=torch.Generator().manual_seed(2)).cuda()
    g = torch.Generator().manual_seed(9)
    many = [(int(i), float(v)) for i, v in zip(torch.randint(0, 40, (500,), generator=g), torch.randn(500, generator=g) * 100)]
    biases = [many, [(3, 1.0), (3, 1e8), (3, -1e8), (699, 2.0)], [(-1, 5.0), (700, 5.0), (0, float("-inf"))]]
    more = listed(biases)
    want = logits.clone().cpu()
    for r, b in enumerate(biases):
        for i, v in b:
            if 0 <= i < 700:
                want[r, i] = want[r, i] + torch.tensor(v)           # 32-bit, one after the other
    for _ in range(3):
        assert torch.equal(edit(logits, **more).cpu(), want)


def test_a_mask_wins_over_a_bias_and_an_infinite_logit():
    logits = torch.zeros((1, 64), device="cuda")
    logits[0, 3] = float("inf")
    allowed = ints([[~(1 << 3) & 0x7fffffff, -1]])
    got = edit(logits, **listed([[(3, 5.0), (31, 9.0), (40, 2.0)]]), allowed=allowed)
    assert float(got[0, 3]) == float("-inf") and float(got[0, 31]) == float("-inf") and float(got[0, 40]) == 2.0


def test_everything_together_on_another_stream_and_in_a_graph():
    logits, kw = draw(7, 9001, 200)
    allowed = torch.randint(-2 ** 31, 2 ** 31 - 1, (7, 282), generator=torch.Generator().manual_seed(4), dtype=torch.int64).int().cuda()
    biases = [[(i * 13 % 9001, 0.5 * i) for i in range(r * 40)] for r in range(7)]
    more = listed(biases)
    want, size = rules(logits.cpu(), biases=biases, allowed=allowed.cpu(), **{k: v.cpu() for k, v in kw.items()})
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = edit(logits, **kw, **more, allowed=allowed)
    torch.cuda.current_stream().wait_stream(stream)
    agree(got, want, size)
    graph, held = torch.cuda.CUDAGraph(), torch.empty_like(logits)
    with torch.cuda.graph(graph):
        edit(logits, **kw, **more, allowed=allowed, out=held)
    held.zero_()
    graph.replay()
    assert torch.equal(held, got)
    kw["lengths"].zero_()                              # the graph reads the rows' present state
    graph.replay()
    want, size = rules(logits.cpu(), biases=biases, allowed=allowed.cpu(), **{k: v.cpu() for k, v in kw.items()})
    agree(held, want, size)


def test_nothing_to_do_copies_and_empty_calls_return():
    logits = torch.randn((3, 50), generator=torch.Generator().manual_seed(1)).cuda()
    got = edit(logits)
    assert torch.equal(got, logits) and got.data_ptr() != logits.data_ptr()
    assert edit(logits[:0]).shape == (0, 50)
    assert edit(torch.zeros((2, 0), device="cuda")).shape == (2, 0)


def test_the_binding_and_the_ordinary_way_are_the_same_call():
    logits, kw = draw(5, 4099, 300)
    more = listed([[(1, 2.0)], [], [(3, -1.0), (3, 5.0)], [], []])
    got = edit(logits, **kw, **more)
    assert torch.equal(got, edit(logits, **kw, **more, out=torch.empty_like(logits)))


def test_extreme_penalties():
    """Quotients by the inverse and its remainder: numbers of every size, infinities, zero, a repetition of zero and infinity."""
    l = torch.tensor([[1e-30, 3e38, -3e38, float("inf"), float("-inf"), 0.0, -0.0, 1.0, 7.0, 1e30]] * 4, device="cuda")
    history = torch.arange(10, dtype=torch.int32, device="cuda").expand(4, 10).contiguous()
    for rep in ([1.3, 0.7, 3.0, 1e3], [1e-3, 1e10, 7.0, 0.9]):
        check(l, history=history, lengths=ints([10] * 4), prompt_lengths=ints([10] * 4), repetition=floats(rep))
    got = edit(l, history=history, lengths=ints([10] * 4), repetition=floats([0.0, float("inf"), float("nan"), 1.0]))
    assert float(got[0, 7]) == float("inf") and float(got[1, 7]) == 0.0 and bool(got[2].isnan().all()) and torch.equal(got[3], l[3])
