"""Rules on logits where a row's vocabulary is several slices and its history too long for 16-bit counters (a capacity above 32,767)."""
import pytest
import torch

from test_logit_rules_gpu import check, ints

pytestmark = pytest.mark.gpu


def draw(rows, vocab, capacity, longest):
    g = torch.Generator().manual_seed(rows + vocab)
    history = torch.randint(-1, vocab + 1, (rows, capacity), generator=g, dtype=torch.int32)
    lengths = torch.randint(0, longest + 1, (rows,), generator=g, dtype=torch.int32)
    lengths[-1] = longest
    pen = torch.rand((3, rows), generator=g)
    kw = {"history": history, "lengths": lengths, "prompt_lengths": (lengths * 0.6).int(), "repetition": 0.7 + pen[0], "frequency": pen[1] - 0.3,
          "presence": pen[2] - 0.3, "allowed": torch.randint(-2 ** 31, 2 ** 31 - 1, (rows, -(-vocab // 32)), generator=g, dtype=torch.int64).int()}
    biases = [[(int(i), float(v)) for i, v in zip(torch.randint(0, vocab, (5 * (r % 3),), generator=g), torch.randn(15, generator=g))] for r in range(rows)]
    return (torch.randn((rows, vocab), generator=g) * 3).cuda(), {k: v.cuda() for k, v in kw.items()}, biases


# Slices of 2,048 tokens for few rows, of 4,096 and 8,192 for more; of 16,384 at most with 16-bit counters.
@pytest.mark.parametrize("rows,vocab", [(1, 70001), (3, 32784), (40, 33001), (160, 24577)])
@pytest.mark.parametrize("capacity", [40000, 900])
def test_several_slices(rows, vocab, capacity):
    logits, kw, biases = draw(rows, vocab, capacity, 300)
    check(logits, biases, **kw)


@pytest.mark.parametrize("shift", [0, 1, 2, 3])
@pytest.mark.parametrize("capacity", [40000, 900])
def test_several_slices_of_rows_off_16_bytes(shift, capacity):
    logits, kw, biases = draw(5, 9001, capacity, 500)
    view = torch.zeros((5, 9012), device="cuda")[:, shift:shift + 9001]
    view.copy_(logits)
    check(view, biases, **kw)


def test_a_history_that_is_full():
    """40,000 ids, the ends of slices among them."""
    vocab = 20000
    ids = [0, 1, 2, 3, 4, 2047, 2048, 2049, 4095, 4096, 8191, 8192, 8195, 16383, 16384, 19999]
    logits, kw, _ = draw(2, vocab, 40000, 0)
    kw["history"] = torch.tensor(ids, dtype=torch.int32, device="cuda").repeat(2, 2500)
    kw["lengths"], kw["prompt_lengths"] = ints([40000, 39999]), ints([1, 20000])
    kw["frequency"] = kw["frequency"] * 1e-3
    check(logits, **kw)
