"""The serving operators as a decode step uses them, one behind the other: adapted projections, rotation and store, attention over the
shared prefix, adapted output projection, logits, rules, a token.  Each stage against 64 bits on what the stage before it left."""
import pytest
import torch

from serving_util import adapters, adapters_error, rules, shared_attention, shared_attention_error

pytestmark = pytest.mark.gpu

HQ, HKV, HD, HIDDEN, VOCAB, PAGE, RANK = 8, 2, 64, 512, 3001, 64, 8


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Batch:
    """Seven requests: four that share 200 tokens, two that share 70, one by itself; adapters 0 .. 2 or none; rules of all kinds."""

    def __init__(self, dtype):
        g = torch.Generator().manual_seed(17)
        r = lambda *s, size=1.0: (torch.randn(s, generator=g) * size).to(dtype).cuda()          # noqa: E731
        self.dtype = dtype
        self.prefix, members, self.own = [200, 70, 0], [4, 2, 1], [1, 30, 70, 5, 9, 1, 40]
        n = sum(members)
        self.x, self.w_qkv, self.w_o = r(n, HIDDEN), r((HQ + 2 * HKV) * HD, HIDDEN, size=HIDDEN ** -0.5), r(HIDDEN, HQ * HD, size=(HQ * HD) ** -0.5)
        self.head = r(VOCAB, HIDDEN, size=3 * HIDDEN ** -0.5)
        self.a_qkv, self.b_qkv = r(3, RANK, HIDDEN, size=HIDDEN ** -0.5), r(3, (HQ + 2 * HKV) * HD, RANK, size=0.3)
        self.a_o, self.b_o = r(3, RANK, HQ * HD, size=(HQ * HD) ** -0.5), r(3, HIDDEN, RANK, size=0.3)
        self.index, self.scales = ints([0, 2, -1, 0, 1, 1, 2]), torch.tensor([1.0, 0.5, 2.0], device="cuda")
        pages = 40
        self.k, self.v = r(pages, PAGE, HKV, HD), r(pages, PAGE, HKV, HD)
        table, free, starts, pos = torch.zeros((n, 6), dtype=torch.int32), list(range(pages)), [0], []
        row = 0
        for p, m in zip(self.prefix, members):
            shared = [free.pop() for _ in range(p // PAGE)]
            tail = None
            for _ in range(m):
                end = p + self.own[row]
                mine = [free.pop() for _ in range(-(-end // PAGE) - len(shared))]
                table[row, :len(shared) + len(mine)] = torch.tensor(shared + mine, dtype=torch.int32)
                if p % PAGE and tail is not None:                     # a copy of the prefix's last keys
                    for c in (self.k, self.v):
                        c[mine[0], :p % PAGE] = c[tail, :p % PAGE]
                tail = mine[0] if tail is None and mine else tail
                pos.append(end - 1)
                row += 1
            starts.append(row)
        self.table, self.starts, self.prefixes, self.positions = table.cuda(), ints(starts), ints(self.prefix), ints(pos)
        self.slots = ints([int(table[i, p // PAGE]) * PAGE + p % PAGE for i, p in enumerate(pos)])
        self.req = ints(list(range(n)))
        from logssms_b200.ops import kernels as K
        inv = 1.0 / (10000.0 ** (torch.arange(0, HD, 2).float() / HD))
        self.rope = K.rope_table(inv.cuda(), 400)
        self.history = torch.randint(0, VOCAB, (n, 64), generator=g, dtype=torch.int32).cuda()
        self.rules = {"history": self.history, "lengths": ints([64, 3, 0, 40, 9, 64, 1]), "prompt_lengths": ints([50, 3, 0, 0, 4, 64, 0]),
                      "repetition": torch.rand(n, generator=g).cuda() + 0.7, "frequency": torch.rand(n, generator=g).cuda(),
                      "presence": torch.rand(n, generator=g).cuda(),
                      "allowed": torch.randint(-2 ** 31, 2 ** 31 - 1, (2, 94), generator=g, dtype=torch.int64).int().cuda(),
                      "allowed_row": ints([-1, 0, -1, 1, -1, 0, -1])}
        self.biases = [[(5, 1.0), (2999, -3.0)], [], [(7, 100.0)], [], [], [], [(0, float("-inf"))]]

    def step(self, keep=None):
        from logssms_b200.ops import kernels as K
        from logssms_b200.sampling import edit_logits, sample_tokens
        keep = {} if keep is None else keep
        keep["qkv0"] = K.linear(self.x, self.w_qkv)
        keep["qkv"] = K.add_adapters(keep["qkv0"], self.x, self.a_qkv, self.b_qkv, self.index, self.scales)
        keep["q"] = K.rope_kv_store(keep["qkv"], HQ, HKV, HD, self.positions, self.slots, self.rope, self.k, self.v, 1.0)
        keep["o"] = K.attention_decode_shared(keep["q"], self.k, self.v, self.table, self.req, self.positions, self.starts, self.prefixes,
                                              HD ** -0.5, max_prefix=200, max_context=400)
        flat = keep["o"].view(len(self.own), HQ * HD)
        keep["y0"] = K.linear(flat, self.w_o)
        keep["y"] = K.add_adapters(keep["y0"], flat, self.a_o, self.b_o, self.index, self.scales)
        keep["logits0"] = K.linear_f32(keep["y"], self.head)
        starts = [0]
        for b in self.biases:
            starts.append(starts[-1] + len(b))
        if not hasattr(self, "listed"):
            self.listed = {"bias_start": ints(starts), "bias_ids": ints([i for b in self.biases for i, _ in b]),
                           "bias_values": torch.tensor([v for b in self.biases for _, v in b], device="cuda")}
        keep["logits"] = edit_logits(keep["logits0"], **self.rules, **self.listed)
        keep["ids"] = sample_tokens(keep["logits"], None, None, None, None, None)
        return keep


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_decode_step_stage_by_stage_and_replayed(dtype):
    from logssms_b200.ops import kernels as K
    b = Batch(dtype)
    kept = b.step()
    for y0, y, x, a, w in ((kept["qkv0"], kept["qkv"], b.x, b.a_qkv, b.b_qkv), (kept["y0"], kept["y"], kept["o"].view(7, -1), b.a_o, b.b_o)):
        want, size = adapters(*(t.cpu() for t in (y0, x, a, w, b.index, b.scales)))
        assert bool(((y.cpu().double() - want).abs() <= adapters_error(y0.cpu(), want, size, x.shape[1], RANK, dtype)).all())
    want, size, reach = shared_attention(*(t.cpu() for t in (kept["q"], b.k, b.v, b.table, b.req, b.positions)), HD ** -0.5)
    assert bool(((kept["o"].cpu().double() - want).abs() <= shared_attention_error(want, size, reach, HD, dtype)).all())
    want, size = rules(kept["logits0"].cpu(), biases=b.biases, **{k: v.cpu() for k, v in b.rules.items()})
    got = kept["logits"].cpu()
    fine = want.isfinite()
    assert torch.equal(got.isfinite(), fine)
    assert bool((torch.where(fine, (got.double() - want).abs(), 0.0) <= 6 * 2.0 ** -24 * size).all())
    assert kept["ids"].tolist() == kept["logits"].argmax(1).tolist()
    K.check_kernel_errors()
    graph, held = torch.cuda.CUDAGraph(), {}
    with torch.cuda.graph(graph):
        b.step(held)
    for _ in range(2):                                               # (the step stores the same keys at the same places)
        graph.replay()
        assert all(torch.equal(held[name], kept[name]) for name in kept)
    b.x.copy_(b.x.flip(0))                                           # another token of each request
    graph.replay()
    again = b.step()
    assert all(torch.equal(held[name], again[name]) for name in kept)
    assert not torch.equal(again["logits"], kept["logits"])
