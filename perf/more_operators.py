"""Operators of a decode step whose requests share one thing and own another, one call at a time, for measuring them.

Three operators: attention of a batch whose requests begin with the same tokens, which reads the keys of that prefix once for
all of them (`attention`); what low-rank adapters, one per request, add to a projection that all share (`adapters`); and each
request's own rules on its logits: penalties for tokens that it has seen, biases, a mask of allowed tokens (`logits`).

Sizes are those of this repository's benchmark models (8 heads of 64 over 2, 6 and 12 heads of 128 over 2, vocabularies of
32,784 / 65,536 / 130,048, hidden sizes 1,024 and 1,280, pages of 64 tokens), its batch sizes and prompt lengths, and odd ones.
"""
from __future__ import annotations

import math
import random

import torch

own = False             # whether `run` calls the framework's kernels

_DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _attention(name, requests, per_request, groups, prefix, own_keys, heads, kv_heads, head_dim, page, dtype):
    case = {"op": "attention", "requests": requests, "per_request": per_request, "groups": groups, "prefix": prefix,
            "own_keys": own_keys, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype}
    return {"name": name, **case} if name else case


def _adapters(name, rows, width, features, adapters, rank, mixed, without, dtype):
    case = {"op": "adapters", "rows": rows, "width": width, "features": features, "adapters": adapters, "rank": rank,
            "mixed": mixed, "without": without, "dtype": dtype}
    return {"name": name, **case} if name else case


def _logits(name, rows, vocab, history, biases, masked):
    case = {"op": "logits", "rows": rows, "vocab": vocab, "history": history, "biases": biases, "masked": masked}
    return {"name": name, **case} if name else case


def listed():
    return [
        # four samples of one user's chat, the smallest model
        _attention("attention-4", 4, 1, 1, 640, 40, 8, 2, 64, 64, "bfloat16"),
        # a full server whose requests share a system prompt, the largest model's heads
        _attention("attention-64-2048", 64, 1, 1, 2048, 512, 12, 2, 128, 64, "bfloat16"),
        # many questions about one long document, the most work
        _attention("attention-256-32768", 256, 1, 1, 32768, 2048, 12, 2, 128, 64, "bfloat16"),
        # a float32 engine with small pages, five prompts with several samples each, two new tokens per request
        _attention("attention-groups-odd", 23, 2, 5, 1531, 203, 6, 2, 128, 16, "float32"),
        # one user with a tuned adapter, the smallest model's gate|up
        _adapters("adapters-1", 1, 1024, 4096, 1, 16, False, 0.0, "bfloat16"),
        # a full server whose every request has an adapter of its own
        _adapters("adapters-64-own", 64, 4096, 4096, 64, 16, True, 0.1, "bfloat16"),
        # a full prompt step: eight requests' portions, each with its adapter
        _adapters("adapters-prompt-8192", 8192, 4096, 12288, 8, 64, False, 0.0, "bfloat16"),
        # a float32 engine, sizes that are multiples of nothing, ranks that differ, rows without an adapter
        _adapters("adapters-203-odd", 203, 1003, 1431, 5, 13, True, 0.3, "float32"),
        # one user's chat, the smallest model
        _logits("logits-1", 1, 32784, 700, 0, 0.0),
        # a full server, half of whose requests answer in a grammar, the largest model
        _logits("logits-64-grammar", 64, 130048, 4096, 300, 0.5),
        # the largest batch, long histories
        _logits("logits-256", 256, 130048, 16384, 0, 0.1),
        # an odd vocabulary, short histories
        _logits("logits-17-odd", 17, 50257, 333, 17, 0.3),
    ]


def _between(rng, low, high):
    """A size from low to high, spread over its logarithm; a third of them rounded to a multiple of 64."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.33 and n >= 64:
        n = n // 64 * 64
    return max(low, min(high, n))


def draw(rng):
    op = rng.choice(["attention", "adapters", "logits"])
    if op == "attention":
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        requests = _between(rng, 1, 256 if dtype == "bfloat16" else 64)
        per_request = rng.choice([1, 1, 2, 4]) if requests <= 64 else 1
        heads = rng.choice([(8, 2, 64), (6, 2, 128), (12, 2, 128), (4, 4, 64), (16, 1, 96)])
        return _attention(None, requests, per_request, min(requests, rng.choice([1, 1, 2, 3, 7])),
                          _between(rng, 1, 32768 if dtype == "bfloat16" else 8192), _between(rng, 1, 2048), *heads,
                          rng.choice([16, 64, 128]), dtype)
    if op == "adapters":
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        return _adapters(None, _between(rng, 1, 8192 if dtype == "bfloat16" else 4096), _between(rng, 64, 4096),
                         _between(rng, 64, 12288), _between(rng, 1, 64), rng.choice([8, 16, 32, 64, rng.randint(1, 64)]),
                         rng.random() < 0.4, rng.choice([0.0, 0.2]), dtype)
    return _logits(None, _between(rng, 1, 256), _between(rng, 1000, 130048), _between(rng, 1, 16384), rng.choice([0, _between(rng, 1, 300)]),
                   rng.choice([0.0, 0.5, 1.0]))


# ------------------------------------------------------------------ how long everything is, by the case alone
def _lengths(case):
    """Of an attention case: per group its first request and the one behind its last, its prefix; per request its own keys."""
    n, g = case["requests"], case["groups"]
    starts = [i * n // g for i in range(g + 1)]
    prefixes = [max(1, case["prefix"] * (2 * g - i) // (2 * g)) for i in range(g)]
    own_keys = [max(case["per_request"], 1 + int((case["own_keys"] - 1) * ((0.618 * (i + 1)) % 1.0))) for i in range(n)]
    own_keys[-1] = max(own_keys[-1], case["own_keys"])
    return starts, prefixes, own_keys


def _histories(case):
    """Of a logits case: per row how many ids it has seen, and how many of them are its prompt's."""
    lengths = [int(case["history"] * ((0.618 * (i + 1)) % 1.0)) for i in range(case["rows"])]
    lengths[-1] = case["history"]
    return lengths, [2 * n // 3 for n in lengths]


def _masked_rows(case):
    return round(case["rows"] * case["masked"])


# ------------------------------------------------------------------ inputs
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_attention(case, gen, rng):
    dtype, page, hd, kv_heads = _DTYPES[case["dtype"]], case["page"], case["head_dim"], case["kv_heads"]
    starts, prefixes, own_keys = _lengths(case)
    n, per = case["requests"], case["per_request"]
    longest = max(prefixes) + max(own_keys)
    columns = -(-longest // page)
    need = sum(p // page for p in prefixes)
    group_of = [g for g in range(case["groups"]) for _ in range(starts[g], starts[g + 1])]
    for r in range(n):
        p = prefixes[group_of[r]]
        need += -(-(p + own_keys[r]) // page) - p // page
    free = list(range(need + 3))                     # a few pages are other requests'
    rng.shuffle(free)
    table = [[0] * columns for _ in range(n)]
    copies = []                                      # (page, page): a prefix's last keys, which every request has in a page of its own
    for g, p in enumerate(prefixes):
        shared = [free.pop() for _ in range(p // page)]
        first = None
        for r in range(starts[g], starts[g + 1]):
            mine = [free.pop() for _ in range(-(-(p + own_keys[r]) // page) - len(shared))]
            table[r][:len(shared) + len(mine)] = shared + mine
            if p % page:
                if first is None:
                    first = mine[0]
                else:
                    copies.append((first, mine[0], p % page))
    k_cache = torch.randn((need + 3, page, kv_heads, hd), generator=gen, device="cuda").to(dtype)
    v_cache = torch.randn((need + 3, page, kv_heads, hd), generator=gen, device="cuda").to(dtype)
    if copies:
        src, dst, keys = copies[0][0], [c[1] for c in copies], [c[2] for c in copies]
        src = torch.tensor([c[0] for c in copies], device="cuda")
        dst = torch.tensor(dst, device="cuda")
        within = (torch.arange(page, device="cuda")[None, :] < torch.tensor(keys, device="cuda")[:, None])[:, :, None, None]
        for cache in (k_cache, v_cache):
            cache[dst] = torch.where(within, cache[src], cache[dst])
    ends = [prefixes[group_of[r]] + own_keys[r] for r in range(n)]
    positions = [e - per + i for e in ends for i in range(per)]
    q = torch.randn((n * per, case["heads"], hd), generator=gen, device="cuda") * 1.5
    return {"q": q.to(dtype), "k_cache": k_cache, "v_cache": v_cache, "block_table": _ints(table),
            "token_req": _ints([r for r in range(n) for _ in range(per)]), "positions": _ints(positions),
            "group_start": _ints([s * per for s in starts]), "prefix_lens": _ints(prefixes), "scale": hd ** -0.5,
            "max_prefix": max(prefixes), "max_context": longest}


def _prepare_adapters(case, gen, rng):
    dtype, rows, n, rank = _DTYPES[case["dtype"]], case["rows"], case["adapters"], case["rank"]

    def normal(*shape, size):
        return (torch.randn(shape, generator=gen, device="cuda") * size).to(dtype)

    if case["mixed"]:                                # decoding requests, in any order
        index = [rng.randrange(n) for _ in range(rows)]
        if n >= rows:
            index = rng.sample(range(n), rows)
    else:                                            # portions of prompts, one behind the other
        index = [i * n // rows for i in range(rows)]
    index = [-1 if rng.random() < case["without"] else a for a in index]
    ranks = [rank if i % 3 == 0 or not case["mixed"] else max(1, rank // (1 + i % 3)) for i in range(n)]
    return {"y": normal(rows, case["features"], size=1.0), "x": normal(rows, case["width"], size=1.0),
            "a": normal(n, rank, case["width"], size=case["width"] ** -0.5), "b": normal(n, case["features"], rank, size=0.5 * rank ** -0.5),
            "index": _ints(index), "scales": torch.rand((n,), generator=gen, device="cuda") + 0.5, "ranks": _ints(ranks)}


def _prepare_logits(case, gen, rng):
    rows, vocab = case["rows"], case["vocab"]
    lengths, prompts = _histories(case)
    logits = torch.randn((rows, vocab), generator=gen, device="cuda") * 3.0
    # words of a text: few of them make up most of it
    words = (vocab * torch.rand((rows, max(max(lengths), 1)), generator=gen, device="cuda") ** 4).int().clamp(max=vocab - 1)
    state = {"logits": logits, "history": words, "lengths": _ints(lengths), "prompt_lengths": _ints(prompts),
             "repetition": 1.0 + 0.3 * torch.rand((rows,), generator=gen, device="cuda"),
             "frequency": 0.5 * torch.rand((rows,), generator=gen, device="cuda"),
             "presence": 0.5 * torch.rand((rows,), generator=gen, device="cuda"),
             "bias_start": None, "bias_ids": None, "bias_values": None, "allowed": None, "allowed_row": None}
    n = min(case["biases"], vocab)
    if n:
        # every other row has biases, of different tokens
        counts = [n if i % 2 == 0 else 0 for i in range(rows)]
        starts = [sum(counts[:i]) for i in range(rows + 1)]
        state["bias_start"] = _ints(starts)
        state["bias_ids"] = _ints([t for c in counts for t in rng.sample(range(vocab), c)])
        state["bias_values"] = torch.randn((starts[-1],), generator=gen, device="cuda") * 4.0
    masked = _masked_rows(case)
    if masked:
        # a grammar allows some hundredth of the tokens in one state and nearly all (inside a string) in another
        words_per_row = -(-vocab // 32)
        few = torch.rand((masked, 1, 1), generator=gen, device="cuda") < 0.5
        bits = torch.rand((masked, words_per_row, 32), generator=gen, device="cuda") < torch.where(few, 0.01, 0.9)
        weights = torch.tensor([1 << i for i in range(31)] + [-(1 << 31)], dtype=torch.int64, device="cuda")
        state["allowed"] = (bits * weights).sum(2).int()
        state["allowed_row"] = _ints(rng.sample(range(masked), masked) + [-1] * (rows - masked))
    return state


def prepare(case, seed):
    gen, rng = torch.Generator("cuda").manual_seed(seed), random.Random(seed)
    made = {"attention": _prepare_attention, "adapters": _prepare_adapters, "logits": _prepare_logits}[case["op"]]
    return {"op": case["op"], **made(case, gen, rng)}


# ------------------------------------------------------------------ one pass
def _plain_attention(s):
    """Every token on its own over its request's keys, filled up to the longest."""
    q, page = s["q"].float(), s["k_cache"].shape[1]
    tokens, heads, hd = q.shape
    kv_heads = s["k_cache"].shape[2]
    j = torch.arange(s["max_context"], device=q.device)
    slots = s["block_table"].long()[:, j // page] * page + j % page                     # [requests, keys]
    slots = slots[s["token_req"].long()]                                                # [tokens, keys]
    k = s["k_cache"].view(-1, kv_heads, hd)[slots].float()                              # [tokens, keys, kv heads, hd]
    v = s["v_cache"].view(-1, kv_heads, hd)[slots].float()
    scores = torch.einsum("tgnd,tkgd->tgnk", q.view(tokens, kv_heads, heads // kv_heads, hd), k) * s["scale"]
    later = j[None, :] > s["positions"][:, None]
    scores = scores.masked_fill(later[:, None, None, :], float("-inf"))
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.einsum("tgnk,tkgd->tgnd", weights, v) / weights.sum(-1, keepdim=True)
    return {"out": out.reshape(tokens, heads, hd).to(s["q"].dtype)}


def _plain_adapters(s):
    """All adapters' parts of every row, of which each row keeps its own."""
    n, rank, width = s["a"].shape
    x, index = s["x"].float(), s["index"]
    h = (x @ s["a"].float().reshape(n * rank, width).t()).view(-1, n, rank)
    keep = (index[:, None] == torch.arange(n, device=index.device))[:, :, None]
    keep = keep & (torch.arange(rank, device=index.device) < s["ranks"][:, None])
    h = torch.where(keep, h * s["scales"][:, None], 0.0).view(-1, n * rank)
    return {"out": (s["y"].float() + h @ s["b"].float().transpose(1, 2).reshape(n * rank, -1)).to(s["y"].dtype)}


def _plain_logits(s):
    logits, history = s["logits"], s["history"].long()
    rows, vocab = logits.shape
    at = torch.arange(history.shape[1], device=logits.device)
    there, answered = at < s["lengths"][:, None], at >= s["prompt_lengths"][:, None]
    zeros = torch.zeros((rows, vocab), device=logits.device)
    seen = zeros.scatter_add(1, history, there.float()) > 0
    count = zeros.scatter_add(1, history, (there & answered).float())
    p = s["repetition"][:, None]
    l = torch.where(seen, torch.where(logits > 0, logits / p, logits * p), logits)
    l = l - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias_start"] is not None:
        row = torch.repeat_interleave(torch.arange(rows, device=l.device), s["bias_start"].diff().long(), output_size=s["bias_ids"].numel())
        l = l.index_put((row, s["bias_ids"].long()), s["bias_values"], accumulate=True)
    if s["allowed"] is not None:
        token = torch.arange(vocab, device=l.device)
        allowed = (s["allowed"][:, token // 32] >> (token % 32)) & 1                   # [masks, vocab]
        row = s["allowed_row"].long()
        l = torch.where((row < 0)[:, None] | (allowed[row.clamp(min=0)] != 0), l, float("-inf"))
    return {"logits": l}


def _framework(s):
    if s["op"] == "attention":
        from logssms_b200.ops import kernels as K
        return {"out": K.attention_decode_shared(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["token_req"], s["positions"],
                                                 s["group_start"], s["prefix_lens"], s["scale"], max_prefix=s["max_prefix"],
                                                 max_context=s["max_context"])}
    if s["op"] == "adapters":
        from logssms_b200.ops import kernels as K
        return {"out": K.add_adapters(s["y"], s["x"], s["a"], s["b"], s["index"], s["scales"], ranks=s["ranks"])}
    from logssms_b200.sampling import edit_logits
    return {"logits": edit_logits(s["logits"], history=s["history"], lengths=s["lengths"], prompt_lengths=s["prompt_lengths"],
                                  repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
                                  bias_start=s["bias_start"], bias_ids=s["bias_ids"], bias_values=s["bias_values"],
                                  allowed=s["allowed"], allowed_row=s["allowed_row"])}


def run(state):
    if own:
        return _framework(state)
    plain = {"attention": _plain_attention, "adapters": _plain_adapters, "logits": _plain_logits}[state["op"]]
    return plain(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "attention":
        size = 2 if case["dtype"] == "bfloat16" else 4
        starts, prefixes, own_keys = _lengths(case)
        per, key = case["per_request"], 2 * case["kv_heads"] * case["head_dim"] * size
        tokens = case["requests"] * per
        pairs = sum((p + k) * per - per * (per - 1) // 2 for g, p in enumerate(prefixes) for k in own_keys[starts[g]:starts[g + 1]])
        return {"bytes": float(2 * tokens * case["heads"] * case["head_dim"] * size + (sum(prefixes) + sum(own_keys)) * key),
                "flops": float(4 * case["heads"] * case["head_dim"] * pairs)}
    if case["op"] == "adapters":
        size = 2 if case["dtype"] == "bfloat16" else 4
        rows, width, features, rank = case["rows"], case["width"], case["features"], case["rank"]
        used = min(case["adapters"], rows) * (1 - case["without"])
        return {"bytes": size * (rows * (width * (1 - case["without"]) + 2 * features) + used * rank * (width + features)),
                "flops": 2.0 * rows * (1 - case["without"]) * rank * (width + features)}
    rows, vocab = case["rows"], case["vocab"]
    biased = min(case["biases"], vocab) * -(-rows // 2)
    return {"bytes": float(8 * rows * vocab + 4 * sum(_histories(case)[0]) + 8 * biased + 4 * _masked_rows(case) * -(-vocab // 32)),
            "flops": float(4 * rows * vocab)}


# ------------------------------------------------------------------ the same in 64 bits
def _exact_attention(case, s):
    starts, prefixes, own_keys = _lengths(case)
    page, per, heads, kv_heads, hd = case["page"], case["per_request"], case["heads"], case["kv_heads"], case["head_dim"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for g, prefix in enumerate(prefixes):
        for r in range(starts[g], starts[g + 1]):
            keys = prefix + own_keys[r]
            pages = s["block_table"][r, :-(-keys // page)].long()
            k = s["k_cache"][pages].flatten(0, 1)[:keys].double().transpose(0, 1)       # [kv heads, keys, hd]
            v = s["v_cache"][pages].flatten(0, 1)[:keys].double().transpose(0, 1)
            q = s["q"][r * per:(r + 1) * per].double().view(per, kv_heads, heads // kv_heads, hd)
            for i in range(per):
                seen = keys - per + 1 + i
                w = torch.softmax(q[i] @ k[:, :seen].transpose(1, 2) * hd ** -0.5, -1)
                out[r * per + i] = (w @ v[:, :seen]).reshape(heads, hd)
    return {"out": out}


def _exact_adapters(case, s):
    out = s["y"].double()
    index = s["index"].tolist()
    for i, (rank, scale) in enumerate(zip(s["ranks"].tolist(), s["scales"].tolist())):
        rows = [t for t, a in enumerate(index) if a == i]
        if rows:
            rows = torch.tensor(rows, device="cuda")
            low = s["x"][rows].double() @ s["a"][i, :rank].double().t()
            out[rows] += scale * (low @ s["b"][i, :, :rank].double().t())
    return {"out": out}


def _exact_logits(case, s):
    l = s["logits"].double()
    lengths, prompts = _histories(case)
    masks = s["allowed_row"].tolist() if s["allowed"] is not None else [-1] * case["rows"]
    for r, (n, p) in enumerate(zip(lengths, prompts)):
        seen = s["history"][r, :n].long().unique()
        if seen.numel():
            v, factor = l[r, seen], s["repetition"][r].double()
            l[r, seen] = torch.where(v > 0, v / factor, v * factor)
        said, times = s["history"][r, p:n].long().unique(return_counts=True)
        l[r, said] -= s["frequency"][r].double() * times + s["presence"][r].double()
        if s["bias_start"] is not None:
            a, b = s["bias_start"][r:r + 2].tolist()
            l[r, s["bias_ids"][a:b].long()] += s["bias_values"][a:b].double()
        if masks[r] >= 0:
            bits = s["allowed"][masks[r]]
            bits = torch.stack([(bits >> i) & 1 for i in range(32)], 1).flatten()[:case["vocab"]]
            l[r, bits == 0] = float("-inf")
    return {"logits": l}


def exact(case, seed):
    made = {"attention": _exact_attention, "adapters": _exact_adapters, "logits": _exact_logits}[case["op"]]
    return made(case, prepare(case, seed))
