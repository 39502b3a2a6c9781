"""The serving operators' definitions in 64 bits, on any device, for the tests."""
import torch


def shared_attention(q, k_cache, v_cache, table, token_req, positions, scale):
    """(out, sum of weights x |values|, largest |scores| sum), token by token, through each token's own table; rows without keys: zeros."""
    tokens, heads, hd = q.shape
    page, kv_heads = k_cache.shape[1], k_cache.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    size, reach = torch.zeros_like(out), torch.zeros((tokens, heads, 1), dtype=torch.float64, device=q.device)
    for t in range(tokens):
        n = int(positions[t]) + 1
        if n <= 0:
            continue
        row = table[int(token_req[t])].long()
        j = torch.arange(n, device=q.device)
        k = k_cache[row[j // page], j % page].double().permute(1, 0, 2)           # [kv heads, keys, hd]
        v = v_cache[row[j // page], j % page].double().permute(1, 0, 2)
        x = q[t].double().view(kv_heads, heads // kv_heads, hd)
        w = torch.softmax(x @ k.transpose(1, 2) * scale, -1)
        out[t] = (w @ v).reshape(heads, hd)
        size[t] = (w @ v.abs()).reshape(heads, hd)
        reach[t] = (x.abs() @ k.abs().transpose(1, 2) * scale).amax(-1).reshape(heads, 1)
    return out, size, reach


def shared_attention_error(out, size, reach, hd, dtype):
    """A score is off by hd + 4 roundings of 2^-24 of its products' sizes (and the exponential by 2^-22 of it, for its argument's
    rounding), a weight by as much relative to itself; bfloat16 weights are rounded once more, and so is the output."""
    score = reach * ((hd + 4) * 2.0 ** -24 + 2.0 ** -22) + 2.0 ** -20
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    return size * (2.5 * score + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0)) + (out.abs() + size * 2.0 ** -7) * half


def adapters(y, x, a, b, index, scales=None, ranks=None):
    """(out, sum of the sizes of all products) in 64 bits."""
    out, size = y.double().clone(), torch.zeros(y.shape, dtype=torch.float64, device=y.device)
    for t, i in enumerate(index.tolist()):
        if not 0 <= i < a.shape[0]:
            continue
        r = a.shape[1] if ranks is None else max(0, min(int(ranks[i]), a.shape[1]))
        s = 1.0 if scales is None else float(scales[i])
        u, v, w = x[t].double(), a[i, :r].double(), b[i, :, :r].double()
        out[t] += s * (w @ (v @ u))
        size[t] = abs(s) * (w.abs() @ (v.abs() @ u.abs()))
    return out, size


def adapters_error(y, out, size, width, rank, dtype):
    """32-bit sums of width, then rank products; in bfloat16 the short sums go into the second product as two bfloat16 numbers,
    which leaves 2^-17 of them; the output is rounded once."""
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    inner = size * ((width + rank + 8) * 2.0 ** -24 + (2.0 ** -16 if dtype == torch.bfloat16 else 0.0))
    return inner + (y.double().abs() + size) * 2.0 ** -23 + (out.abs() + inner) * half


def rules(logits, history=None, lengths=None, prompt_lengths=None, slots=None, repetition=None, frequency=None, presence=None,
          biases=None, allowed=None, allowed_row=None):
    """(edited logits, sum of the sizes of what was added) in 64 bits; `biases`: per row a list of (id, value)."""
    rows, vocab = logits.shape
    l = logits.double().clone()
    size = torch.where(l.isfinite(), l.abs(), 0.0)
    for r in range(rows):
        slot = r if slots is None else int(slots[r])
        if history is not None and 0 <= slot < history.shape[0]:
            n = max(0, min(int(lengths[r]), history.shape[1]))
            p = 0 if prompt_lengths is None else max(0, min(int(prompt_lengths[r]), n))
            ids = [i for i in history[slot, :n].tolist()]
            rep = 1.0 if repetition is None else float(repetition[r])
            freq, pres = (0.0 if v is None else float(v[r]) for v in (frequency, presence))
            for i in {i for i in ids if 0 <= i < vocab}:
                v = float(l[r, i])
                v = v / rep if v > 0 else v * rep
                count = ids[p:].count(i)
                size[r, i] = max(float(size[r, i]), abs(v) if v == v and abs(v) != float("inf") else 0.0) + abs(freq) * count + abs(pres)
                l[r, i] = v - freq * count - (pres if count else 0.0)
        for i, v in (biases[r] if biases is not None else ()):
            if 0 <= i < vocab:
                l[r, i] += v
                size[r, i] += abs(v)
        m = r if allowed_row is None else int(allowed_row[r])
        if allowed is not None and 0 <= m < allowed.shape[0]:
            t = torch.arange(vocab, device=logits.device)
            l[r, ((allowed[m, t // 32] >> (t % 32)) & 1) == 0] = float("-inf")
    return l, size
