"""Each request's own rules on its logits, in front of sampling: penalties, biases, a mask of allowed tokens."""
from __future__ import annotations

from ctypes import c_int, c_long, c_void_p

import torch

from ..ops import kernels as K


def _vector(t, dtype, n: int, name: str) -> None:
    if t is not None:
        K._need(t.dtype == dtype and t.shape == (n,) and t.is_contiguous(), f"{name} must be a contiguous {dtype} vector of {n}")


def _matrix(t, name: str) -> None:
    K._need(t.dim() == 2 and t.dtype == torch.int32 and (t.stride(1) == 1 or t.shape[1] <= 1) and max(t.shape) < 1 << 31,
            f"{name} must be a row-major int32 matrix")


def edit_logits(logits: torch.Tensor, *, history: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                prompt_lengths: torch.Tensor | None = None, slots: torch.Tensor | None = None,
                repetition: torch.Tensor | None = None, frequency: torch.Tensor | None = None,
                presence: torch.Tensor | None = None, bias_start: torch.Tensor | None = None,
                bias_ids: torch.Tensor | None = None, bias_values: torch.Tensor | None = None,
                allowed: torch.Tensor | None = None, allowed_row: torch.Tensor | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """The rows' rules applied to float32 `logits` [rows, vocab], in one kernel; a new tensor, or `out` (which may be `logits`).
    In this order, in 32 bits:

      a token in the row's history:  l / repetition where l > 0, else l * repetition
      l - frequency * count - presence * [count > 0], `count` being how often the token stands in the history behind the prompt
      + the row's biases of the token, one after the other as they are listed
      -inf where the row's mask does not allow the token, whatever l is

    `history`: int32 [slots, capacity], ids in any order of slots, the first `lengths[row]` of them (int32; at most the capacity)
    count, `prompt_lengths[row]` of which (int32; none: 0) are the prompt.  `slots` (int32) names each row's slot; without, row i's is
    i; a row whose slot is none of the history's (-1) has seen nothing.  Ids outside of the vocabulary count nowhere.
    `repetition`, `frequency`, `presence`: float32, one per row; without: 1, 0, 0.
    `bias_start`: int32 [rows + 1], row i's biases are `bias_ids[bias_start[i]:bias_start[i + 1]]` (int32) with `bias_values` (float32).
    `allowed`: int32 [masks, at least ceil(vocab / 32)], token t is bit t % 32 of word t // 32, set: allowed.  `allowed_row` (int32)
    names each row's mask; without, row i's is i; a row whose mask is none of these (-1) allows every token.  A mask that allows
    nothing leaves a row of -inf.  Row strides of `logits`, `history`, `allowed` and `out` are free."""
    if out is None and not K.PROFILER.enabled:
        got = (K._serving_binding or K._serving_calls("rules")).rules(logits, history, lengths, prompt_lengths, slots, repetition, frequency, presence,
                                                               bias_start, bias_ids, bias_values, allowed, allowed_row)
        if got is not None:
            return K._serving_done(got, "edit_logits", 1)
    K._cuda(logits, history, lengths, prompt_lengths, slots, repetition, frequency, presence, bias_start, bias_ids, bias_values,
            allowed, allowed_row, out)
    K._need(logits.dtype == torch.float32, "logits must be float32")
    ld_in = K._rows_of(logits, "logits")
    rows, V = logits.shape
    here = logits.device
    for t, name in ((history, "history"), (lengths, "lengths"), (prompt_lengths, "prompt_lengths"), (slots, "slots"),
                    (repetition, "repetition"), (frequency, "frequency"), (presence, "presence"), (bias_start, "bias_start"),
                    (bias_ids, "bias_ids"), (bias_values, "bias_values"), (allowed, "allowed"), (allowed_row, "allowed_row"), (out, "out")):
        if t is not None:
            K._need(t.device == here, f"{name} must be on the logits' device")
    for t, name in ((lengths, "lengths"), (prompt_lengths, "prompt_lengths"), (slots, "slots"), (allowed_row, "allowed_row")):
        _vector(t, torch.int32, rows, name)
    for t, name in ((repetition, "repetition"), (frequency, "frequency"), (presence, "presence")):
        _vector(t, torch.float32, rows, name)
    n_slots = capacity = ld_history = 0
    if history is not None:
        _matrix(history, "history")
        K._need(lengths is not None, "a history needs lengths")
        n_slots, capacity = history.shape
        ld_history = history.stride(0)
        K._need(slots is not None or n_slots >= rows, "without slots the history needs a row for every row of logits")
    else:
        K._need(lengths is None and prompt_lengths is None and slots is None and repetition is None and frequency is None
                and presence is None, "penalties need a history")
    n_biases = 0
    if bias_start is not None:
        K._need(bias_ids is not None and bias_values is not None, "biases need bias_start, bias_ids and bias_values")
        _vector(bias_start, torch.int32, rows + 1, "bias_start")
        n_biases = bias_ids.numel()
        _vector(bias_ids, torch.int32, n_biases, "bias_ids")
        _vector(bias_values, torch.float32, n_biases, "bias_values")
    else:
        K._need(bias_ids is None and bias_values is None, "biases need bias_start, bias_ids and bias_values")
    n_masks = ld_allowed = 0
    if allowed is not None:
        _matrix(allowed, "allowed")
        n_masks, ld_allowed = allowed.shape[0], allowed.stride(0)
        K._need(allowed.shape[1] * 32 >= V, f"a mask of {V} tokens needs {-(-V // 32)} words")
        K._need(allowed_row is not None or n_masks >= rows, "without allowed_row there must be a mask for every row")
    else:
        K._need(allowed_row is None, "allowed_row needs allowed")
    if out is None:
        out = torch.empty((rows, V), dtype=torch.float32, device=here)
    else:
        K._need(out.shape == logits.shape and out.dtype == torch.float32, "out must match the logits")
        K._rows_out(out, "out")
        K._same_place(out, logits, "out")
    ld_out = out.stride(0)
    if rows == 0 or V == 0:
        return out
    K._serving_calls("rules")                    # (where another operator's call has loaded the binding)
    f = K._fn("logit_rules", "lb_logit_rules",
              [c_void_p, c_long, c_void_p, c_long, c_int, c_int, c_void_p, c_long, c_int, c_int, c_void_p, c_void_p, c_void_p, c_void_p,
               c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_long, c_int, c_void_p, c_void_p])
    K._check(f(K._ptr(logits), ld_in, K._ptr(out), ld_out, rows, V, K._ptr(history), ld_history, capacity, n_slots, K._ptr(slots),
               K._ptr(lengths), K._ptr(prompt_lengths), K._ptr(repetition), K._ptr(frequency), K._ptr(presence), K._ptr(bias_start),
               K._ptr(bias_ids), K._ptr(bias_values), n_biases, K._ptr(allowed), ld_allowed, n_masks, K._ptr(allowed_row), K._stream()),
             "edit_logits", f"([{rows}, {V}])")
    return out
