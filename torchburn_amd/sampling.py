"""Token sampling on the device (reference src/llm/decoder.rs:878-1020), and the
penalties, biases and masks on batches of logits before it.

``sample_logits`` applies the repetition penalty and draws one token from a
device logits vector without reading it back: greedy when the temperature is
not finite or <= 0 or top_k == 1, else top-k (ties to the lower index),
temperature softmax, nucleus cut at top_p and one draw.  The reference's draw
comes from an unseeded generator; here draw number ``counter`` of ``seed`` uses
u = ``sample_uniform(seed, counter)``, so a seed fixes the sequence.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence, Union

import torch

from . import _lib
from ._lib import UnsupportedOpError
from .quantization import _int32_on_gpu, _on_gpu, _ptr, _stream, _target


def sample_uniform(seed: int, counter: int) -> float:
    """The uniform in [0, 1) of draw ``counter`` under ``seed``."""
    return float(_lib.lib().tb_sample_uniform(int(seed) & (2 ** 64 - 1),
                                               int(counter) & (2 ** 64 - 1)))


def sample_logits(logits: torch.Tensor, temperature: float = 0.7, top_k: int = 40,
                  top_p: float = 1.0, repetition_penalty: float = 1.0,
                  recent_tokens: Optional[Sequence[int]] = None, seed: int = 0,
                  counter: int = 0, return_u: bool = False):
    """One token from ``logits`` (vocab,) on the GPU; the caller's tensor is not
    modified (the penalty works on a copy)."""
    dev = _target(logits)
    lg = _on_gpu(logits.reshape(-1), torch.float32, dev)
    rec = list(recent_tokens or [])
    rt = None
    if repetition_penalty > 1.0 and rec:
        lg = lg.clone() if lg.data_ptr() == logits.data_ptr() else lg
        rt = torch.tensor(rec, dtype=torch.int64, device=dev)
    tok, u = C.c_int64(), C.c_float()
    _lib.call("tb_sample_logits", _ptr(lg), lg.numel(), float(temperature), int(top_k),
              float(top_p), float(repetition_penalty), _ptr(rt), 0 if rt is None else rt.numel(),
              int(seed) & (2 ** 64 - 1), int(counter) & (2 ** 64 - 1), C.byref(tok), C.byref(u),
              _stream(dev))
    return (int(tok.value), float(u.value)) if return_u else int(tok.value)


def _bad(op: str, msg: str) -> UnsupportedOpError:
    return UnsupportedOpError(f"{_lib.UNSUPPORTED_MARKER} {op}: {msg}")


def _groups(op: str, name: str, t: Optional[torch.Tensor], rows: int, dtype, dev):
    """(tensor [groups, n], groups, n) of per-group lists: 1-D is one list for every row."""
    if t is None:
        return None, 1, 0
    if t.ndim not in (1, 2):
        raise _bad(op, f"{name} must be [n] or [groups, n], got {list(t.shape)}")
    g = t.shape[0] if t.ndim == 2 else 1
    if rows and (g == 0 or rows % g != 0):
        raise _bad(op, f"{name}: {g} lists do not divide {rows} rows")
    return _on_gpu(t, dtype, dev), g, int(t.shape[-1])


def _lengths(op: str, name: str, t, groups: int, dev):
    """(device int32 [groups] or None, host int) of lengths given as a tensor or a number."""
    if not isinstance(t, torch.Tensor):
        return None, _lib.int64(t)
    if t.numel() != groups:
        raise _bad(op, f"{name} must have {groups} elements, got {list(t.shape)}")
    return _int32_on_gpu(t.reshape(-1), dev), 0


def _penalty(op: str, name: str, t, rows: int, dev):
    """(device f32 [rows] or None, host float) of a penalty given as a tensor or a number."""
    if not isinstance(t, torch.Tensor):
        return None, float(t)
    if t.numel() != rows:
        raise _bad(op, f"{name} must have {rows} elements, got {list(t.shape)}")
    return _on_gpu(t.reshape(-1), torch.float32, dev), 1.0


def _process(op: str, want_tokens: bool, logits, history, history_len, prompt_len,
             repetition_penalty, presence_penalty, frequency_penalty, bias_ids, bias_values,
             allowed, draft_tokens, tree_mask, out):
    if logits.ndim < 1:
        raise _bad(op, "logits need at least one dimension")
    dev = _target(logits)
    vocab = int(logits.shape[-1])
    if vocab == 0:
        raise _bad(op, "empty vocabulary")
    x = _on_gpu(logits.detach(), torch.float32, dev)
    rows = x.numel() // vocab
    h, groups, hist = _groups(op, "history", history, rows, torch.int64, dev)
    hl, n_hist = (None, hist) if history_len is None or h is None else \
        _lengths(op, "history_len", history_len, groups, dev)
    if hl is None and not 0 <= n_hist <= hist:
        raise ValueError(f"{op}: history_len {n_hist} outside 0..{hist}")
    if hl is None and n_hist != hist:      # the first n_hist tokens of every list
        h, hist = h[..., :n_hist].contiguous(), n_hist
    pl, prompt = _lengths(op, "prompt_len", prompt_len, groups, dev)
    rr, rep = _penalty(op, "repetition_penalty", repetition_penalty, rows, dev)
    pr, pres = _penalty(op, "presence_penalty", presence_penalty, rows, dev)
    fr, freq = _penalty(op, "frequency_penalty", frequency_penalty, rows, dev)
    if (bias_ids is None) != (bias_values is None):
        raise _bad(op, "bias_ids and bias_values come together")
    bi, bgroups, n_bias = _groups(op, "bias_ids", bias_ids, rows, torch.int64, dev)
    bv, vgroups, n_val = _groups(op, "bias_values", bias_values, rows, torch.float32, dev)
    if (bgroups, n_bias) != (vgroups, n_val):
        raise _bad(op, f"bias_ids {list(bias_ids.shape)} and bias_values "
                       f"{list(bias_values.shape)} differ")
    am, words = None, (vocab + 31) // 32
    if allowed is not None:
        if allowed.dtype != torch.int32 or allowed.shape[-1:] != (words,) or \
                allowed.numel() not in (words, rows * words):
            raise _bad(op, f"allowed must be int32 [{words}] or [{rows}, {words}], got "
                           f"{allowed.dtype} {list(allowed.shape)}")
        am = _on_gpu(allowed, torch.int32, dev)
    dt, tm, nodes = None, None, 0
    if (draft_tokens is None) != (tree_mask is None):
        raise _bad(op, "draft_tokens and tree_mask come together")
    if draft_tokens is not None:
        nodes = int(draft_tokens.shape[-1]) if draft_tokens.ndim else 0
        if tree_mask.dtype != torch.int32 or not draft_tokens.ndim or \
                draft_tokens.numel() != rows or \
                tuple(tree_mask.shape) != (*draft_tokens.shape, (nodes + 31) // 32):
            raise _bad(op, f"draft_tokens [.., n] of {rows} nodes in all and tree_mask int32 "
                           f"[.., n, ceil(n / 32)] needed, got {list(draft_tokens.shape)} and "
                           f"{tree_mask.dtype} {list(tree_mask.shape)}")
        dt, tm = _on_gpu(draft_tokens, torch.int64, dev), _on_gpu(tree_mask, torch.int32, dev)
    y = tokens = scratch = None
    size = 0
    if want_tokens:
        tokens = torch.empty(rows, dtype=torch.int64, device=dev)
        size = _lib.lib().tb_process_logits_scratch(rows, vocab)
        scratch = torch.empty(size, dtype=torch.uint8, device=dev)
    elif out is None:
        y = torch.empty_like(x)
    else:
        if out.shape != logits.shape or out.dtype != torch.float32:
            raise _bad(op, f"out must be float32 {list(logits.shape)}, got {out.dtype} "
                           f"{list(out.shape)}")
        y = out if out.device == dev and out.is_contiguous() else torch.empty_like(x)
    _lib.call_on(dev, "tb_process_logits", _ptr(x), _ptr(y), _ptr(tokens), rows, vocab, _ptr(h),
                 _ptr(hl), _ptr(pl), groups, hist, prompt, rep, pres, freq, _ptr(rr), _ptr(pr),
                 _ptr(fr), _ptr(bi), _ptr(bv), bgroups, n_bias, _ptr(am),
                 0 if am is None or am.numel() == words else words, _ptr(dt), _ptr(tm), nodes,
                 _ptr(scratch), size, _stream(dev))
    if want_tokens:
        return tokens.reshape(logits.shape[:-1]).to(logits.device)
    if out is None:
        return y.to(logits.device)
    if y is not out:
        out.copy_(y)
    return out


_Rows = Union[float, torch.Tensor]


def process_logits(logits: torch.Tensor, history: Optional[torch.Tensor] = None,
                   history_len: Union[int, torch.Tensor, None] = None,
                   prompt_len: Union[int, torch.Tensor] = 0, repetition_penalty: _Rows = 1.0,
                   presence_penalty: _Rows = 0.0, frequency_penalty: _Rows = 0.0,
                   bias_ids: Optional[torch.Tensor] = None,
                   bias_values: Optional[torch.Tensor] = None,
                   allowed: Optional[torch.Tensor] = None,
                   draft_tokens: Optional[torch.Tensor] = None,
                   tree_mask: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Penalties for repeated tokens, biases and masks on logits (.., vocab).

    For token t of a row, with ``count`` its occurrences in the generated part of
    the row's history and on its tree path, and ``seen`` when it occurs anywhere:

        y = (x / repetition if x > 0 else x * repetition) if seen else x
        y = (y - frequency * count) - presence            if count > 0
        y = y + bias[t], and -inf where ``allowed`` has no bit for t

    ``history`` (n,) for every row or (groups, n), row r reading list
    r // (rows // groups); its first ``history_len`` tokens count (a number, or one
    per list), the first ``prompt_len`` of those as seen only.  Tokens outside the
    vocabulary (-1 as padding) are skipped.  A penalty is a number or one per row.
    ``bias_ids`` / ``bias_values`` (m,) or (groups, m); a token named twice gets the
    sum.  ``allowed`` int32 words (ceil(vocab / 32),) or one row each, bit t % 32 of
    word t // 32 set where token t may be taken; a row without bits becomes all
    -inf.  ``draft_tokens`` (.., n) and ``tree_mask`` (.., n, ceil(n / 32)) of
    tree_masks(): row r is node r % n of tree r // n, and the tokens of the node
    and its ancestors are part of its generated history, after ``history`` (which
    ends before node 0's token, or that counts twice).

    Returns y, a new tensor or ``out`` (which may be ``logits`` itself).  Does not
    wait for the device.  No reference counterpart beyond the repetition penalty
    (src/llm/decoder.rs:878-899).
    """
    return _process("process_logits", False, logits, history, history_len, prompt_len,
                    repetition_penalty, presence_penalty, frequency_penalty, bias_ids,
                    bias_values, allowed, draft_tokens, tree_mask, out)


def greedy_tokens(logits: torch.Tensor, history: Optional[torch.Tensor] = None,
                  history_len: Union[int, torch.Tensor, None] = None,
                  prompt_len: Union[int, torch.Tensor] = 0, repetition_penalty: _Rows = 1.0,
                  presence_penalty: _Rows = 0.0, frequency_penalty: _Rows = 0.0,
                  bias_ids: Optional[torch.Tensor] = None,
                  bias_values: Optional[torch.Tensor] = None,
                  allowed: Optional[torch.Tensor] = None,
                  draft_tokens: Optional[torch.Tensor] = None,
                  tree_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The best token of every row of process_logits(...), int64 of shape
    logits.shape[:-1], without writing the processed logits: the largest one, the
    lowest index on ties; NaN and -inf are never taken, and a row with nothing
    else gives -1.  Does not wait for the device."""
    return _process("greedy_tokens", True, logits, history, history_len, prompt_len,
                    repetition_penalty, presence_penalty, frequency_penalty, bias_ids,
                    bias_values, allowed, draft_tokens, tree_mask, None)
