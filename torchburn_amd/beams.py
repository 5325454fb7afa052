"""Decoding several sequences from one shared prompt: samples side by side, or the
beams of a beam search.

The sequences of a group share the cache of their prompt (the prefix) and have
a short cache each for what they added.  A step reads a long prefix for many of
them at once; a beam search then takes the best continuations of the group and moves the
short caches after them, while the prefix stays.  No reference counterpart: it
decodes one sequence over one cache (src/llm/decoder.rs:788-832).

A batch has ``groups`` as its leading dimension; without it, one group.  Caches are
used where they are when they are f32 on the device with 16-byte rows, contiguous or
not; prefix_attention's sequences have to be a constant stride apart over all groups.
Any others are converted whole at every call (and written back by beam_reorder):
keep them in that form.
"""
from __future__ import annotations

import ctypes as C
import math
from operator import attrgetter
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib
from ._lib import UnsupportedOpError
from .quantization import _int32_on_gpu, _on_gpu, _ptr, _stream, _target
from .rotary import _give_back, _ready

_dtype = attrgetter("dtype")
_ALIGNED = bytes(range(0, 256, 16))   # the low bytes of 16-byte aligned addresses


def _bad(op: str, msg: str) -> UnsupportedOpError:
    return UnsupportedOpError(f"{_lib.UNSUPPORTED_MARKER} {op}: {msg}")


# The checks below are most of a small call's time (0.1 us for each thing asked of a tensor):
# what the kernels can take as it is passes with as few of them as tell that.


def _usable(c: torch.Tensor, st, index) -> bool:
    """Whether the kernels can take a cache of strides st where it is."""
    odd = 0
    for s in st[:-1]:
        odd |= s
    return c.dtype is torch.float32 and c.get_device() == index and not odd & 3 and \
        (st[-1] == 1 or c.shape[-1] == 1) and not c.data_ptr() & 15


def _copied(c: torch.Tensor, dev: torch.device) -> torch.Tensor:
    return c.detach().to(device=dev, dtype=torch.float32, copy=True).contiguous()


def _cache(op: str, name: str, c: torch.Tensor, ndim: int, dev: torch.device):
    """A cache that the kernels can take, and its strides."""
    st = c.stride()
    if len(st) != ndim:
        raise _bad(op, f"{name} must have {ndim} dimensions, got {list(c.shape)}")
    if not _usable(c, st, dev.index):
        c = _copied(c, dev)
        st = c.stride()
    return c, st


def _sequences(op: str, name: str, c: torch.Tensor, batched: bool, dev: torch.device):
    """A cache of every sequence and its strides of sequence, KV head and position."""
    c, st = _cache(op, name, c, 5 if batched else 4, dev)
    if not batched:
        return c, st
    if c.shape[0] > 1 and st[0] != c.shape[1] * st[1]:      # groups apart
        c = _copied(c, dev)
        st = c.stride()
    return c, st[1:]


def _lengths(op: str, name: str, t, shape, dev) -> Tuple[Optional[torch.Tensor], int]:
    if not isinstance(t, torch.Tensor):
        return None, _lib.int64(t)
    # flat or with other dimensions of 1: still in this order
    if t.dtype.is_floating_point or (t.shape != shape and not (
            t.numel() == math.prod(shape) and (t.ndim == 1 or [n for n in t.shape if n != 1] ==
                                    [n for n in shape if n != 1]))):
        raise _bad(op, f"{name} must be a number or integers {list(shape)}, got {t.dtype} "
                       f"{list(t.shape)}")
    return (t if _ready(t, torch.int32, dev.index) else _int32_on_gpu(t, dev)), 0


def prefix_attention(q: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor,
                     prefix_len: Union[int, torch.Tensor], k_cache: Optional[torch.Tensor] = None,
                     v_cache: Optional[torch.Tensor] = None, kv_len: Union[int, torch.Tensor] = 0,
                     scale: Optional[float] = None) -> torch.Tensor:
    """GQA attention of one token of each sequence over the group's prefix and its own cache.

    ``q`` (rows, num_heads, head_dim); ``k_prefix`` / ``v_prefix`` (num_kv_heads, max_prefix,
    head_dim), whose first ``prefix_len`` positions every row sees; ``k_cache`` / ``v_cache``
    (rows, num_kv_heads, max_seq, head_dim), of which row i sees the first ``kv_len``, its new
    token's among them.  All with a leading ``groups`` dimension for several prompts.
    ``prefix_len`` is a number or integers () / (groups,), ``kv_len`` a number or integers
    (rows,) / (groups, rows), or flat in that order; numbers past the caches raise ValueError,
    tensors are clamped on the device.  Without k_cache and v_cache there is the prefix only.  Positions past the
    lengths take no part, whatever the caches hold there; a row that sees none gives zeros.
    ``scale`` defaults to head_dim ** -0.5; head_dim is a multiple of 32 up to 256.  f32, in
    q's shape; with more than 32 query rows of a KV head factors are kept to 2 ** -27 of
    themselves and 2 ** -134.  Infinities and NaN that a row sees count as in f32: a weight
    that is 0 there makes NaN of them.  A number and a tensor of the same length may differ in their last bits, since
    the work is split by what the call knows.  Does not wait for the device."""
    op = "prefix_attention"
    shape = q.shape
    if len(shape) == 4:
        groups, rows, heads, hd = shape
        batched = True
    elif len(shape) == 3:
        rows, heads, hd = shape
        groups, batched = 1, False
    else:
        raise _bad(op, f"q must be [rows, num_heads, head_dim] or [groups, rows, num_heads, "
                       f"head_dim], got {list(shape)}")
    dev = _target(q)
    x = q if _ready(q, torch.float32, dev.index) else _on_gpu(q.detach(), torch.float32, dev)
    if x.data_ptr() & 15:      # a view that starts inside a 16-byte unit
        x = x.detach().clone()
    kp, kps = _cache(op, "k_prefix", k_prefix, 4 if batched else 3, dev)
    vp, vps = _cache(op, "v_prefix", v_prefix, 4 if batched else 3, dev)
    *lead, kvh, max_prefix, width = kp.shape
    if vp.shape != kp.shape or width != hd or (batched and lead[0] != groups):
        raise _bad(op, f"prefixes {list(k_prefix.shape)} / {list(v_prefix.shape)} do not fit q "
                       f"{list(shape)}")
    if not batched:
        kps, vps = (0, *kps), (0, *vps)
    if (k_cache is None) != (v_cache is None):
        raise _bad(op, "k_cache and v_cache come together")
    max_own, kc, vc, ks, vs = 0, None, None, (0, 0, 0), (0, 0, 0)
    if k_cache is not None:
        kc, ks = _sequences(op, "k_cache", k_cache, batched, dev)
        vc, vs = _sequences(op, "v_cache", v_cache, batched, dev)
        own = kc.shape
        max_own = own[-2]
        want = (groups, rows, kvh, max_own, hd) if batched else (rows, kvh, max_own, hd)
        if own != want or vc.shape != want:
            raise _bad(op, f"caches {list(k_cache.shape)} / {list(v_cache.shape)} do not fit q "
                           f"{list(shape)} and {kvh} KV heads")
    pl, p = _lengths(op, "prefix_len", prefix_len, (groups,) if batched else (), dev)
    ol, o = _lengths(op, "kv_len", kv_len, (groups, rows) if batched else (rows,), dev)
    out = torch.empty_like(x, requires_grad=False)
    # scratch of this call's own, so that graphs captured on one stream share none
    size = _lib.lib().tb_prefix_attention_scratch(groups, rows, heads, kvh, hd,
                                                  p if pl is None else max_prefix,
                                                  o if ol is None else max_own)
    scratch = x.new_empty((size + 3) // 4) if size > 0 else None
    _lib.call_on(dev, "tb_prefix_attention", x.data_ptr(), kp.data_ptr(), vp.data_ptr(), _ptr(pl),
                 _ptr(kc), _ptr(vc), _ptr(ol), out.data_ptr(), groups, rows, heads, kvh, hd,
                 max_prefix, max_own, p, o, kps[0], kps[1], kps[2], vps[0], vps[1], vps[2], ks[0],
                 ks[1], ks[2], vs[0], vs[1], vs[2], hd ** -0.5 if scale is None else float(scale),
                 _ptr(scratch), size, _stream(dev))
    return out if q.is_cuda else out.to(q.device)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, k: Optional[int] = None,
                finished: Optional[torch.Tensor] = None, eos: Optional[int] = None
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``k`` best continuations of each group of beams, best first: (scores float32,
    tokens int64, beams int64), each (.., k).

    Token t after beam b has the value scores[b] + log_softmax(logits[b])[t], for ``logits``
    (.., beams, vocab) and ``scores`` (.., beams); ``k`` defaults to the number of beams (twice
    as many leave enough when some of them end).  Of equal values the lowest beam's and then
    the lowest token is taken; scores are rounded once.  The order is exact among a beam's
    tokens, and that of values in 64 bits among beams of the same logits; a beam's log-sum is
    good to 1e-10 (logits up to 10^5), so that tokens of other beams whose values are within
    2e-10 may change places.  A beam that is ``finished`` (.., beams) goes on with the token
    ``eos`` alone and keeps its score.  Logits of -inf (process_logits() masks) are never
    taken; a beam whose score is infinite or NaN, or that has a logit of NaN or +inf, has no
    continuation (scores of a group's first step: 0 and then -inf).  Where fewer than k are
    left, scores are -inf and tokens and beams -1, no index of anything.  Up to 64 beams, k up
    to 64, a vocabulary up to 2 ** 20.  Does not wait for the device."""
    op = "beam_select"
    *lead, beams, vocab = logits.shape if logits.ndim in (2, 3) else (0, 0, 0, -1)
    if vocab < 0 or scores.shape != (*lead, beams):
        raise _bad(op, f"logits must be [.., beams, vocab] and scores [.., beams], got "
                       f"{list(logits.shape)} and {list(scores.shape)}")
    dev = _target(logits)
    groups = lead[0] if lead else 1
    k = beams if k is None else _lib.int64(k)
    x = logits if _ready(logits, torch.float32, dev.index) else \
        _on_gpu(logits.detach(), torch.float32, dev)
    sc = scores if _ready(scores, torch.float32, dev.index) else \
        _on_gpu(scores.detach(), torch.float32, dev)
    done = None
    if finished is not None:
        if finished.shape != scores.shape or eos is None:
            raise _bad(op, f"finished {list(finished.shape)} needs the scores' shape "
                           f"{list(scores.shape)}, and eos")
        done = _on_gpu(finished if finished.dtype is torch.bool else finished != 0, torch.bool, dev)
    out = x.new_empty((*lead, max(k, 0)))
    tokens = torch.empty_like(out, dtype=torch.int64)
    parents = torch.empty_like(tokens)
    size = _lib.lib().tb_beam_select_scratch(groups, beams, vocab, k)
    scratch = x.new_empty(size // 4) if size > 0 else None
    _lib.call_on(dev, "tb_beam_select", x.data_ptr(), sc.data_ptr(), _ptr(done), out.data_ptr(),
                 tokens.data_ptr(), parents.data_ptr(), groups, beams, vocab, k,
                 0 if done is None else _lib.int64(eos), _ptr(scratch), size, _stream(dev))
    if logits.is_cuda:
        return out, tokens, parents
    to = logits.device
    return out.to(to), tokens.to(to), parents.to(to)


def beam_reorder(beams: torch.Tensor, k_caches: Sequence[torch.Tensor],
                 v_caches: Sequence[torch.Tensor], kv_len: Union[int, torch.Tensor]) -> None:
    """Beam j of each group takes over the cache rows of beam ``beams[.., j]``, in place.

    ``beams`` (.., n) of beam_select(); ``k_caches`` / ``v_caches``: every layer's cache (..,
    n, num_kv_heads, max_seq, head_dim), all of one shape and one layout, none sharing memory
    with another, as lists or stacked in one tensor.  A beam takes the first ``kv_len``
    positions of the one that it goes on from: a number (ValueError past max_seq) or integers
    (.., n), the lengths of the beams before the step (clamped on the device).  All beams are
    read before any is written; one may be taken over many times or never.  Rows past the
    length keep what they held, as does a beam whose entry is itself or no beam (-1).  Up to
    64 beams.  Does not wait for the device."""
    op = "beam_reorder"
    if beams.ndim not in (1, 2) or beams.dtype.is_floating_point:
        raise _bad(op, f"beams must be integers (n,) or (groups, n), got {beams.dtype} "
                       f"{list(beams.shape)}")
    dev, batched = _target(beams), beams.ndim == 2
    b = _on_gpu(beams, torch.int64, dev)
    n = beams.shape[-1]
    groups = beams.shape[0] if batched else 1
    lens, ln = _lengths(op, "kv_len", kv_len, beams.shape, dev)
    layers, ndim = len(k_caches), 5 if batched else 4
    if len(v_caches) != layers:
        raise _bad(op, f"{layers} k_caches against {len(v_caches)} v_caches")
    if not layers:
        return
    given, caches, stacked = (), (), True
    for c in (k_caches, v_caches):
        stacked = stacked and isinstance(c, torch.Tensor) and c.ndim == ndim + 1 and \
            _usable(c, c.stride(), dev.index)
    if stacked:      # a stack's caches differ by their addresses
        shape, ks, vs = k_caches.shape[1:], k_caches.stride(), v_caches.stride()
        alike = v_caches.shape == k_caches.shape
        ptrs = (C.c_void_p * (2 * layers))(
            *(c.data_ptr() + 4 * s[0] * i for c, s in ((k_caches, ks), (v_caches, vs))
              for i in range(layers)))
        ks, vs = ks[1:], vs[1:]
    if not stacked or not alike:
        # Device caches of one layout are used as they are, checked as whole lists.
        ks_in, vs_in = list(k_caches), list(v_caches)
        given = ks_in + vs_in
        k0, v0, T = given[0], given[layers], torch.Tensor
        shape, ks, vs = k0.shape, k0.stride(), v0.stride()
        ptrs = (C.c_void_p * len(given))(*map(T.data_ptr, given))
        alike = set(map(T.get_device, given)) == {dev.index} and \
            set(map(_dtype, given)) == {torch.float32} and \
            list(map(T.size, given)) == [shape] * len(given) and \
            list(map(T.stride, ks_in)) == [ks] * layers and \
            list(map(T.stride, vs_in)) == [vs] * layers and \
            not bytes(ptrs)[::8].translate(None, _ALIGNED) and _usable(k0, ks, dev.index) and \
            _usable(v0, vs, dev.index)
    if len(shape) != ndim or shape[-4] != n or (batched and shape[0] != groups):
        raise _bad(op, f"caches {list(shape)} do not fit beams {list(beams.shape)}")
    if not alike:
        if any(c.shape != shape for c in given):
            raise _bad(op, "the layers' caches differ in shape")
        if len(set(ptrs)) != len(given) and k0.numel():
            raise _bad(op, "a cache is given twice")
        caches = [_copied(c, dev) for c in given]
        ks, vs = caches[0].stride(), caches[layers].stride()
        ptrs = (C.c_void_p * len(given))(*map(T.data_ptr, caches))
    if not batched:
        ks, vs = (0, *ks), (0, *vs)
    kp = C.addressof(ptrs)
    _lib.call_on(dev, "tb_beam_reorder", _ptr(b), _ptr(lens), ln, kp,
                 kp + layers * C.sizeof(C.c_void_p), layers, groups, n, shape[-3], shape[-1],
                 shape[-2], ks[0], ks[1], ks[2], ks[3], vs[0], vs[1], vs[2], vs[3], _stream(dev))
    if not alike:
        for c, g in zip(given, caches):
            _give_back(c, g)
