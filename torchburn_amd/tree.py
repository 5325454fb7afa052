"""Speculative decoding over a drafted tree, the device side.

A drafter proposes a tree of tokens; one forward verifies all of its nodes over
the KV cache, and the path that the model agrees with is kept.  The reference
verifies chains only (src/llm/decoder.rs:565-727).

A tree's nodes are in topological order: ``parents[i]`` is -1 (a root: a child of
the prefix's last token) or the index of an earlier node; anything else marks
node i as padding, and its descendants with it.  Node i's K / V row is in the
caches at position kv_len + i.  Batches hold trees of one node count, padded.
Acceptance starts at node 0, usually the last token chosen: other roots are
verified, but no path leads to them.

Caches are used where they are when they are f32 on q's (parents') device with
16-byte rows, contiguous or not.  Any others are converted whole, max_seq rows of
them, at every call (and written back by tree_accept): keep them in that form.
"""
from __future__ import annotations

import ctypes as C
from operator import attrgetter

from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib
from ._lib import UnsupportedOpError
from .quantization import _int32_on_gpu, _on_gpu, _ptr, _stream, _target, _write_back


_dtype = attrgetter("dtype")
_ALIGNED = bytes(range(0, 256, 16))   # the low bytes of 16-byte aligned addresses


def _bad(op: str, msg: str) -> UnsupportedOpError:
    return UnsupportedOpError(f"{_lib.UNSUPPORTED_MARKER} {op}: {msg}")


def _trees(op: str, t: torch.Tensor, dtype, dev) -> torch.Tensor:
    """Per-node values (n,) or (batch, n) as a device tensor."""
    if t.ndim not in (1, 2):
        raise _bad(op, f"trees must be (n,) or (batch, n), got {list(t.shape)}")
    return _int32_on_gpu(t, dev) if dtype is torch.int32 else _on_gpu(t, dtype, dev)


def _cache(op: str, name: str, c: torch.Tensor, batched: bool, dev: torch.device) -> torch.Tensor:
    """A cache as a [batch, heads, positions, head_dim] f32 device tensor with 16-byte rows:
    the caller's own memory when it already is one (any strides), else a copy."""
    if c.ndim != (4 if batched else 3):
        want = "[batch, num_kv_heads, max_seq, head_dim]" if batched else \
            "[num_kv_heads, max_seq, head_dim]"
        raise _bad(op, f"{name} must be {want}, got {list(c.shape)}")
    c = c.detach()
    ok = c.device == dev and c.dtype is torch.float32 and c.data_ptr() % 16 == 0 and \
        (c.stride(-1) == 1 or c.shape[-1] == 1) and all(s % 4 == 0 for s in c.stride()[:-1])
    if not ok:
        c = c.to(device=dev, dtype=torch.float32, memory_format=torch.contiguous_format,
                 copy=True).contiguous()
    return c if batched else c.unsqueeze(0)


def _kv_len(op: str, kv_len, batch: int, dev) -> Tuple[Optional[torch.Tensor], int]:
    if not isinstance(kv_len, torch.Tensor):
        return None, _lib.int64(kv_len)
    if kv_len.numel() != batch:
        raise _bad(op, f"kv_len must have {batch} elements, got {list(kv_len.shape)}")
    return _int32_on_gpu(kv_len.reshape(-1), dev), 0


def tree_masks(parents: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(mask int32 (.., n, ceil(n / 32)), depth int32 (.., n)) of trees given by their
    parents (n,) or (batch, n): bit j % 32 of word j // 32 of mask row i is set when node
    j is node i or an ancestor of it; node i's token has position kv_len + depth[i].  A
    padding node has no bits and depth 0."""
    dev = _target(parents)
    p = _trees("tree_masks", parents, torch.int32, dev)
    n = int(p.shape[-1])
    mask = torch.empty((*p.shape, (n + 31) // 32), dtype=torch.int32, device=dev)
    depth = torch.empty(p.shape, dtype=torch.int32, device=dev)
    _lib.call_on(dev, "tb_tree_masks", _ptr(p), _ptr(mask), _ptr(depth),
                 p.shape[0] if p.ndim == 2 else 1, n, _stream(dev))
    return mask.to(parents.device), depth.to(parents.device)


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   mask: torch.Tensor, kv_len: Union[int, torch.Tensor],
                   scale: Optional[float] = None) -> torch.Tensor:
    """GQA attention of a tree's nodes over the prefix and their own ancestors.

    ``q`` (n, num_heads, head_dim), ``k_cache`` / ``v_cache`` (num_kv_heads, max_seq,
    head_dim) already holding the nodes' rows at kv_len + i; all with a leading batch
    dimension for several sequences.  ``mask`` (n, ceil(n / 32)) of tree_masks(), one for
    all sequences or one each: node i sees the positions below ``kv_len`` and kv_len + j
    for every bit j of its row, and a row without bits gives zeros.  Positions that a row
    does not see take no part, whatever the caches hold there.  ``kv_len`` is a number
    (ValueError when kv_len + n exceeds max_seq) or a tensor with one per sequence (clamped
    on the device); the two may differ in their last bits, since the work is split by the
    length known at the call.  ``scale`` defaults to head_dim ** -0.5.  f32, in q's shape.
    Does not wait for the device."""
    op = "tree_attention"
    if q.ndim not in (3, 4):
        raise _bad(op, f"q must be [n, num_heads, head_dim] or [batch, n, num_heads, head_dim], "
                       f"got {list(q.shape)}")
    dev, batched = _target(q), q.ndim == 4
    n, heads, hd = (int(s) for s in q.shape[-3:])
    batch = int(q.shape[0]) if batched else 1
    x = _on_gpu(q.detach(), torch.float32, dev)
    if x.data_ptr() % 16:      # a view that starts inside a 16-byte unit
        x = x.clone()
    kc = _cache(op, "k_cache", k_cache, batched, dev)
    vc = _cache(op, "v_cache", v_cache, batched, dev)
    if kc.shape != vc.shape or kc.shape[0] != batch or kc.shape[3] != hd:
        raise _bad(op, f"caches {list(k_cache.shape)} / {list(v_cache.shape)} do not fit q "
                       f"{list(q.shape)}")
    words = (n + 31) // 32
    if mask.dtype != torch.int32 or tuple(mask.shape) not in ((n, words), (batch, n, words)):
        raise _bad(op, f"mask must be int32 [{n}, {words}] or [{batch}, {n}, {words}], got "
                       f"{mask.dtype} {list(mask.shape)}")
    mk = _on_gpu(mask, torch.int32, dev)
    lens, ln = _kv_len(op, kv_len, batch, dev)
    out = torch.empty(x.shape, dtype=torch.float32, device=dev)
    ks, vs = kc.stride(), vc.stride()
    # scratch of this call's own, so that graphs captured on one stream share none
    size = _lib.lib().tb_tree_attention_scratch(batch, n, heads, kc.shape[1], hd,
                                                kc.shape[2] if lens is not None else ln + n)
    scratch = torch.empty(size, dtype=torch.uint8, device=dev) if size > 0 else None
    _lib.call_on(dev, "tb_tree_attention", _ptr(x), _ptr(kc), _ptr(vc), _ptr(mk), _ptr(lens),
                 _ptr(out), batch, n, heads, kc.shape[1], hd, kc.shape[2], ln, ks[0], ks[1], ks[2],
                 vs[0], vs[1], vs[2], n * words if mk.ndim == 3 else 0,
                 hd ** -0.5 if scale is None else float(scale), _ptr(scratch), size, _stream(dev))
    return out if q.is_cuda else out.to(q.device)


def tree_accept(parents: torch.Tensor, draft_tokens: torch.Tensor, next_tokens: torch.Tensor,
                kv_len: Union[int, torch.Tensor] = 0,
                k_caches: Optional[Sequence[torch.Tensor]] = None,
                v_caches: Optional[Sequence[torch.Tensor]] = None
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The path of each tree that the model agrees with, kept in the caches.

    From node 0 (a root) the path goes to the lowest child whose ``draft_tokens`` entry is
    the node's ``next_tokens`` entry, the token that the model chose there (a negative one
    matches none).  Returns (path int32 (.., n) padded with -1, n_path int32 (..), token
    int64 (..): the next token of the path's last node; -1 without a path).

    ``k_caches`` / ``v_caches``: every layer's cache, as tree_attention takes them (all of
    one shape and one layout, none sharing memory with another), as lists or stacked in one
    tensor; row kv_len + path[j] moves to kv_len + j in each of them, in
    place, so the sequence's new length is kv_len + n_path.  Rows past the path keep what
    they held.  Does not wait for the device."""
    op = "tree_accept"
    dev = _target(parents)
    p = _trees(op, parents, torch.int32, dev)
    d = _trees(op, draft_tokens, torch.int64, dev)
    nx = _trees(op, next_tokens, torch.int64, dev)
    if d.shape != p.shape or nx.shape != p.shape:
        raise _bad(op, f"parents {list(p.shape)}, draft_tokens {list(d.shape)} and next_tokens "
                       f"{list(nx.shape)} differ")
    batched, n = p.ndim == 2, int(p.shape[-1])
    batch = int(p.shape[0]) if batched else 1
    if n == 0 and batch:
        raise _bad(op, "empty trees")
    lens, ln = _kv_len(op, kv_len, batch, dev)
    ks_in, vs_in = ([] if c is None else list(c) for c in (k_caches, v_caches))
    if len(ks_in) != len(vs_in):
        raise _bad(op, f"{len(ks_in)} k_caches against {len(vs_in)} v_caches")
    layers, given, caches = len(ks_in), ks_in + vs_in, ()
    kp = vp = None
    shape, ks, vs = (0, 1, 0, 32), (0, 0, 0, 0), (0, 0, 0, 0)
    if layers:
        # Device caches of one layout are used as they are (checked as whole lists: a cache
        # more costs 0.3 us, 1.5 through _cache).
        k0, v0, T = given[0], given[layers], torch.Tensor
        ptrs = (C.c_void_p * len(given))(*map(T.data_ptr, given))
        alike = set(map(T.get_device, given)) == {dev.index} and \
            set(map(_dtype, given)) == {torch.float32} and \
            list(map(T.size, given)) == [k0.shape] * len(given) and \
            list(map(T.stride, ks_in)) == [k0.stride()] * layers and \
            list(map(T.stride, vs_in)) == [v0.stride()] * layers and \
            not bytes(ptrs)[::8].translate(None, _ALIGNED) and \
            _cache(op, "cache", k0, batched, dev).data_ptr() == k0.data_ptr() and \
            _cache(op, "cache", v0, batched, dev).data_ptr() == v0.data_ptr()
        caches = given if alike else [_cache(op, "cache", x, batched, dev) for x in given]
        for part in () if alike else (slice(0, layers), slice(layers, None)):
            # a copy beside caches of other strides: those are copied too
            if any(c.data_ptr() != x.data_ptr() for c, x in zip(caches[part], given[part])):
                caches[part] = [c.contiguous() for c in caches[part]]
        if caches is not given and any(c.shape != caches[0].shape or
                                       c.stride() != caches[i // layers * layers].stride()
                                       for i, c in enumerate(caches)):
            raise _bad(op, "the layers' caches differ in shape or layout")
        k0, v0 = caches[0], caches[layers]
        if not batched and k0.ndim == 3:
            k0, v0 = k0.unsqueeze(0), v0.unsqueeze(0)
        shape, ks, vs = k0.shape, k0.stride(), v0.stride()
        if shape[0] != batch:
            raise _bad(op, f"caches {list(given[0].shape)} do not fit {batch} trees")
        if caches is not given:
            ptrs = (C.c_void_p * len(caches))(*map(T.data_ptr, caches))
        kp = C.addressof(ptrs)
        vp = kp + layers * C.sizeof(C.c_void_p)
    path = torch.empty(p.shape, dtype=torch.int32, device=dev)
    count = torch.empty(p.shape[:-1], dtype=torch.int32, device=dev)
    token = torch.empty(p.shape[:-1], dtype=torch.int64, device=dev)
    _lib.call_on(dev, "tb_tree_accept", _ptr(p), _ptr(d), _ptr(nx), _ptr(lens), ln, _ptr(path),
                 _ptr(count), _ptr(token), kp, vp, layers, batch, n, shape[1], shape[3], shape[2],
                 ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], _stream(dev))
    if caches is not given:
        for c, g in zip(given, caches):
            _write_back(c, g)
    to = parents.device
    return path.to(to), count.to(to), token.to(to)
