"""Norms of the query and key heads and their rotary positions, in one pass.

The reference rotates whole heads by halves, unscaled and without head norms
(python/torchburn/llm/model.py:99-140, src/llm/decoder.rs:334-350), as
RustQwenDecoder does inside its QKV projection; this is the general operator,
for models whose steps a host puts together itself.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from . import _lib
from ._lib import UnsupportedOpError
from .quantization import _int32_on_gpu, _on_gpu, _ptr, _stream, _target, _write_back


def _bad(op: str, msg: str) -> UnsupportedOpError:
    return UnsupportedOpError(f"{_lib.UNSUPPORTED_MARKER} {op}: {msg}")


def rope_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: Optional[str] = None,
                     factor: float = 1.0, original_max: int = 0, low_freq_factor: float = 1.0,
                     high_freq_factor: float = 4.0, beta_fast: float = 32.0,
                     beta_slow: float = 1.0, device=None) -> Tuple[torch.Tensor, float]:
    """(inv_freq float64 (rotary_dim / 2,), attention_factor) of norm_rope(): the radians that
    pair i turns a position, theta ** (-2 i / rotary_dim), scaled for contexts ``factor`` times
    as long as the ``original_max`` positions that the model learned:

      None      not at all
      "linear"  every frequency by 1 / factor
      "ntk"     theta becomes theta * factor ** (rotary_dim / (rotary_dim - 2))
      "bands"   1 / factor where fewer than ``low_freq_factor`` turns fit original_max, not at
                all where more than ``high_freq_factor`` do, and a share between by the turns
      "yarn"    the same by the pair's number, between those that turn ``beta_fast`` and
                ``beta_slow`` times; attention_factor 0.1 ln(factor) + 1

    Worked out on the host; ``device`` defaults to the GPU where there is one."""
    op, r, s = "rope_frequencies", int(rotary_dim), float(factor)
    if r < 0 or r % 2:
        raise _bad(op, f"rotary_dim must be even, got {rotary_dim}")
    theta = float(theta)
    if not (theta > 0.0 and math.isfinite(theta)) or not (s > 0.0 and math.isfinite(s)):
        raise ValueError(f"{op}: theta and factor must be positive, got {theta} and {factor}")
    if scaling not in (None, "linear", "ntk", "bands", "yarn"):
        raise ValueError(f"{op}: unknown scaling {scaling!r}")
    if scaling in ("bands", "yarn") and original_max <= 0:
        raise ValueError(f"{op}: {scaling} needs original_max")
    if scaling == "ntk" and r > 2:
        theta *= s ** (r / (r - 2))
    pair = torch.arange(r // 2, dtype=torch.float64)
    f = theta ** (-2.0 * pair / r) if r else pair
    attention = 1.0
    if scaling == "linear":
        f = f / s
    elif scaling == "bands":
        if not high_freq_factor > low_freq_factor:
            raise ValueError(f"{op}: high_freq_factor must be above low_freq_factor")
        turns = original_max * f / (2 * math.pi)
        keep = ((turns - low_freq_factor) / (high_freq_factor - low_freq_factor)).clamp(0.0, 1.0)
        f = f * keep + f / s * (1.0 - keep)
    elif scaling == "yarn":
        if not (beta_fast > beta_slow > 0) or theta == 1.0:
            raise ValueError(f"{op}: yarn needs beta_fast > beta_slow > 0 and a theta but 1")

        def turning(times):      # the pair that turns so often in original_max positions
            return r * math.log(original_max / (times * 2 * math.pi)) / (2 * math.log(theta))
        low = max(math.floor(turning(beta_fast)), 0)
        high = min(math.ceil(turning(beta_slow)), r - 1)
        scaled = ((pair - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        f = f / s * scaled + f * (1.0 - scaled)
        attention = 0.1 * math.log(s) + 1.0 if s > 1.0 else 1.0
    if device is None:
        device = "cuda" if torch.cuda.is_available() else "cpu"
    return f.to(device), attention


def _ready(t: torch.Tensor, dtype: torch.dtype, index: int) -> bool:
    """Whether the kernels can read t where it is."""
    return t.dtype is dtype and t.get_device() == index and t.is_contiguous()


def _heads(op: str, name: str, t: torch.Tensor, lead, hd: int, dev):
    """(tensor, heads, token stride, head stride): the caller's memory where a token's heads
    are a constant number of elements apart and the tokens too, else a copy."""
    *first, heads, width = t.shape if t.ndim >= 2 else (0, 0, -1)
    if width != hd or first != lead:
        raise _bad(op, f"{name} must be [{', '.join(map(str, lead))}, heads, {hd}], got "
                       f"{list(t.shape)}")
    st = t.stride()
    if t.dtype is not torch.float32 or t.get_device() != dev.index or (st[-1] != 1 and hd > 1):
        t = _on_gpu(t.detach(), torch.float32, dev)
        st = t.stride()
    if len(st) == 3:
        return t, heads, st[0], st[1]
    if len(st) == 2:
        return t, heads, 0, st[0]
    flat = _flat(t.detach(), 2)
    return flat, heads, flat.stride(0), flat.stride(1)


def _flat(t: torch.Tensor, last: int) -> torch.Tensor:
    """t with one dimension before its last ones: a view, or a copy where there is none."""
    return t.flatten(0, -1 - last)


def _give_back(c: torch.Tensor, new: torch.Tensor) -> None:
    """A converted cache's rows to the caller's.  What did not change stays as it was there:
    a type that f32 does not hold is rounded only in rows that are written."""
    with torch.no_grad():
        if c.dtype is not torch.float32 and c.dtype.itemsize > 2:
            same = new.reshape(c.shape) == c.to(new.device, torch.float32)
            new = torch.where(same, c.to(new.device), new.reshape(c.shape).to(c.dtype))
        _write_back(c, new)


def _own_caches(op: str, name: str, c: torch.Tensor, lead, heads: int, hd: int, dev):
    """A cache [.., heads, positions, head_dim] as an f32 device tensor whose sequences are a
    constant number of elements apart, its positions and those strides: the caller's memory
    or a copy."""
    *first, kvh, rows, width = c.shape if c.ndim >= 3 else (0, 0, 0, -1)
    if width != hd or kvh != heads or first != lead:
        raise _bad(op, f"{name} must be [{', '.join(map(str, lead))}, {heads}, max_seq, {hd}], "
                       f"got {list(c.shape)}")
    st = c.stride()
    if c.dtype is not torch.float32 or c.get_device() != dev.index or (st[-1] != 1 and hd > 1):
        c = c.detach().to(device=dev, dtype=torch.float32, copy=True).contiguous()
        st = c.stride()
    if len(st) == 4:
        return c, rows, st
    if len(st) == 3:
        return c, rows, (0, *st)
    flat = _flat(c.detach(), 3)
    return flat, rows, flat.stride()


def _call(op, q, k, v, positions, inv_freq, q_weight, k_weight, eps, interleaved,
          attention_factor, k_cache, v_cache, at):
    if q.ndim < 2:
        raise _bad(op, f"q must be [.., num_heads, head_dim], got {list(q.shape)}")
    dev = _target(q)
    index = dev.index
    *lead, hq, hd = q.shape
    x, hq, q_st, q_sh = _heads(op, "q", q, lead, hd, dev)
    y, hkv, k_st, k_sh = _heads(op, "k", k, lead, hd, dev)
    if not isinstance(positions, torch.Tensor) or [*positions.shape] != lead or \
            positions.dtype.is_floating_point:
        raise _bad(op, f"positions must be integers {lead}, one a token")
    pairs = inv_freq.numel()
    if 2 * pairs > hd or inv_freq.ndim != 1:
        raise _bad(op, f"inv_freq must hold at most head_dim / 2 = {hd // 2} frequencies, got "
                       f"{list(inv_freq.shape)}")
    pos = positions if _ready(positions, torch.int64, index) else \
        _on_gpu(positions, torch.int64, dev)
    freq = inv_freq if _ready(inv_freq, torch.float64, index) else \
        _on_gpu(inv_freq, torch.float64, dev)
    weights = []
    for w in (q_weight, k_weight):
        if w is not None:
            if w.numel() != hd or w.ndim != 1:
                raise _bad(op, f"the heads' weights must be [{hd}], got {list(w.shape)}")
            if not _ready(w, torch.float32, index):
                w = _on_gpu(w, torch.float32, dev)
        weights.append(w)
    qw, kw = weights
    out = x.new_empty((*lead, hq, hd))
    z = kc = vc = lens = k_out = None
    v_st = v_sh = where = rows = 0
    ks = vs = (0, 0, 0)
    if v is None:
        k_out = x.new_empty((*lead, hkv, hd))
    else:
        z, v_heads, v_st, v_sh = _heads(op, "v", v, lead, hd, dev)
        if v_heads != hkv:
            raise _bad(op, f"k has {hkv} heads, v {v_heads}")
        kc, rows, ks = _own_caches(op, "k_cache", k_cache, lead, hkv, hd, dev)
        vc, v_rows, vs = _own_caches(op, "v_cache", v_cache, lead, hkv, hd, dev)
        if v_rows != rows:
            raise _bad(op, f"k_cache has {rows} positions, v_cache {v_rows}")
        if (kc is not k_cache or vc is not v_cache) and k_cache.numel() and \
                k_cache.data_ptr() == v_cache.data_ptr():
            raise _bad(op, "k_cache and v_cache share memory")
        if isinstance(at, torch.Tensor):
            if [*at.shape] != lead or at.dtype.is_floating_point:
                raise _bad(op, f"kv_len must be integers {lead}, got {at.dtype} {list(at.shape)}")
            lens = at if _ready(at, torch.int32, index) else _int32_on_gpu(at, dev)
        else:
            where = _lib.int64(at)
    _lib.call_on(dev, "tb_norm_rope", x.data_ptr(), y.data_ptr(), _ptr(z), pos.data_ptr(),
                 freq.data_ptr(), _ptr(qw), _ptr(kw), out.data_ptr(), _ptr(k_out), _ptr(kc),
                 _ptr(vc), _ptr(lens), pos.numel(), hq, hkv, hd, 2 * pairs, q_st, q_sh, k_st, k_sh,
                 v_st, v_sh, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], rows, where,
                 1 if interleaved else 0, float(attention_factor), float(eps), _stream(dev))
    if v is not None:
        if kc.data_ptr() != k_cache.data_ptr():
            _give_back(k_cache, kc)
        if vc.data_ptr() != v_cache.data_ptr():
            _give_back(v_cache, vc)
    if q.is_cuda:
        return out, k_out
    return out.to(q.device), None if k_out is None else k_out.to(q.device)


def norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
              q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
              eps: float = 1e-6, interleaved: bool = False, attention_factor: float = 1.0
              ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Head norms and rotary positions of ``q`` (.., num_heads, head_dim) and ``k`` (..,
    num_kv_heads, head_dim), a token at each of the leading places; new tensors (f32).

    With ``q_weight`` / ``k_weight`` (head_dim,) each head x becomes
    x / sqrt(mean(x ** 2) + eps) * weight.  Then the pairs i of the first
    2 * len(inv_freq) dimensions r, (i, i + r / 2) or ``interleaved`` (2 i, 2 i + 1), turn by
    ``positions`` (..) * inv_freq[i] and are multiplied by ``attention_factor``
    (rope_frequencies() gives both); other dimensions do not turn.  Angles are worked out
    in 64 bits.  q and k in f32 on the device with head_dim contiguous (as views of a fused
    projection's output) are read where they are.  Does not wait for the device."""
    return _call("norm_rope", q, k, None, positions, inv_freq, q_weight, k_weight, eps,
                 interleaved, attention_factor, None, None, 0)


def norm_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                     inv_freq: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                     kv_len: Union[int, torch.Tensor], q_weight: Optional[torch.Tensor] = None,
                     k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                     interleaved: bool = False, attention_factor: float = 1.0) -> torch.Tensor:
    """norm_rope() of one token of each of several sequences, whose key and value rows go to
    the sequences' caches: row ``kv_len`` (a number, or integers (..), one per sequence) of
    ``k_cache`` / ``v_cache`` (.., num_kv_heads, max_seq, head_dim) takes the turned key and
    ``v`` as it is.  Returns the turned queries.

    A number outside the caches raises ValueError; a sequence whose kv_len is outside has no
    row written; no two rows of the caches may share memory.  Caches in f32 on q's device with
    head_dim contiguous and sequences a constant stride apart are written in place; any others
    are converted whole at every call.  Does not wait for the device."""
    return _call("norm_rope_append", q, k, v, positions, inv_freq, q_weight, k_weight, eps,
                 interleaved, attention_factor, k_cache, v_cache, kv_len)[0]
