"""norm_rope / norm_rope_append against their definition in 64 bits.

The bound of an output, u = 2^-24: a head's scale is rounded once (its square sum is
taken in 64 bits), x scale w twice, the cosine and sine once each, then a cos - b sin
with three roundings, and the attention factor is part of the cosine: 7 u of |a| + |b|
after the norm.  Angles have 2^-51 of themselves from two products in 64 bits, the
cosine's and sine's sums 3e-9.  Dimensions that do not turn have 3 u; what is only
copied is equal.
"""
import math

import numpy as np
import pytest
import torch

import torchburn_amd as tb

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def reference(x, w, pos, f, eps, interleaved, factor):
    """(out, bound) in float64: x [n, heads, D], f [r / 2]."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    bound = 3 * U * np.abs(x)
    h = len(f)
    a, b = (x[..., 0:2 * h:2], x[..., 1:2 * h:2]) if interleaved else (x[..., :h], x[..., h:2 * h])
    t = pos.astype(np.float64)[:, None] * f
    c, s = (factor * np.cos(t))[:, None], (factor * np.sin(t))[:, None]
    out = x.copy()
    size = (np.abs(a) + np.abs(b)) * abs(factor) * (7 * U + 3e-9 + 2.0 ** -51 * np.abs(t)[:, None])
    if interleaved:
        out[..., 0:2 * h:2], out[..., 1:2 * h:2] = a * c - b * s, b * c + a * s
        bound[..., 0:2 * h:2] = bound[..., 1:2 * h:2] = size
    else:
        out[..., :h], out[..., h:2 * h] = a * c - b * s, b * c + a * s
        bound[..., :h] = bound[..., h:2 * h] = size
    return out, bound


def check(got, want, bound):
    got = got.cpu().numpy().astype(np.float64)
    assert got.shape == want.shape
    err = np.abs(got - want)
    worst = float((err / np.maximum(bound, 1e-300)).max()) if err.size else 0.0
    print(f"worst error {worst:.3g} of the bound", flush=True)
    assert (err <= bound + 1e-37).all(), worst


CASES = [
    # n, hq, hkv, D, r, interleaved, norm, start
    (1, 1, 1, 2, 2, False, True, 0),
    (1, 14, 2, 64, 64, False, True, 1),
    (3, 14, 2, 64, 64, False, False, 1000000),
    (5, 32, 8, 128, 128, False, True, 99999),
    (5, 32, 8, 128, 64, True, True, 7),
    (33, 7, 1, 96, 24, False, True, 5),
    (33, 7, 1, 96, 24, True, False, 5),
    (2, 5, 5, 72, 18, False, True, 123),      # pairs of no multiple of four
    (2, 5, 5, 72, 36, True, True, 123),
    (2, 3, 1, 80, 80, False, True, 3),
    (4, 4, 2, 256, 256, False, True, 12345),
    (4, 4, 2, 512, 130, True, True, 12345),   # four units a lane
    (2, 4, 2, 512, 512, False, True, 12345),
    (2, 4, 2, 34, 30, False, True, 9),
    (9, 6, 2, 160, 0, False, True, 9),        # nothing turns
    (700, 28, 4, 128, 128, False, True, 0),   # several heads a group
    (1777, 8, 8, 96, 48, True, True, 40),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_norm_rope(cuda, case):
    n, hq, hkv, d, r, inter, norm, start = case
    print(f"case norm_rope {case}", flush=True)
    g = np.random.default_rng(n + d + r)
    qkv = g.standard_normal((n, (hq + 2 * hkv) * d)).astype(np.float32) * 3
    pos = start + g.integers(0, 50, n)
    f, _ = tb.rope_frequencies(r, 10000.0, device="cpu")
    f = f.numpy()
    qw, kw = (g.standard_normal(d).astype(np.float32) if norm else None for _ in range(2))
    T = lambda a: None if a is None else torch.from_numpy(a).to(cuda)
    x = T(qkv)
    q, k, v = (t.view(n, -1, d) for t in x.split((hq * d, hkv * d, hkv * d), -1))
    how = dict(q_weight=T(qw), k_weight=T(kw), eps=1e-5, interleaved=inter, attention_factor=1.25)
    a, b = tb.norm_rope(q, k, T(pos), T(f), **how)
    want = [reference(t.cpu().numpy(), w, pos, f, 1e-5, inter, 1.25) for t, w in ((q, qw), (k, kw))]
    check(a, *want[0])
    check(b, *want[1])
    # a step: the same rows into caches of strides of their own, the rest as it was
    rows = 5
    base = torch.full((2, hkv, n, rows, d), float("nan"), device=cuda)
    kc, vc = (c.transpose(0, 1) for c in base)       # [n, hkv, rows, d], not contiguous
    at = g.integers(0, rows, n)
    at[n // 2] = rows      # outside: not written
    if n > 2:
        at[1] = -1
    o = tb.norm_rope_append(q, k, v, T(pos), T(f), kc, vc, T(at), **how)
    assert torch.equal(o, a)
    for i in range(n):
        if 0 <= at[i] < rows:
            assert torch.equal(kc[i, :, at[i]], b[i]) and torch.equal(vc[i, :, at[i]], v[i])
    wrote = torch.zeros((n, rows), dtype=torch.bool, device=cuda)
    ok = (at >= 0) & (at < rows)
    wrote[np.flatnonzero(ok), at[ok]] = True
    for c in (kc, vc):
        assert torch.equal(~torch.isnan(c).any(-1).any(1), wrote)
    # and one position for all
    kc2, vc2 = torch.zeros_like(kc), torch.zeros_like(vc)
    tb.norm_rope_append(q, k, v, T(pos), T(f), kc2, vc2, 3, **how)
    assert torch.equal(kc2[:, :, 3], b) and torch.equal(vc2[:, :, 3], v)
    assert int((kc2[:, :, [0, 1, 2, 4]] != 0).sum()) == 0


def test_forms_of_inputs(cuda):
    """Host tensors, other types, groups, one token, misaligned and unpacked heads."""
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn((3, 4, 6, 64), generator=g), torch.randn((3, 4, 2, 64), generator=g)
    pos = torch.randint(0, 1000, (3, 4), generator=g)
    f, _ = tb.rope_frequencies(64, 1e6, device="cpu")
    a, b = tb.norm_rope(q, k, pos, f)
    assert a.device.type == "cpu" and a.shape == q.shape and b.shape == k.shape
    f = f.to(cuda)
    c, d = tb.norm_rope(q.to(cuda), k.to(cuda), pos.to(cuda), f)
    assert torch.equal(c.cpu(), a) and torch.equal(d.cpu(), b)
    # int32 positions, float64 heads
    e, _ = tb.norm_rope(q.to(cuda).double(), k.to(cuda).double(), pos.to(cuda).int(), f)
    assert torch.equal(e, c)
    # unpacked: heads last but one of a wider buffer, starting inside a 16-byte unit
    wide = torch.zeros((3, 4, 7, 67), device=cuda)
    wide[..., 1:, 1:65] = q.to(cuda)
    e, _ = tb.norm_rope(wide[..., 1:, 1:65], k.to(cuda), pos.to(cuda), f)
    assert (e - c).abs().max() <= 4 * U * c.abs().max()
    # groups that are not a constant stride apart
    turned = q.to(cuda).transpose(0, 1).contiguous().transpose(0, 1)
    e, _ = tb.norm_rope(turned, k.to(cuda), pos.to(cuda), f)
    assert torch.equal(e, c)
    one, _ = tb.norm_rope(q[0, 0].to(cuda), k[0, 0].to(cuda), pos[0, 0].to(cuda), f)
    assert torch.equal(one, c[0, 0])
    none, _ = tb.norm_rope(q[:0].to(cuda), k[:0].to(cuda), pos[:0].to(cuda), f)
    assert none.shape == (0, 4, 6, 64)


def test_ranges(cuda):
    """Heads of the largest and smallest numbers, zeros, and NaN in one head."""
    f, _ = tb.rope_frequencies(64, device=cuda)
    q = torch.randn((1, 5, 64), device=cuda)
    q[0, 0] *= 1e30
    q[0, 1] *= 1e-30
    q[0, 2] = 0.0
    q[0, 3, 5] = float("nan")
    w = torch.ones(64, device=cuda)
    pos = torch.tensor([77], device=cuda)
    a, b = tb.norm_rope(q, q[:, :2], pos, f, w, w, eps=1e-6)
    assert torch.equal(b, a[:, :2])
    want, bound = reference(q.cpu().numpy(), w.cpu().numpy(), np.array([77]), f.cpu().numpy(), 1e-6,
                            False, 1.0)
    keep = [0, 1, 2, 4]
    check(a[:, keep], want[:, keep], bound[:, keep])
    assert torch.isnan(a[0, 3]).all()


def test_converted_caches(cuda):
    """Caches elsewhere or of another type are converted and written back."""
    f, _ = tb.rope_frequencies(32, device=cuda)
    q, k, v = (torch.randn((3, 2, 32), device=cuda) for _ in range(3))
    pos = torch.tensor([4, 5, 6], device=cuda)
    kc, vc = (torch.zeros((3, 2, 4, 32), device=cuda) for _ in range(2))
    a = tb.norm_rope_append(q, k, v, pos, f, kc, vc, 2)
    hk, hv = torch.zeros((3, 2, 4, 32)), torch.zeros((3, 2, 4, 32), dtype=torch.float16, device=cuda)
    assert torch.equal(tb.norm_rope_append(q, k, v, pos, f, hk, hv, 2), a)
    assert torch.equal(hk, kc.cpu()) and torch.equal(hv, vc.half())


def test_captured(cuda):
    """Captured and replayed, with other inputs between the replays."""
    f, _ = tb.rope_frequencies(64, device=cuda)
    q, k, v = (torch.randn((2, 4, 64), device=cuda) for _ in range(3))
    pos, at = torch.tensor([9, 3], device=cuda), torch.tensor([1, 0], device=cuda, dtype=torch.int32)
    kc, vc = (torch.zeros((2, 4, 8, 64), device=cuda) for _ in range(2))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        tb.norm_rope_append(q, k, v, pos, f, kc, vc, at)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tb.norm_rope_append(q, k, v, pos, f, kc, vc, at)
    for step in range(3):
        q.normal_()
        k.normal_()
        pos += 1
        at += 1
        graph.replay()
        a, b = tb.norm_rope(q, k, pos, f)
        torch.cuda.synchronize()
        assert torch.equal(out, a)
        for i in range(2):
            assert torch.equal(kc[i, :, int(at[i])], b[i])


def test_frequencies_turn_as_documented(cuda):
    for kw in (dict(), dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=8.0),
               dict(scaling="bands", factor=8.0, original_max=8192),
               dict(scaling="yarn", factor=16.0, original_max=4096)):
        f, c = tb.rope_frequencies(128, 500000.0, **kw)
        assert f.dtype is torch.float64 and f.is_cuda and f.shape == (64,)
        q = torch.randn((2, 3, 128), device=cuda)
        pos = np.array([0, 131071])
        a, _ = tb.norm_rope(q, q, torch.from_numpy(pos).to(cuda), f, attention_factor=c)
        check(a, *reference(q.cpu().numpy(), None, pos, f.cpu().numpy(), 0.0, False, c))
    assert math.isclose(c, 0.1 * math.log(16.0) + 1.0)


def test_converted_caches_keep_their_other_rows(cuda):
    """Of a cache in 64 bits only the row that is written is rounded; no cache is both."""
    f, _ = tb.rope_frequencies(32, device=cuda)
    q, k, v = (torch.randn((3, 2, 32), device=cuda) for _ in range(3))
    pos = torch.tensor([4, 5, 6], device=cuda)
    kc, vc = (torch.randn((3, 2, 4, 32), device=cuda, dtype=torch.float64) for _ in range(2))
    was = kc.clone(), vc.clone()
    tb.norm_rope_append(q, k, v, pos, f, kc, vc, 2)
    for c, w, row in zip((kc, vc), was, (tb.norm_rope(q, k, pos, f)[1], v)):
        assert torch.equal(c[:, :, 2], row.double())
        c[:, :, 2] = w[:, :, 2]
        assert torch.equal(c, w)
    for c in (kc, kc.half(), kc.float(), kc.float().cpu()):
        with pytest.raises(tb.UnsupportedOpError):
            tb.norm_rope_append(q, k, v, pos, f, c, c, 2)


def test_no_heads(cuda):
    """A batch of two dimensions whose keys have no heads."""
    f, _ = tb.rope_frequencies(32, device=cuda)
    q, k = torch.randn((2, 3, 4, 32), device=cuda), torch.randn((2, 3, 0, 32), device=cuda)
    pos = torch.arange(6, device=cuda).view(2, 3)
    a, b = tb.norm_rope(q, k, pos, f)
    assert torch.equal(a, tb.norm_rope(q, q, pos, f)[0]) and b.shape == k.shape


def test_positions_far_apart(cuda):
    """Element offsets past 32 bits, between a cache's positions and between its sequences."""
    f, _ = tb.rope_frequencies(32, device=cuda)
    q, k, v = (torch.randn((2, 3, 32), device=cuda) for _ in range(3))
    pos = torch.tensor([4, 5], device=cuda)
    want = tb.norm_rope(q, k, pos, f)[1]
    far = torch.empty((1 << 32) + (1 << 20), device=cuda)
    for strides in ((4096, 32, 1 << 31, 1), (1 << 32, 32, 4096, 1)):
        kc, vc = (far[off:].as_strided((2, 3, 3 if strides[0] == 4096 else 2, 32), strides)
                  for off in (0, 1 << 16))
        at = kc.shape[2] - 1
        kc.zero_(), vc.zero_()
        tb.norm_rope_append(q, k, v, pos, f, kc, vc, at)
        assert torch.equal(kc[:, :, at], want) and torch.equal(vc[:, :, at], v)
        assert not kc[:, :, :at].any() and not vc[:, :, :at].any()


@pytest.mark.parametrize("d", [64, 34])
def test_norms_at_the_ends_of_f32(cuda, d):
    """Heads whose scale is past f32's largest number or below its smallest normal one: the
    largest finite numbers, subnormal ones, and a single element that is not 0, without eps."""
    g = np.random.default_rng(d)
    f, _ = tb.rope_frequencies(16, device=cuda)
    x = g.uniform(0.5, 1.0, (1, 6, d)) * g.choice((-1, 1), (1, 6, d))
    x *= np.array([3.4e38, 1.2e38, 1e-38, 1e-40, 1e-43, 1.0])[:, None]
    x = x.astype(np.float32)
    x[0, 5] = 0
    x[0, 5, 3] = 2.0 ** -149
    w = g.standard_normal(d).astype(np.float32)
    T = lambda a: torch.from_numpy(a).to(cuda)
    for inter in (False, True):
        a, b = tb.norm_rope(T(x), T(x[:, 1:]), torch.tensor([77], device=cuda), f, T(w), T(w),
                            eps=0.0, interleaved=inter)
        assert torch.equal(b, a[:, 1:])
        check(a, *reference(x, w, np.array([77]), f.cpu().numpy(), 0.0, inter, 1.0))
