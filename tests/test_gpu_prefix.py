"""prefix_attention against its definition in 64 bits, and a run of the operators of a
step from a shared prompt together.

The bound, row by row, u = 2^-24.  A score is a sum of D products of f32 factors, or of
6 D products of their bf16 parts, whose dropped ones are 2^-25 of the factors' in all,
taken as a random walk with a factor of 4 to spare: ds = scale sum|q k| (2 u +
4 sqrt(6 D) u) + 8 u (|s| + 8), the last for the scaling, the reference's subtraction and
the exponential's argument.  A softmax weight is then off by a share of 2 ds + 8 u (both
the weight and the sum it is divided by), the weighted sum over T keys by 2 u +
4 sqrt(6 T) u more, so |error| <= sum_p w_p |v_p| (2 ds + 10 u + 4 sqrt(6 T) u).
"""
import numpy as np
import pytest
import torch

import torchburn_amd as tb
from torchburn_amd import _lib

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def reference(q, kp, vp, plen, k, v, olen, scale):
    """(out, bound) in float64 from numpy arrays: q [S, N, H, D], kp / vp [S, KVH, P, D], k / v
    [S, N, KVH, L, D] or None, plen [S], olen [S][N]."""
    S, N, H, D = q.shape
    KVH = kp.shape[1]
    G = H // KVH
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for s in range(S):
        p = min(max(plen[s], 0), kp.shape[2])
        for n in range(N):
            o = 0 if k is None else min(max(olen[s][n], 0), k.shape[3])
            if p + o == 0:
                continue
            for j in range(KVH):
                kk, vv = kp[s, j, :p].astype(np.float64), vp[s, j, :p].astype(np.float64)
                if o:
                    kk = np.concatenate((kk, k[s, n, j, :o].astype(np.float64)))
                    vv = np.concatenate((vv, v[s, n, j, :o].astype(np.float64)))
                x = q[s, n, j * G:(j + 1) * G].astype(np.float64)
                a = x @ kk.T * scale
                e = np.exp(a - a.max(-1, keepdims=True))
                w = e / e.sum(-1, keepdims=True)
                out[s, n, j * G:(j + 1) * G] = w @ vv
                # a position's own error counts with its weight
                ds = abs(scale) * (np.abs(x) @ np.abs(kk).T) * (2 * U + 4 * (6 * D) ** 0.5 * U) + \
                    8 * U * (np.abs(a) + 8)
                mean = (w * ds).sum(-1, keepdims=True)
                bound[s, n, j * G:(j + 1) * G] = (w * (ds + mean + 10 * U +
                                                       4 * (6 * (p + o)) ** 0.5 * U)) @ np.abs(vv)
    return out, bound


def inputs(seed, S, N, H, KVH, D, P, L, kscale=1.0):
    g = np.random.default_rng(seed)
    f = lambda *s: g.standard_normal(s).astype(np.float32)
    return (2 * f(S, N, H, D), kscale * f(S, KVH, P, D), f(S, KVH, P, D),
            kscale * f(S, N, KVH, L, D), f(S, N, KVH, L, D))


def check(got, want, bound):
    got = got.cpu().numpy().astype(np.float64)
    assert np.isfinite(got).all()
    err = np.abs(got - want)
    worst = float((err / np.maximum(bound, 1e-300))[bound > 0].max()) if (bound > 0).any() else 0.0
    print(f"worst error {worst:.3g} of the bound", flush=True)
    assert (err <= bound).all(), worst


CASES = [
    # S, N, H, KVH, D, prefix lengths, P, own lengths, L
    (1, 1, 1, 1, 32, [0], 1, [[0]], 1),                # sees nothing
    (1, 1, 1, 1, 32, [1], 1, [[0]], 1),
    (1, 2, 4, 2, 64, [0], 3, [[1, 0]], 1),             # no prefix
    (1, 4, 14, 2, 64, [200], 256, [[7, 3, 0, 1]], 8),
    (1, 8, 32, 8, 128, [1000], 1024, [[64, 60, 1, 0, 17, 33, 64, 5]], 64),
    (2, 5, 28, 4, 128, [300, 77], 320, [[9, 10, 11, 12, 13], [1, 2, 3, 4, 5]], 16),
    (3, 3, 8, 8, 96, [0, 15, 16], 40, [[0, 15, 16], [17, 31, 32], [33, 63, 64]], 70),
    (1, 1, 40, 1, 64, [500], 512, [[130]], 140),       # a group of 40 heads
    (1, 33, 4, 4, 64, [129], 140, None, 20),
    (1, 50, 7, 1, 160, [65], 80, None, 33),
    (1, 20, 16, 4, 256, [190], 200, None, 40),
    (1, 64, 32, 8, 128, [700], 704, None, 100),        # many rows
    (1, 128, 8, 2, 192, [333], 400, None, 10),
    (2, 70, 5, 1, 32, [90, 1500], 1500, None, 3),
    (1, 100, 64, 8, 64, [2049], 2060, None, 5),
    (7, 2, 6, 2, 224, [5, 100, 64, 1, 0, 63, 48], 128, None, 50),
    (1, 3, 4, 4, 128, [9001], 9001, [[2000, 1, 700]], 2001),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:5])) + f"-P{c[6]}-L{c[8]}")
def test_attention(cuda, case):
    S, N, H, KVH, D, plen, P, olen, L = case
    print(f"case prefix_attention {case}", flush=True)
    arrays = inputs(S + N + D + P, S, N, H, KVH, D, P, L)
    if olen is None:
        olen = np.random.default_rng(P).integers(0, L + 1, (S, N)).tolist()
    q, kp, vp, k, v = (torch.from_numpy(a).to(cuda) for a in arrays)
    for i in range(S):      # what no row sees
        kp[i, :, plen[i]:], vp[i, :, plen[i]:] = float("nan"), float("inf")
        for n in range(N):
            k[i, n, :, olen[i][n]:], v[i, n, :, olen[i][n]:] = float("inf"), float("nan")
    want, bound = reference(*arrays[:3], plen, *arrays[3:], olen, D ** -0.5)
    pl = torch.tensor(plen, device=cuda)
    ol = torch.tensor(olen, device=cuda, dtype=torch.int32)
    got = tb.prefix_attention(q, kp, vp, pl, k, v, ol)
    assert got.shape == q.shape
    check(got, want, bound)
    empty = np.array([[plen[i] + olen[i][n] == 0 for n in range(N)] for i in range(S)])
    assert (got.cpu().numpy()[empty] == 0).all()
    if S == 1:      # numbers, and without the groups' dimension
        check(tb.prefix_attention(q[0], kp[0], vp[0], plen[0], k[0], v[0], ol[0]), want[0], bound[0])
    # the prefix alone
    want, bound = reference(*arrays[:3], plen, None, None, None, D ** -0.5)
    check(tb.prefix_attention(q, kp, vp, pl), want, bound)
    # and the own caches alone, in a length for all
    want, bound = reference(*arrays[:3], [0] * S, *arrays[3:], [[L] * N] * S, 0.3)
    k, v = (torch.from_numpy(a).to(cuda) for a in arrays[3:])
    check(tb.prefix_attention(q, kp, vp, 0, k, v, L, scale=0.3), want, bound)


@pytest.mark.parametrize("rows", [4, 40])
def test_layouts(cuda, rows):
    """Positions before heads, spare rows, expanded prefixes, a misaligned q, other types,
    lengths outside of the caches, host tensors; each against the plain layout."""
    H, KVH, D, P, L = 8, 4, 64, 150, 20
    arrays = inputs(3, 2, rows, H, KVH, D, P, L)
    q, kp, vp, k, v = (torch.from_numpy(a).to(cuda) for a in arrays)
    kp, vp = kp[:1], vp[:1]
    pl = torch.tensor([140, 33], device=cuda)
    ol = torch.arange(2 * rows, device=cuda).reshape(2, rows) % (L + 1)
    both = [c.expand(2, -1, -1, -1) for c in (kp, vp)]      # one prompt under both groups
    want = tb.prefix_attention(q, *(c.contiguous() for c in both), pl, k, v, ol)
    assert torch.equal(tb.prefix_attention(q, *both, pl, k, v, ol), want)
    wide = [torch.full((2, P + 3, KVH, D + 4), float("nan"), device=cuda) for _ in range(2)]
    views = []
    for w, c in zip(wide, both):
        w[:, :P, :, :D] = c.transpose(1, 2)
        views.append(w[:, :P, :, :D].transpose(1, 2))
    own = [torch.full((2, rows, L, KVH, D), 0.0, device=cuda) for _ in range(2)]
    mine = []
    for w, c in zip(own, (k, v)):
        w.copy_(c.transpose(2, 3))
        mine.append(w.transpose(2, 3))
    assert torch.equal(tb.prefix_attention(q, *views, pl, *mine, ol), want)
    # groups that are not a constant stride apart
    apart = [torch.stack((c[0], c[0], c[1])) for c in (k, v)]
    assert torch.equal(tb.prefix_attention(q, *both, pl, *(c[::2] for c in apart), ol), want)
    off = torch.empty(q.numel() + 1, device=cuda)[1:].view(q.shape).copy_(q)
    assert torch.equal(tb.prefix_attention(off, *both, pl, k, v, ol), want)
    got = tb.prefix_attention(q, *both, pl, k.double(), v, ol)
    assert torch.equal(got, want)
    host = tb.prefix_attention(q.cpu(), kp.cpu().expand(2, -1, -1, -1), vp.cpu().expand(2, -1, -1, -1),
                               pl.cpu(), k.cpu(), v.cpu(), ol.cpu())
    assert host.device.type == "cpu" and torch.equal(host, want.cpu())
    low = tb.prefix_attention(q, *both, torch.tensor([-5, 1 << 40], device=cuda), k, v, ol)
    assert torch.equal(low, tb.prefix_attention(q, *both, torch.tensor([0, P], device=cuda), k, v, ol))
    none = tb.prefix_attention(q[:, :0], *both, pl, k[:, :0], v[:, :0], ol[:, :0])
    assert none.shape == (2, 0, H, D)


@pytest.mark.parametrize("rows", [3, 48])
@pytest.mark.parametrize("kind", ["steep", "wide", "zero_v", "small", "large"])
def test_ranges(cuda, rows, kind):
    """Scores far apart, factors of a wide range, weights that count although they are small,
    and the smallest and largest factors."""
    S, N, H, KVH, D, P, L = 1, rows, 4, 2, 64, 777, 30
    q, kp, vp, k, v = inputs(9, S, N, H, KVH, D, P, L)
    g = np.random.default_rng(2)
    if kind == "steep":
        kp *= 12
        k *= 12
    if kind == "wide":
        for c in (kp, vp, k, v):
            c *= 2.0 ** g.integers(-30, 5, c.shape)
    if kind == "zero_v":      # the large weights meet a V of zero
        kp[0, :, 5] = 4 * q[0, 0, ::2].mean(0)
        vp[0, :, 5] = 0
        q[:] = q[0, 0, 0] + 0.01 * q
    if kind == "small":
        q, kp, vp, k, v = q * 1e-15, kp * 1e-15, vp * 1e-30, k * 1e-15, v * 1e-30
    if kind == "large":
        q, kp, vp, k, v = q * 1e15, kp * 1e-15, vp * 1e30, k * 1e-15, v * 1e30
    q, kp, vp, k, v = (a.astype(np.float32) for a in (q, kp, vp, k, v))
    olen = g.integers(0, L + 1, (S, N)).tolist()
    want, bound = reference(q, kp, vp, [P], k, v, olen, D ** -0.5)
    T = lambda a: torch.from_numpy(a).to(cuda)
    check(tb.prefix_attention(T(q), T(kp), T(vp), P, T(k), T(v), torch.tensor(olen, device=cuda)),
          want, bound)


@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("rows", [5, 25, 50, 100])
def test_every_width(cuda, d, rows):
    """Each head_dim on every route: few rows, two tiles of them, 64 and 128 a block; the prefix
    split and ending inside of a tile, ragged groups, a negative scale."""
    print(f"case prefix_attention d={d} rows={rows}", flush=True)
    arrays = inputs(d + rows, 2, rows, 2, 2, d, 703, 21)
    q, kp, vp, k, v = (torch.from_numpy(a).to(cuda) for a in arrays)
    plen = [703, 518 + rows]
    olen = np.random.default_rng(rows).integers(0, 22, (2, rows)).tolist()
    kp[1, :, plen[1]:], vp[1, :, plen[1]:] = float("inf"), float("nan")
    want, bound = reference(*arrays[:3], plen, *arrays[3:], olen, -0.05)
    got = tb.prefix_attention(q, kp, vp, torch.tensor(plen, device=cuda), k, v,
                              torch.tensor(olen, device=cuda), scale=-0.05)
    check(got, want, bound)


@pytest.mark.parametrize("rows", [5, 25, 50, 100])
@pytest.mark.parametrize("d", [64, 128, 192])
def test_errors_are_those_of_f32(cuda, d, rows):
    """The bound above takes every rounding at its largest.  The errors' root mean square is
    held to twice that of the same formula in f32 products and sums, whose order is another:
    a limb or product of limbs that is lost makes it a hundred times as large."""
    arrays = inputs(d + rows, 1, rows, 2, 2, d, 3000, 9)
    want, _ = reference(*arrays[:3], [3000], *arrays[3:], [[0] * rows], d ** -0.5)
    q, kp, vp = (torch.from_numpy(a).to(cuda) for a in arrays[:3])
    x = q[0].transpose(0, 1)
    a = (x @ kp[0].transpose(-1, -2)) * d ** -0.5
    e = torch.exp(a - a.amax(-1, keepdim=True))
    plain = ((e @ vp[0]) / e.sum(-1, keepdim=True)).transpose(0, 1).cpu().numpy()
    got = tb.prefix_attention(q, kp, vp, 3000)[0].cpu().numpy()
    rms = [float(np.sqrt(((g - want[0]) ** 2).mean())) for g in (got, plain)]
    print(f"root mean square error {rms[0]:.3g}, in f32 {rms[1]:.3g}", flush=True)
    assert rms[0] <= 2 * rms[1]


@pytest.mark.parametrize("rows", [2, 20, 48, 100])
@pytest.mark.parametrize("P", [100, 700])
def test_infinities_and_nan(cuda, rows, P):
    """What a row sees counts as the formula has it: a K of -inf or +inf against factors of one
    sign, infinities and NaN in V, NaN in a query."""
    H, KVH, D, L = 2, 2, 32, 9
    q, kp, vp, k, v = inputs(4, 1, rows, H, KVH, D, P, L)
    q[0, 0] = np.abs(q[0, 0])
    q[0, 1] = -np.abs(q[0, 1])
    kp[0, 0, 40, 3] = -np.inf       # head 0: weight 0 for row 0, NaN for row 1
    vp[0, 1, 60, 7] = np.inf        # head 1: dimension 7 infinite, for every row
    vp[0, 1, 61, 9] = -np.inf
    vp[0, 1, 62, 11] = np.nan
    k[0, 1, 1, 2, 5] = np.nan       # row 1, head 1
    T = lambda a: torch.from_numpy(a).to(cuda)
    got = tb.prefix_attention(T(q), T(kp), T(vp), P, T(k), T(v), L).cpu().numpy()
    assert np.isnan(got[0, 1]).all()
    keep = np.arange(P) != 40
    want, bound = reference(q[:, :1, :1], kp[:, :1, keep], vp[:, :1, keep], [P - 1], k[:, :1, :1],
                            v[:, :1, :1], [[L]], D ** -0.5)
    assert (np.abs(got[0, 0, 0] - want[0, 0, 0]) <= bound[0, 0, 0]).all()
    for r in (0, *range(2, rows)):
        assert got[0, r, 1, 7] == np.inf and got[0, r, 1, 9] == -np.inf and np.isnan(got[0, r, 1, 11])
        rest = np.delete(got[0, r, 1], [7, 9, 11])
        assert np.isfinite(rest).all()
    # NaN in one row's query stays there
    q[0, 0, 0, 0] = np.nan
    clean = inputs(4, 1, rows, H, KVH, D, P, L)
    got = tb.prefix_attention(T(q), *(T(a) for a in clean[1:3]), P, *(T(a) for a in clean[3:]), L)
    got = got.cpu().numpy()
    assert np.isnan(got[0, 0, 0]).all() and np.isfinite(got[0, 1:]).all()
    assert np.isfinite(got[0, 0, 1]).all()


def test_positions_far_apart(cuda):
    """Element offsets past 32 bits, of the prefix and of the own caches."""
    P, L, D = 20, 3, 32
    q, kp, vp, k, v = inputs(8, 1, 2, 2, 1, D, P, L)
    want, bound = reference(q, kp, vp, [P], k, v, [[L, 2]], D ** -0.5)
    step = 1 << 28
    room = torch.empty(P * step, device=cuda)      # 21 GB
    views = [room[i * 64:].as_strided((1, P, D), (0, step, 1)) for i in range(2)]
    own = [room[128 + i * 64:].as_strided((2, 1, L, D), (9 * step, 0, step, 1)) for i in range(2)]
    for w, a in zip(views, (kp[0], vp[0])):
        w.copy_(torch.from_numpy(a))
    for w, a in zip(own, (k[0], v[0])):
        w.copy_(torch.from_numpy(a))
    got = tb.prefix_attention(torch.from_numpy(q[0]).to(cuda), *views, P, *own,
                              torch.tensor([L, 2], device=cuda))
    check(got, want[0], bound[0])


def test_captured_two_graphs(cuda):
    """Two graphs with scratch of their own, replayed in turn with other inputs and lengths."""
    arrays = inputs(6, 1, 40, 8, 2, 128, 600, 32)
    q, kp, vp, k, v = (torch.from_numpy(a[0]).to(cuda) for a in arrays)
    pl = torch.tensor(1, device=cuda, dtype=torch.int32)
    ol = torch.zeros(40, device=cuda, dtype=torch.int32)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        tb.prefix_attention(q, kp, vp, pl, k, v, ol)
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = tb.prefix_attention(q, kp, vp, pl, k, v, ol)
        graphs.append((graph, out))
    for step in range(4):
        q.normal_()
        pl.fill_((1, 600, 0, 333)[step])
        ol.copy_(torch.arange(40) * (step + 1) % 33)
        for graph, _ in graphs:
            graph.replay()
        want = tb.prefix_attention(q, kp, vp, pl, k, v, ol)
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, want)


def test_the_streams_workspace(cuda):
    """Without scratch of the caller's the C entries take the stream's, and refuse a capture."""
    arrays = inputs(6, 1, 6, 8, 2, 64, 900, 32)
    q, kp, vp, k, v = (torch.from_numpy(a[0]).to(cuda) for a in arrays)
    want = tb.prefix_attention(q, kp, vp, 900, k, v, 32)
    got = torch.empty_like(want)
    x, scores = torch.randn((3, 4001), device=cuda), torch.zeros(3, device=cuda)
    s, t, b = (torch.empty(3, dtype=d, device=cuda) for d in (torch.float32, torch.int64, torch.int64))
    P = lambda a: a.data_ptr()

    def calls():
        stream = torch.cuda.current_stream().cuda_stream
        yield _lib.lib().tb_prefix_attention(
            P(q), P(kp), P(vp), None, P(k), P(v), None, P(got), 1, 6, 8, 2, 64, 900, 32, 900, 32, 0,
            900 * 64, 64, 0, 900 * 64, 64, 2 * 32 * 64, 32 * 64, 64, 2 * 32 * 64, 32 * 64, 64, 0.125,
            None, 0, stream)
        yield _lib.lib().tb_beam_select(P(x), P(scores), None, P(s), P(t), P(b), 1, 3, 4001, 3, 0,
                                        None, 0, stream)
    assert list(calls()) == [_lib.TB_OK] * 2
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    for a, c in zip((s, t, b), tb.beam_select(x, scores)):
        assert torch.equal(a, c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert list(calls()) == [_lib.TB_ERR_UNSUPPORTED] * 2
        got.zero_()


def test_streams_side_by_side(cuda):
    arrays = inputs(7, 1, 12, 8, 2, 64, 3000, 32)
    q, kp, vp, k, v = (torch.from_numpy(a[0]).to(cuda) for a in arrays)
    want = tb.prefix_attention(q, kp, vp, 3000, k, v, 32)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(tb.prefix_attention(q, kp, vp, 3000, k, v, 32))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_a_beam_search(cuda):
    """Several steps of a beam search of two groups, as they are used together: rotation into the
    beams' caches, attention over prompt and beams, a vocabulary's logits, penalties, the
    selection and the caches' reordering; against the same search in 64 bits that keeps each
    beam's whole history."""
    g = np.random.default_rng(12)
    S, B, H, KVH, D, P, V, steps, layers = 2, 3, 4, 2, 64, 70, 211, 6, 2
    embed = g.standard_normal((layers, V, (H + 2 * KVH) * D)) * 0.7
    head = g.standard_normal((H * D, V)) * 0.3
    w = 1 + 0.1 * g.standard_normal(D)
    f, _ = tb.rope_frequencies(D, 10000.0)
    fn = f.cpu().numpy()
    eos = 5
    T = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(cuda)
    plen = [70, 41]
    kp, vp = g.standard_normal((layers, S, KVH, P, D)), g.standard_normal((layers, S, KVH, P, D))
    E, HD, W, KP, VP = (T(a) for a in (embed, head, w, kp, vp))
    E32, H32, W32, KP32, VP32 = (t.cpu().numpy().astype(np.float64) for t in (E, HD, W, KP, VP))

    # ---- on the device
    kc, vc = (torch.zeros((layers, S, B, KVH, steps + 1, D), device=cuda) for _ in range(2))
    pl = torch.tensor(plen, device=cuda, dtype=torch.int32)
    tokens = torch.full((S, B), 7, device=cuda)
    scores = torch.full((S, B), float("-inf"), device=cuda)
    scores[:, 0] = 0
    done = torch.zeros((S, B), dtype=torch.bool, device=cuda)
    trace = []
    for step in range(steps):
        pos = (pl.long()[:, None] + step).expand(S, B)
        x = 0
        for layer in range(layers):
            qkv = E[layer][tokens]
            q, k, v = (t.unflatten(-1, (-1, D)) for t in qkv.split((H * D, KVH * D, KVH * D), -1))
            q = tb.norm_rope_append(q, k, v, pos, f, kc[layer], vc[layer], step, W, W)
            x = x + tb.prefix_attention(q, KP[layer], VP[layer], pl, kc[layer], vc[layer], step + 1)
        logits = tb.process_logits((x.flatten(-2) @ HD), bias_ids=torch.tensor([eos], device=cuda),
                                   bias_values=torch.tensor([3.0], device=cuda))
        scores, tokens, parents = tb.beam_select(logits, scores, finished=done, eos=eos)
        done = done.gather(1, parents) | (tokens == eos)
        tb.beam_reorder(parents, list(kc), list(vc), step + 1)
        trace.append((scores.cpu().numpy(), tokens.cpu().numpy(), parents.cpu().numpy()))
    assert done.any()

    # ---- in 64 bits, each beam with its own history of rows
    def rotate(x, pos):
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * W32
        a, b, t = x[..., :D // 2], x[..., D // 2:], pos * fn
        return np.concatenate((a * np.cos(t) - b * np.sin(t), b * np.cos(t) + a * np.sin(t)), -1)

    def attend(q, k, v):
        a = q @ k.T / D ** 0.5
        e = np.exp(a - a.max())
        return e / e.sum() @ v

    for s in range(S):
        beams = [(0.0 if b == 0 else -np.inf, 7, False, [([], []) for _ in range(layers)])
                 for b in range(B)]
        for step in range(steps):
            items = []
            rows = []
            for b, (score, token, ended, hist) in enumerate(beams):
                x, new = np.zeros(H * D), []
                for layer in range(layers):
                    row = E32[layer][token].reshape(-1, D)
                    q, k = rotate(row[:H], plen[s] + step), rotate(row[H:H + KVH], plen[s] + step)
                    ks, vs = hist[layer][0] + [k], hist[layer][1] + [row[H + KVH:]]
                    new.append((ks, vs))
                    for h in range(H):
                        j = h // (H // KVH)
                        kk = np.concatenate((KP32[layer, s, j, :plen[s]], [r[j] for r in ks]))
                        vv = np.concatenate((VP32[layer, s, j, :plen[s]], [r[j] for r in vs]))
                        x[h * D:(h + 1) * D] += attend(q[h], kk, vv)
                rows.append(new)
                if not np.isfinite(score):
                    continue
                y = x @ H32
                y[eos] += 3.0
                y = y - np.log(np.exp(y - y.max()).sum()) - y.max() + score
                items += [(score, eos, b)] if ended else [(y[t], t, b) for t in range(V)]
            items.sort(key=lambda i: -i[0])
            got = trace[step]
            for j in range(B):
                assert abs(items[j][0] - got[0][s, j]) < 1e-4
                assert (items[j][1], items[j][2]) == (got[1][s, j], got[2][s, j]), (s, step, j)
            beams = [(float(got[0][s, j]), t, beams[b][2] or t == eos, rows[b])
                     for j, (_, t, b) in enumerate(items[:B])]


@pytest.mark.parametrize("rows", [2, 20, 48, 100])
@pytest.mark.parametrize("P", [100, 700])
def test_nan_beside_far_larger_scores(cuda, rows, P):
    """A NaN that a row sees is in its result, however small the weights around it are: another
    wave's or split's scores are so much larger (200 and more) that all of its are 0 in f32."""
    H, KVH, D, L = 2, 2, 32, 9
    q, kp, vp, k, v = inputs(5, 1, rows, H, KVH, D, P, L)
    q = np.abs(q) + 0.5
    kp[0, :, 5] = 100
    kp[0, 0, 40, 3] = np.nan        # head 0: every row's score of position 40
    vp[0, 1, 40, 7] = np.nan        # head 1: a weight of 0 in f32 meets NaN and infinity
    vp[0, 1, P - 30, 9] = np.inf
    v[0, 0, 1, 3, 11] = np.nan      # row 0's own cache
    T = lambda a: torch.from_numpy(a).to(cuda)
    got = tb.prefix_attention(T(q), T(kp), T(vp), P, T(k), T(v), L).cpu().numpy()[0]
    assert np.isnan(got[:, 0]).all()
    assert np.isnan(got[:, 1, 7]).all() and not np.isfinite(got[:, 1, 9]).any()
    assert np.isnan(got[0, 1, 11]) and np.isfinite(got[1:, 1, 11]).all()
    # the one position that counts, whose weight is 1 to f32's last bit
    rest = np.delete(got[:, 1], [7, 9, 11], 1)
    want = np.delete(vp[0, 1, 5], [7, 9, 11])
    assert (np.abs(rest - want) <= 32 * U * np.abs(want)).all()


def split_scratch(S, rows, H, KVH, D, P, L):
    """The scratch of a call whose prefix is split: past the one launch of short caches."""
    size = _lib.lib().tb_prefix_attention_scratch(S, rows, H, KVH, D, P, L)
    assert size > 0
    return size


@pytest.mark.parametrize("d", [64, 160])
@pytest.mark.parametrize("rows", [4, 12, 30, 70])
def test_layouts_of_split_prefixes(cuda, rows, d):
    """The layouts of test_layouts where the prefix is split over blocks, two query heads a KV
    head: 8, 24, 60 and 140 rows of it are a tile, two tiles and blocks of 64 and 128 rows; own
    caches of up to three splits (with 4 rows)."""
    print(f"case prefix_attention layouts rows={rows} d={d}", flush=True)
    S, H, KVH, P, L = 2, 8, 4, 700, 150
    split_scratch(S, rows, H, KVH, d, P, L)
    arrays = inputs(rows + d, 1, S * rows, H, KVH, d, P, L)
    q, k, v = (a.reshape(S, rows, *a.shape[2:]) for a in (arrays[0], *arrays[3:]))
    olen = np.arange(S * rows).reshape(S, rows) * 37 % (L + 1)
    plen = [690, 333]
    both = [np.broadcast_to(a, (S, *a.shape[1:])) for a in arrays[1:3]]
    expected, bound = reference(q, *both, plen, k, v, olen.tolist(), d ** -0.5)
    q, k, v, kp, vp = (torch.from_numpy(a).to(cuda) for a in (q, k, v, *arrays[1:3]))
    pl, ol = torch.tensor(plen, device=cuda), torch.from_numpy(olen).to(cuda)
    both = [c.expand(S, -1, -1, -1) for c in (kp, vp)]      # one prompt under both groups
    want = tb.prefix_attention(q, *(c.contiguous() for c in both), pl, k, v, ol)
    check(want, expected, bound)
    assert torch.equal(tb.prefix_attention(q, *both, pl, k, v, ol), want)
    # positions before heads, wider rows, spare positions, with NaN in the gaps
    wide = [torch.full((S, P + 3, KVH, d + 4), float("nan"), device=cuda) for _ in range(2)]
    views = []
    for w, c in zip(wide, both):
        w[:, :P, :, :d] = c.transpose(1, 2)
        views.append(w[:, :P, :, :d].transpose(1, 2))
    own = [torch.full((S, rows, L + 1, KVH, d + 8), float("nan"), device=cuda) for _ in range(2)]
    mine = []
    for w, c in zip(own, (k, v)):
        w[..., :L, :, :d] = c.transpose(2, 3)
        mine.append(w[..., :L, :, :d].transpose(2, 3))
    assert torch.equal(tb.prefix_attention(q, *views, pl, *mine, ol), want)
    # K laid out one way, V another; own caches whose groups are not a constant stride apart
    apart = [torch.stack((c[0], c[0], c[1])) for c in (k, v)]
    assert torch.equal(tb.prefix_attention(q, views[0], both[1], pl, *(c[::2] for c in apart), ol),
                       want)
    # one own cache under every sequence of a group
    alone = [c[:, :1].contiguous() for c in (k, v)]
    shared = [c.expand(-1, rows, -1, -1, -1) for c in alone]
    assert torch.equal(tb.prefix_attention(q, *both, pl, *shared, ol),
                       tb.prefix_attention(q, *both, pl, *(c.contiguous() for c in shared), ol))
    off = torch.empty(q.numel() + 1, device=cuda)[1:].view(q.shape).copy_(q)
    assert torch.equal(tb.prefix_attention(off, *both, pl, k, v, ol), want)
    # lengths outside of the caches
    low = tb.prefix_attention(q, *both, torch.tensor([-5, 1 << 40], device=cuda), k, v, ol - 20)
    assert torch.equal(low, tb.prefix_attention(q, *both, torch.tensor([0, P], device=cuda), k, v,
                                                (ol - 20).clamp(min=0)))
    high = tb.prefix_attention(q, *both, pl, k, v, ol + (1 << 33))
    assert torch.equal(high, tb.prefix_attention(q, *both, pl, k, v, torch.full_like(ol, L)))


@pytest.mark.parametrize("rows", [2, 12, 24, 50])
@pytest.mark.parametrize("far", ["positions", "heads", "groups"])
def test_split_prefixes_far_apart(cuda, rows, far):
    """Element offsets past 32 bits on the routes that split the prefix: 4, 24, 48 and 100 rows
    of a KV head, and the own caches beside them."""
    print(f"case prefix_attention far apart rows={rows} {far}", flush=True)
    S, H, KVH, D, P, L = 2, 4, 2, 32, 345, 70
    split_scratch(S, rows, H, KVH, D, P, L)
    arrays = inputs(rows, S, rows, H, KVH, D, P, L)
    olen = (np.arange(S * rows).reshape(S, rows) * 29 % (L + 1)).tolist()
    plen = [P, 340]
    want, bound = reference(*arrays[:3], plen, *arrays[3:], olen, D ** -0.5)
    q, kp, vp, k, v = (torch.from_numpy(a).to(cuda) for a in arrays)
    # strides of group, KV head and position of the prefix, of sequence, KV head and position of
    # the own caches; where V lies behind K; where the own caches begin; elements in all
    big, small = 1 << 32, 1 << 15
    if far == "positions":      # the prefix's at 2^24, the own ones' at 2^26
        st, own = (1 << 10, 1 << 11, 1 << 24), (1 << 13, 1 << 12, 1 << 26)
        behind, v_prefix, v_own, room = 1 << 20, 1 << 9, 1 << 11, (P + 1) << 24
    elif far == "heads":
        st, own = (small, big, 32), (small, big, 32)
        behind, v_prefix, v_own, room = 4 * small, 2 * small, 1 << 22, big + (1 << 23)
    else:                       # the last of 100 sequences at 99 * 2^26
        st, own = (big, small, 32), (1 << 26, small, 32)
        behind, v_prefix, v_own = 4 * small, 2 * small, 1 << 22
        room = max(big, S * rows << 26) + (1 << 23)
    room = torch.empty(room, device=cuda)      # 17 to 27 GB
    views = [room[x:].as_strided((S, KVH, P, D), (*st, 1)) for x in (0, v_prefix)]
    mine = [room[behind + x:].as_strided((S, rows, KVH, L, D), (rows * own[0], *own, 1))
            for x in (0, v_own)]
    for w, a in zip((*views, *mine), (kp, vp, k, v)):
        w.copy_(a)
    for w, a in zip((*views, *mine), (kp, vp, k, v)):
        assert torch.equal(w, a)      # no two of them share memory
    got = tb.prefix_attention(q, *views, torch.tensor(plen, device=cuda), *mine,
                              torch.tensor(olen, device=cuda))
    check(got, want, bound)


@pytest.mark.parametrize("rows,P,joined", [(32, 304, True), (38, 304, True), (39, 304, False),
                                           (128, 80, True), (129, 80, False), (4, 305, False)])
def test_one_launch_or_two(cuda, rows, P, joined):
    """Short caches in one launch for few sequences only: at the borders of 20 tiles in all and of
    blocks times tiles, of which 6144 are 307 blocks of 20 tiles and 1024 of 6."""
    H, KVH, D, L = 16, 8, 64, 16
    size = _lib.lib().tb_prefix_attention_scratch(1, rows, H, KVH, D, P, L)
    assert (size == 0) == joined
    arrays = inputs(rows + P, 1, rows, H, KVH, D, P, L)
    olen = np.random.default_rng(rows).integers(0, L + 1, (1, rows)).tolist()
    want, bound = reference(*arrays[:3], [P], *arrays[3:], olen, D ** -0.5)
    q, kp, vp, k, v = (torch.from_numpy(a).to(cuda) for a in arrays)
    check(tb.prefix_attention(q, kp, vp, P, k, v, torch.tensor(olen, device=cuda)), want, bound)
