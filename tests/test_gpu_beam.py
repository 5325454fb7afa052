"""beam_select and beam_reorder against their definitions: tokens, beams and moved rows have to
be equal; a score is rounded once (2^-24 of it) and its sum of exponentials kept in 64
bits (1e-9 allows for every rounding there)."""
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest
import torch

import torchburn_amd as tb

pytestmark = pytest.mark.gpu


def select(x, scores, k, ended=None, eos=None):
    """(scores, tokens, beams) of one group, in float64: x [B, V]."""
    x = x.astype(np.float64)
    B, V = x.shape
    items = []
    for b in range(B):
        s = float(scores[b])
        if not np.isfinite(s):
            continue
        if ended is not None and ended[b]:
            items.append((-s, b, 0.0, eos))
            continue
        if np.isnan(x[b]).any() or (x[b] == np.inf).any() or (x[b] == -np.inf).all():
            continue
        top = x[b].max()
        lse = np.log(np.exp(x[b] - top).sum()) + top
        for t in np.argsort(-x[b], kind="stable")[:k]:
            if x[b, t] > -np.inf:
                items.append((-(x[b, t] - lse + s), b, -x[b, t], int(t)))
    items = sorted(items)[:k]
    items += [(np.inf, -1, 0.0, -1)] * (k - len(items))
    return (np.array([-i[0] for i in items]), np.array([i[3] for i in items]),
            np.array([i[1] for i in items]))


def check(got, x, scores, k, ended=None, eos=None):
    s, t, b = (a.cpu().numpy() for a in got)
    G = x.shape[0]
    assert s.shape == t.shape == b.shape == (G, k)
    for g in range(G):
        ws, wt, wb = select(x[g], scores[g], k, None if ended is None else ended[g], eos)
        assert np.array_equal(t[g], wt) and np.array_equal(b[g], wb), (g, t[g], wt, b[g], wb)
        real = wt >= 0
        assert (np.abs(s[g][real] - ws[real]) <= 2.0 ** -24 * np.abs(ws[real]) + 1e-9).all()
        assert np.isneginf(s[g][~real]).all()


CASES = [
    # groups, beams, vocab, k
    (1, 1, 1, 1), (1, 1, 3, 5), (1, 2, 5, 4), (2, 3, 1000, 3), (1, 4, 1023, 8), (1, 4, 1024, 8),
    (3, 4, 1025, 8), (1, 4, 32003, 8), (5, 8, 4099, 16), (2, 16, 50257, 32), (1, 64, 3001, 64),
    (1, 1, 151936, 64), (2, 5, 128256, 10), (40, 16, 9001, 1), (1, 3, 1 << 20, 64),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("kind", ["plain", "ties", "masked"])
def test_select(cuda, case, kind):
    G, B, V, k = case
    print(f"case beam_select {case} {kind}", flush=True)
    g = np.random.default_rng(V + k)
    x = (3 * g.standard_normal((G, B, V))).astype(np.float32)
    scores = -np.cumsum(3 * g.random((G, B)), -1).astype(np.float32)
    ended, eos = None, None
    if kind == "ties":      # a few values many times, beams alike in part
        x = np.round(x * 2) / 2
        x[:, B // 2:] = x[:, :1]
        scores[:, B // 2:] = scores[:, :1]
        x[x == 0] = -0.0
    if kind == "masked":
        x[g.random(x.shape) < 0.7] = -np.inf
        x[0, 0] = -np.inf           # a row without any
        x[0, -1, 1:] = -np.inf      # and one with a single token
        ended = g.random((G, B)) < 0.3
        eos = V - 1
    T = lambda a: None if a is None else torch.from_numpy(a).to(cuda)
    got = tb.beam_select(T(x), T(scores), k=k, finished=T(ended), eos=eos)
    check(got, x, scores, k, ended, eos)
    if G > 1:
        return
    one = tb.beam_select(T(x[0]), T(scores[0]), k=k, finished=T(None if ended is None else ended[0]),
                         eos=eos)
    for a, b in zip(got, one):
        assert torch.equal(a[0], b)


def test_select_values_out_of_range(cuda):
    """Scores of -inf, NaN, inf and very low ones; logits with NaN, inf, the lowest number; rows
    of equal logits; the largest spread."""
    g = np.random.default_rng(5)
    B, V, k = 12, 5001, 24
    x = (3 * g.standard_normal((1, B, V))).astype(np.float32)
    scores = np.array([[0, -np.inf, np.nan, np.inf, -1e9, -3e38, -1, -2, -3, -4, -5, -6]],
                      np.float32)
    x[0, 6, 17] = np.nan
    x[0, 7, 4000] = np.inf
    x[0, 8] = np.finfo(np.float32).min      # masked by the lowest value, but for two
    x[0, 8, 100] = x[0, 8, 99] = 2.0
    x[0, 9] = 0.25
    x[0, 10] = np.linspace(-3e38, 3e38, V)
    x[0, 11] *= 200
    T = lambda a: torch.from_numpy(a).to(cuda)
    check(tb.beam_select(T(x), T(scores), k=k), x, scores, k)
    only = tb.beam_select(T(x[:, 8:10]), T(scores[:, 8:10]), k=64)
    check(only, x[:, 8:10], scores[:, 8:10], 64)
    # the first step: every beam the same, one of them alive
    x[0, :] = x[0, :1]
    scores = np.full((1, B), -np.inf, np.float32)
    scores[0, 0] = 0
    got = tb.beam_select(T(x), T(scores))
    check(got, x, scores, B)
    assert (got[2] == 0).all()


def test_select_forms(cuda):
    """Host tensors, halves, unaligned views, k past the candidates, no groups."""
    x = torch.randn((2, 3, 41), dtype=torch.float16)
    scores = torch.tensor([[0.0, -1, -2], [-3, -4, -5]])
    got = tb.beam_select(x, scores, k=50)
    assert all(t.device.type == "cpu" for t in got)
    check(got, x.numpy(), scores.numpy(), 50)
    wide = torch.randn((2, 3, 45), device=cuda)
    check(tb.beam_select(wide[..., 1:42], scores.to(cuda), k=7), wide[..., 1:42].cpu().numpy(),
          scores.numpy(), 7)
    flat = torch.randn(1 + 6 * 4097, device=cuda)[1:].view(2, 3, 4097)      # 4 bytes off
    check(tb.beam_select(flat, scores.to(cuda), k=7), flat.cpu().numpy(), scores.numpy(), 7)
    none = tb.beam_select(torch.zeros((0, 3, 41), device=cuda), torch.zeros((0, 3), device=cuda))
    assert none[0].shape == none[1].shape == (0, 3)


@pytest.mark.parametrize("beams", [1, 2, 3, 4, 5, 8, 13, 16, 31, 33, 64])
@pytest.mark.parametrize("form", ["number", "lengths"])
def test_reorder(cuda, beams, form):
    print(f"case beam_reorder {beams} {form}", flush=True)
    g = np.random.default_rng(beams)
    G, L, H, S, D = 2, 3, 2, 21, 96
    k, v = (torch.randn((L, G, beams, H, S, D), device=cuda) for _ in range(2))
    par = g.integers(-2, beams + 2, (G, beams))
    par[0] = g.permutation(beams)      # a permutation in one group
    lens = g.integers(0, S + 1, (G, beams))
    if form == "number":
        lens[:] = 17
    want = []
    for c in (k, v):
        was, c = c.cpu().numpy(), c.cpu().numpy().copy()
        for i in range(G):
            for j in range(beams):
                p = par[i, j]
                if 0 <= p < beams:
                    c[:, i, j, :, :lens[i, p]] = was[:, i, p, :, :lens[i, p]]
        want.append(c)
    n = 17 if form == "number" else torch.from_numpy(lens).to(cuda)
    tb.beam_reorder(torch.from_numpy(par).to(cuda), list(k), list(v), n)
    assert np.array_equal(k.cpu().numpy(), want[0]) and np.array_equal(v.cpu().numpy(), want[1])


def test_reorder_layouts(cuda):
    """Positions before heads, spare rows, one group without its dimension, lengths past the
    cache, caches that are converted and written back, more layers than a launch takes."""
    par = torch.tensor([2, 0, 0, 3], device=cuda)
    base = torch.randn((2, 4, 11, 3, 64), device=cuda)
    k, v = (c[:, :9].transpose(1, 2) for c in base)      # [4, 3, 9, 64]
    rows = base.clone()
    tb.beam_reorder(par, [k], [v], torch.tensor([5, 7, 100, -3], device=cuda))
    want = rows.clone()
    want[:, 0, :9] = rows[:, 2, :9]
    want[:, 1, :5] = rows[:, 0, :5]
    want[:, 2, :5] = rows[:, 0, :5]
    assert torch.equal(base, want)
    hk, hv = rows[0, :, :9].transpose(1, 2).cpu(), rows[1, :, :9].transpose(1, 2).double()
    tb.beam_reorder(par, [hk], [hv], torch.tensor([5, 7, 100, -3], device=cuda))
    assert torch.equal(hk, k.cpu()) and torch.equal(hv, v.double())
    many = torch.randn((2, 70, 4, 1, 3, 32), device=cuda)
    was = many.clone()
    tb.beam_reorder(par, many[0], many[1], 3)
    assert torch.equal(many, was[:, :, par])
    tb.beam_reorder(par, [], [], 3)


def test_captured_and_two_streams(cuda):
    x = torch.randn((2, 4, 5000), device=cuda)
    scores = torch.zeros((2, 4), device=cuda)
    k, v = (torch.randn((2, 2, 4, 2, 8, 64), device=cuda) for _ in range(2))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            _, _, b = tb.beam_select(x, scores)
            tb.beam_reorder(b, list(k), list(v), 5)
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = tb.beam_select(x, scores)
            tb.beam_reorder(out[2], list(k), list(v), 5)
        graphs.append((graph, out))
    for step in range(4):
        x.normal_()
        was = k.clone()
        graph, out = graphs[step % 2]
        graph.replay()
        want = tb.beam_select(x, scores)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
        for i in range(2):
            assert torch.equal(k[:, i, :, :, :5], was[:, i, out[2][i], :, :5])
            assert torch.equal(k[:, i, :, :, 5:], was[:, i, :, :, 5:])


def test_captured_widest(cuda):
    """64 beams and 64 results, whose selection needs more LDS than a launch has by itself."""
    x, scores = torch.randn((64, 3001), device=cuda), torch.randn(64, device=cuda)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tb.beam_select(x, scores, k=64)
    for _ in range(3):
        x.normal_()
        graph.replay()
        want = tb.beam_select(x, scores, k=64)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_a_cache_given_twice(cuda):
    k = torch.randn((2, 1, 3, 32), device=cuda)
    par = torch.tensor([1, 0], device=cuda)
    for c in (k, k.cpu()):
        with pytest.raises(tb.UnsupportedOpError, match="twice"):
            tb.beam_reorder(par, [c], [c], 2)


def test_reorder_converted_rows_stay(cuda):
    """Of caches in 64 bits only what is taken over is rounded."""
    par = torch.tensor([1, 1, 0], device=cuda)
    k, v = (torch.randn((3, 2, 5, 32), device=cuda, dtype=torch.float64) for _ in range(2))
    want = []
    for c in (k, v):
        w = c.clone()
        w[:, :, :3] = c[par, :, :3].float().double()
        w[1] = c[1]      # goes on from itself
        want.append(w)
    tb.beam_reorder(par, [k], [v], 3)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_reorder_stacked(cuda):
    """Stacks with spare layers, positions and unlike strides, as the lists of their layers."""
    par = torch.tensor([[2, 0, 1], [1, 1, 1]], device=cuda)
    kb = torch.randn((4, 2, 3, 2, 9, 64), device=cuda)
    vb = torch.randn((3, 2, 5, 2, 3, 2, 64), device=cuda)
    kb2, vb2 = kb.clone(), vb.clone()

    def stacks(kb, vb):
        k = kb[1:, :, :, :, 2:7]                            # [3, 2, 3, 2, 5, 64]
        return k, vb.permute(0, 1, 4, 3, 2, 5, 6)[..., 1, :]  # [3, 2, 3, 2, 5, 64]
    k, v = stacks(kb, vb)
    assert k.shape == v.shape
    tb.beam_reorder(par, k, v, 4)
    k2, v2 = stacks(kb2, vb2)
    for c in (k2, v2):
        for g in range(2):
            c[:, g, :, :, :4] = c[:, g, par[g], :, :4].clone()
    assert torch.equal(kb, kb2) and torch.equal(vb, vb2)
    tb.beam_reorder(par, list(k), v, 4)
    for c in (k2, v2):
        for g in range(2):
            c[:, g, :, :, :4] = c[:, g, par[g], :, :4].clone()
    assert torch.equal(kb, kb2) and torch.equal(vb, vb2)
    with pytest.raises(tb.UnsupportedOpError, match="twice"):
        tb.beam_reorder(par, k, k, 4)
    with pytest.raises(tb.UnsupportedOpError, match="twice"):
        tb.beam_reorder(par, k[:1].expand(3, -1, -1, -1, -1, -1), v, 4)


def test_far_apart(cuda):
    """Element offsets past 32 bits: between beams, positions and groups, and in the logits."""
    par = torch.tensor([[1, 0], [1, 1]], device=cuda)
    far = torch.empty((1 << 32) + (1 << 20), device=cuda)
    shape = (2, 2, 1, 3, 32)
    for strides in ((4096, 1 << 32, 32, 128, 1), (4096, 1024, 32, 1 << 31, 1),
                    (1 << 32, 1024, 32, 128, 1)):
        k, v = (far[off:].as_strided(shape, strides) for off in (0, 1 << 16))
        for c in (k, v):
            c.copy_(torch.randn(shape, device=cuda))
        want = [c.clone() for c in (k, v)]
        for c in want:
            c[0, :, :, :2] = c[0, [1, 0], :, :2]
            c[1, :, :, :2] = c[1, [1, 1], :, :2]
        tb.beam_reorder(par, [k], [v], 2)
        assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    del far, k, v
    vocab, beams, groups = 1 << 20, 64, 65      # 4160 rows
    logits = torch.empty((groups, beams, vocab), device=cuda)
    logits[:-1] = 0.0
    last = torch.randn((1, beams, vocab), device=cuda)
    logits[-1] = last[0]
    scores = torch.randn((groups, beams), device=cuda)
    got = tb.beam_select(logits, scores, k=5)
    for a, b in zip(got, tb.beam_select(last, scores[-1:], k=5)):
        assert torch.equal(a[-1:], b)
    assert torch.equal(got[1][0], torch.arange(5, device=cuda))     # ties: the lowest tokens
    assert torch.equal(got[2][0], scores[0].argmax().expand(5))


@pytest.mark.parametrize("case", [(1, 47, 2000, 64), (1, 48, 2000, 64), (1, 49, 2000, 64), (2, 63, 9001, 64),
                                  (1, 64, 1000, 64)], ids=lambda c: "-".join(map(str, c)))
def test_select_at_the_border_of_lds(cuda, case):
    """Selections whose second kernel takes about the 64 KiB that a launch has by itself."""
    test_select(cuda, case, "plain")
    test_select(cuda, case, "ties")


def test_wide_selections_side_by_side(cuda):
    """Threads whose selections need LDS of different sizes past what a launch has by itself."""
    shapes = [(64, 1000), (64, 3001), (64, 70001), (60, 200001)]
    inputs = [(torch.randn(s, device=cuda), torch.randn(s[0], device=cuda)) for s in shapes]
    want = [tb.beam_select(x, s, k=64) for x, s in inputs]
    torch.cuda.synchronize()

    def many(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [tb.beam_select(*inputs[i], k=64) for _ in range(25)]
            torch.cuda.current_stream().synchronize()
        return got
    with ThreadPoolExecutor(len(shapes)) as pool:
        for got, w in zip(pool.map(many, range(len(shapes))), want):
            assert all(torch.equal(a, b) for g in got for a, b in zip(g, w))


def test_two_streams_and_graphs(cuda):
    """Two searches, each eager and captured on a stream of its own, side by side: every result,
    and both K and V, after every replay."""
    B, L, S = 4, 2, 9
    searches = []
    for i in range(2):
        stream = torch.cuda.Stream()
        x, scores = torch.randn((2, B, 30011), device=cuda), torch.randn((2, B), device=cuda)
        k, v = (torch.randn((L, 2, B, 2, S, 64), device=cuda) for _ in range(2))
        lens = torch.randint(0, S + 1, (2, B), device=cuda)
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = tb.beam_select(x, scores)
            tb.beam_reorder(out[2], k, list(v), lens)
        searches.append((stream, x, scores, k, v, lens, graph, out))
    for step in range(4):
        torch.cuda.synchronize()
        was, eager = [], []
        for stream, x, scores, k, v, lens, graph, out in searches:
            with torch.cuda.stream(stream):
                x.normal_()
                lens.random_(0, S + 1)
                was.append((k.clone(), v.clone()))
        for stream, x, scores, k, v, lens, graph, out in searches:
            with torch.cuda.stream(stream):
                if step != 2:
                    graph.replay()
                else:      # an eager step between the replays
                    got = tb.beam_select(x, scores)
                    tb.beam_reorder(got[2], list(k), list(v), lens)
                    for a, b in zip(out, got):
                        a.copy_(b)
        torch.cuda.synchronize()
        for (stream, x, scores, k, v, lens, graph, out), before in zip(searches, was):
            check(out, x.cpu().numpy(), scores.cpu().numpy(), B)
            par, n = out[2].tolist(), lens.tolist()
            for now, w in zip((k, v), before):
                want = w.clone()
                for g in range(2):
                    for j, p in enumerate(par[g]):
                        want[:, g, j, :, :n[g][p]] = w[:, g, p, :, :n[g][p]]
                assert torch.equal(now, want)


@pytest.mark.parametrize("V", [1000, 5003, 128256])
@pytest.mark.parametrize("step", [1, -1])
def test_order_between_beams(cuda, V, step):
    """Beams with the same logits at other places and moved by whole numbers: their values differ
    by their scores alone, 2e-10 from beam to beam, twice what a log-sum may be off: the fit's
    5.5e-11 and 3.4e-16 of a logit up to 10^3."""
    g = np.random.default_rng(V)
    B = 16
    base = np.round(3 * g.standard_normal(V) * 1024) / 1024      # moved without a rounding
    base[7] = np.abs(base).max() + 2
    x = np.stack([g.permutation(base) + b * 60 for b in range(B)]).astype(np.float32)
    assert (np.sort(x, -1) == np.sort(base) + 60.0 * np.arange(B)[:, None]).all()
    scores = (2e-10 * step * np.arange(B)).astype(np.float32)
    got = tb.beam_select(torch.from_numpy(x).to(cuda), torch.from_numpy(scores).to(cuda))
    order = np.arange(B)[::-step]
    assert got[2].tolist() == order.tolist()
    assert got[1].tolist() == x.argmax(-1)[order].tolist()


def test_a_search_with_few_continuations(cuda):
    """A loop of selection and reordering whose groups have fewer continuations than beams at
    first and in one group for good, with own caches of different lengths and beams that end:
    each beam's cache holds its own history, against a search over lists in 64 bits."""
    g = np.random.default_rng(3)
    G, B, V, D, S, steps, eos = 2, 7, 5, 32, 12, 6, 4
    table = (2 * g.standard_normal((G, V, V))).astype(np.float32)      # logits by the last token
    table[:, :, 3] = -np.inf
    table[0, :, eos] += 3          # group 0: beams end
    table[1, :, 1:] = -np.inf      # group 1: token 0 alone
    start = np.array([2, 5])
    T = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)
    logits_of, group = T(table), torch.arange(G, device=cuda)[:, None]
    # ---- on the device: a cache's rows are the tokens taken
    k, v = (torch.full((1, G, B, 1, S, D), -7.0, device=cuda) for _ in range(2))
    none_to_turn = torch.zeros(0, dtype=torch.float64, device=cuda)
    tokens = torch.zeros((G, B), dtype=torch.int64, device=cuda)
    scores = torch.full((G, B), float("-inf"), device=cuda)
    scores[:, 0] = 0
    ended = torch.zeros((G, B), dtype=torch.bool, device=cuda)
    kv_len = T(start).int()[:, None].repeat(1, B)
    for _ in range(steps):
        rows = tokens.float()[..., None, None].expand(G, B, 1, D)
        tb.norm_rope_append(rows, rows, -rows, kv_len.long(), none_to_turn, k[0], v[0], kv_len)
        scores, tokens, beams = tb.beam_select(logits_of[group, tokens], scores, finished=ended,
                                               eos=eos)
        tb.beam_reorder(beams, k, v, kv_len + 1)
        source, none = beams.clamp(min=0), beams < 0
        ended = (ended.gather(-1, source) | (tokens == eos)) & ~none
        kv_len = (kv_len + 1).gather(-1, source)
        tokens = tokens.clamp(min=0)
    assert ended[0].any() and (beams[1, 1:] == -1).all() and (beams[0] >= 0).all()
    # ---- over lists
    x = table.astype(np.float64)
    with np.errstate(divide="ignore"):
        x = x - np.log(np.exp(x).sum(-1, keepdims=True))
    for i in range(G):
        held = [(0.0, [0], False)]
        for _ in range(steps):
            items = []
            for s, hist, done in held:
                items += [(s, hist + [eos], True)] if done else \
                    [(np.float32(s + x[i, hist[-1], t]), hist + [t], t == eos)
                     for t in range(V) if x[i, hist[-1], t] > -np.inf]
            held = sorted(items, key=lambda c: -c[0])[:B]
        assert len(held) == int((beams[i] >= 0).sum())
        for j, (s, hist, done) in enumerate(held):
            assert abs(float(scores[i, j]) - s) < 1e-5 and bool(ended[i, j]) == done
            assert int(tokens[i, j]) == hist[-1] and int(kv_len[i, j]) == start[i] + steps
            n = start[i]
            row = k[0, i, j, 0, :, 0].tolist()
            assert row[n:n + steps] == hist[:steps] and row[:n] == [-7.0] * n
            assert row[n + steps:] == [-7.0] * (S - n - steps)
            assert torch.equal(v[0, i, j, 0, n:n + steps], -k[0, i, j, 0, n:n + steps])
