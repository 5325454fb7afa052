"""process_logits and greedy_tokens against the definition in 64 bits.

Bound: every operation rounds to f32 once, off by u = 2^-24 of its result: the
division or product by the repetition penalty (which is itself held to u), the
product and difference of the frequency penalty, the presence and the bias: six
roundings of values no larger than |x| max(rep, 1 / rep) + freq count + |pres| +
sum|bias|, and one per further entry of a bias named several times.
"""
import numpy as np
import pytest
import torch

import torchburn_amd as tb

pytestmark = pytest.mark.gpu


def pack(bits):
    n = bits.shape[-1]
    w = np.zeros((*bits.shape[:-1], (n + 31) // 32 * 32), bool)
    w[..., :n] = bits
    return np.packbits(w.reshape(*bits.shape[:-1], -1, 32), axis=-1, bitorder="little") \
        .view(np.uint32)[..., 0].astype(np.int32, casting="unsafe").reshape(*bits.shape[:-1], -1)


def reference(x, hist, lens, prompts, rep, pres, freq, ids, bias, allowed, paths):
    """(y, bound) in float64; per-row lists: hist[r] tokens, paths[r] tokens, ids[r], bias[r]."""
    R, V = x.shape
    y, bound = x.astype(np.float64), np.zeros((R, V))
    for r in range(R):
        path = [t for t in paths[r] if 0 <= t < V]
        toks = [t for t in hist[r][:lens[r]] if 0 <= t < V]
        made = [t for i, t in enumerate(hist[r][:lens[r]]) if 0 <= t < V and i >= prompts[r]]
        size = np.abs(y[r]) * max(rep[r], 1 / rep[r])
        for t in set(toks) | set(path):
            y[r, t] = y[r, t] / rep[r] if y[r, t] > 0 else y[r, t] * rep[r]
        count = np.bincount(np.array(made + path, dtype=np.int64), minlength=V)
        y[r] -= freq[r] * count + pres[r] * (count > 0)
        size += abs(freq[r]) * count + abs(pres[r]) * (count > 0)
        k = 6
        for t, b in zip(ids[r], bias[r]):
            if 0 <= t < V:
                y[r, t] += b
                size[t] += abs(b)
                k += 1
        if allowed is not None:
            y[r, ~allowed[r]] = -np.inf
        bound[r] = k * 2.0 ** -24 * size + 2.0 ** -149
    return y, bound


def best(y):
    out = []
    for row in np.where(np.isnan(y), -np.inf, y):
        t = int(np.argmax(row))
        out.append(t if row[t] > -np.inf else -1)
    return out


CASES = [
    # R, V, groups, hist, n_bias, bias groups, allow, nodes
    (1, 1, 1, 4, 0, 1, None, 0),
    (1, 151936, 1, 300, 0, 1, None, 0),
    (3, 33, 3, 7, 5, 1, 0.5, 0),
    (5, 4097, 1, 60, 40, 5, 0.9, 5),
    (6, 1000, 2, 50, 8, 3, 0.3, 3),
    (64, 32003, 1, 2000, 0, 1, 0.02, 64),
    (40, 8191, 4, 100, 300, 2, 0.01, 10),
    (70, 513, 1, 0, 0, 1, 0.7, 70),
    (2, 65536, 2, 5000, 17, 1, None, 1),
    (130, 50001, 130, 333, 3, 130, 0.97, 0),
    (7, 100, 1, 0, 0, 1, None, 0),         # nothing to do
]


@pytest.mark.parametrize("R,V,G,hist,nb,bg,allow,nodes", CASES)
@pytest.mark.parametrize("per_row", [False, True])
def test_process_logits(cuda, R, V, G, hist, nb, bg, allow, nodes, per_row):
    print(f"case process_logits R={R} V={V} groups={G} hist={hist} bias={nb} allow={allow} "
          f"nodes={nodes} per_row={per_row}", flush=True)
    g = np.random.default_rng(R * V + hist)
    x = (g.standard_normal((R, V)) * 3).astype(np.float32)
    toks = g.integers(-2, V + 2, (G, hist)) if V > 8 else g.integers(-1, V + 1, (G, hist))
    toks[:, ::3] = toks[:, :1] if hist else toks[:, ::3]      # one token many times
    lens = g.integers(0, hist + 1, G)
    lens[0] = hist
    prompts = g.integers(0, hist + 1, G)
    ids = g.integers(-1, V + 1, (bg, nb))
    bias = (g.standard_normal((bg, nb)) * 2).astype(np.float32)
    if nb > 4:
        ids[:, 3] = ids[:, 1]
        ids[:, 4] = ids[:, 1]
    allowed = None if allow is None else g.random((R, V)) < allow
    if allowed is not None and R > 2:
        allowed[1] = False                    # nothing left
        allowed[2] = False
        allowed[2, V - 1] = True              # one token left
    pen = {}
    for name, lo, hi in (("rep", 0.5, 2.0), ("pres", -1.0, 1.0), ("freq", -0.5, 0.5)):
        pen[name] = g.uniform(lo, hi, R).astype(np.float32) if per_row else \
            np.full(R, np.float32(g.uniform(lo, hi)))
    T = lambda a: torch.from_numpy(a).to(cuda)
    kw, paths = {}, [[] for _ in range(R)]
    if nodes:
        par = [[-1] + [int(g.integers(0, i)) for i in range(1, nodes)] for _ in range(R // nodes)]
        draft = g.integers(-1, V + 1, (R // nodes, nodes))
        mask, _ = tb.tree_masks(torch.tensor(par, dtype=torch.int32, device=cuda))
        kw = dict(draft_tokens=T(draft), tree_mask=mask)
        for r in range(R):
            b, at = r // nodes, r % nodes
            while at >= 0:
                paths[r].append(int(draft[b, at]))
                at = par[b][at]
    if hist:
        kw.update(history=T(toks), history_len=T(lens), prompt_len=T(prompts))
    if nb:
        kw.update(bias_ids=T(ids), bias_values=T(bias))
    if allowed is not None:
        kw.update(allowed=T(pack(allowed)))
    one = (lambda a: T(a)) if per_row else (lambda a: float(a[0]))
    kw.update(repetition_penalty=one(pen["rep"]), presence_penalty=one(pen["pres"]),
              frequency_penalty=one(pen["freq"]))
    rows = np.arange(R)
    want, bound = reference(x, toks[rows // (R // G)].tolist(), lens[rows // (R // G)],
                            prompts[rows // (R // G)], pen["rep"].astype(float),
                            pen["pres"].astype(float), pen["freq"].astype(float),
                            ids[rows // (R // bg)].tolist(), bias[rows // (R // bg)].tolist(),
                            allowed, paths)
    dx = T(x)
    got = tb.process_logits(dx, **kw)
    assert torch.equal(dx, T(x)) and got.shape == dx.shape
    y = got.cpu().numpy()
    inf = np.isinf(want)
    assert np.array_equal(inf, np.isinf(y)) and (y[inf] < 0).all()
    assert (np.abs(y - want)[~inf] <= bound[~inf]).all()
    # in place, into another tensor, and each row's best token, that of the result
    out = torch.full_like(dx, 7.0)
    assert tb.process_logits(dx, **kw, out=out) is out and torch.equal(out, got)
    into = dx.clone()
    tb.process_logits(into, **kw, out=into)
    assert torch.equal(into, got)
    tok = tb.greedy_tokens(dx, **kw)
    assert tok.dtype == torch.int64 and tok.tolist() == best(y)


def test_greedy_ties_and_bad_values(cuda):
    """Ties go to the lowest index (-0 and 0 tie), NaN and -inf are never taken, +inf is;
    masked NaN and infinities give -inf."""
    print("case greedy_tokens ties, NaN, infinities", flush=True)
    V = 9000
    x = np.full((9, V), -1.0, np.float32)
    x[0, [8191, 4096, 70]] = 5.0
    x[1, :] = np.nan
    x[2, :] = -np.inf
    x[3, [10, 8000]] = [np.nan, 3.0]
    x[4, [100, 8500]] = [np.inf, np.inf]
    x[5, :] = np.nan
    x[5, 4500] = -3.4e38
    x[6, [5, 7]] = [-0.0, 0.0]
    x[6, [4, 9]] = [-1e-45, -2.0]
    x[7, [0, 8999]] = [np.nan, 0.5]
    want = [70, -1, -1, 8000, 100, 4500, 5, 8999, 0]
    T = lambda a: torch.from_numpy(a).to(cuda)
    assert tb.greedy_tokens(T(x)).tolist() == want == best(x)
    assert int(tb.greedy_tokens(T(x[3]))) == 8000           # one row without a batch
    assert tb.greedy_tokens(T(x).reshape(3, 3, V)).tolist() == np.reshape(want, (3, 3)).tolist()
    y = tb.process_logits(T(x), torch.tensor([10, 70, 100], device=cuda), repetition_penalty=2.0)
    w = x.copy()
    for t in (10, 70, 100):
        w[:, t] = np.where(w[:, t] > 0, w[:, t] / 2, w[:, t] * 2)
    assert np.array_equal(y.cpu().numpy(), w, equal_nan=True)
    allowed = np.zeros(V, bool)
    allowed[[3, 8191]] = True
    y = tb.process_logits(T(x), allowed=T(pack(allowed))).cpu().numpy()
    assert np.array_equal(y[:, [3, 8191]], x[:, [3, 8191]], equal_nan=True)
    assert (np.delete(y, [3, 8191], 1) == -np.inf).all()
    assert tb.greedy_tokens(T(x), allowed=T(pack(allowed))).tolist() == \
        [8191, -1, -1, 3, 3, -1, 3, 3, 3]


def test_history_forms(cuda):
    """A number for history_len and prompt_len, int32 tokens, a float16 row, host tensors."""
    print("case process_logits history forms", flush=True)
    V = 500
    g = np.random.default_rng(1)
    x = torch.from_numpy(g.standard_normal((4, V)).astype(np.float32)).to(cuda)
    h = torch.from_numpy(g.integers(0, V, 40)).to(cuda)
    kw = dict(repetition_penalty=1.5, presence_penalty=0.25, frequency_penalty=0.125)
    a = tb.process_logits(x, h[:25], prompt_len=10, **kw)
    assert torch.equal(tb.process_logits(x, h, history_len=25, prompt_len=10, **kw), a)
    assert torch.equal(tb.process_logits(x, h.int(), history_len=torch.tensor([25]),
                                         prompt_len=torch.tensor(10), **kw), a)
    assert torch.equal(tb.process_logits(x, h.expand(2, -1), history_len=25, prompt_len=10, **kw), a)
    assert torch.equal(tb.process_logits(x.cpu(), h.cpu(), history_len=25, prompt_len=10, **kw),
                       a.cpu())
    assert torch.equal(tb.process_logits(x, h, history_len=25, prompt_len=99, **kw),
                       tb.process_logits(x, h[:25], repetition_penalty=1.5, prompt_len=25))
    half = x.half()
    assert torch.equal(tb.process_logits(half, h, **kw), tb.process_logits(half.float(), h, **kw))
    assert tb.process_logits(x[:0], h, **kw).shape == (0, V)
    assert tb.greedy_tokens(x[:0], h).shape == (0,)


def test_alignment_and_many_biases(cuda):
    """Rows at every distance from a 16-byte boundary, input and output apart or alike, and
    more biases than one block lists, some tokens named many times."""
    print("case process_logits alignment, many biases", flush=True)
    V, R = 2053, 5
    g = np.random.default_rng(3)
    x = (g.standard_normal((R, V)) * 2).astype(np.float32)
    hist = g.integers(0, V, (1, 200))
    ids = g.integers(0, 300, (1, 4000))
    bias = g.standard_normal((1, 4000)).astype(np.float32) / 16
    ids[:, 600:] += 1000
    T = lambda a: torch.from_numpy(a).to(cuda)
    kw = dict(history=T(hist), repetition_penalty=1.5, presence_penalty=0.5, frequency_penalty=0.25,
              bias_ids=T(ids), bias_values=T(bias), allowed=T(pack(g.random((R, V)) < 0.8)))
    want = tb.process_logits(T(x), **kw)
    ref, bound = reference(x, np.repeat(hist, R, 0).tolist(), [200] * R, [0] * R, [1.5] * R,
                           [0.5] * R, [0.25] * R, np.repeat(ids, R, 0).tolist(),
                           np.repeat(bias, R, 0).tolist(), None, [[]] * R)
    y = want.cpu().numpy()
    fin = np.isfinite(y)
    assert fin.any() and (np.abs(y - ref)[fin] <= bound[fin]).all()
    buf = torch.empty(R * V + 8, device=cuda)
    obuf = torch.empty(R * V + 8, device=cuda)
    for a in range(4):
        xs = buf[a:a + R * V].view(R, V)
        for b in range(4):
            xs.copy_(T(x))
            out = obuf[b:b + R * V].view(R, V)
            assert torch.equal(tb.process_logits(xs, **kw, out=out), want)
        assert tb.greedy_tokens(xs, **kw).tolist() == best(y)
        tb.process_logits(xs, **kw, out=xs)
        assert torch.equal(xs, want)


@pytest.mark.parametrize("R,V,n,style", [
    (3, 700, 5000, "few"), (2, 2053, 1537, "one"), (2, 33333, 33333, "all"),
    (512, 5000, 900, "few"),        # blocks of 8192 tokens
    (1, 9000, 20000, "mixed"), (5, 40, 513, "few"),
])
def test_long_bias_lists(cuda, R, V, n, style):
    """More biases than a block lists, in the order of the list: every sum is the one of f32
    additions one after the other, bit by bit, with and without 16-byte vectors."""
    print(f"case process_logits long bias list R={R} V={V} n={n} {style}", flush=True)
    g = np.random.default_rng(V + n)
    if style == "all":
        ids = g.permutation(V)
    elif style == "one":
        ids = np.full(n, 1234)
    else:
        ids = g.integers(-3, min(V, 300) + 3, n)
        if style == "mixed":
            ids[n // 2:] = g.integers(0, V, n - n // 2)
            ids[::7] = 5
    bias = g.standard_normal(n).astype(np.float32)
    x = g.standard_normal((R, V)).astype(np.float32)
    total, named = np.zeros(V, np.float32), np.zeros(V, bool)
    for t, b in zip(ids, bias):
        if 0 <= t < V:
            total[t] = total[t] + b if named[t] else b
            named[t] = True
    allowed = g.random(V) < 0.8
    want = np.where(allowed, np.where(named, x + total, x), -np.inf).astype(np.float32)
    T = lambda a: torch.from_numpy(a).to(cuda)
    kw = dict(bias_ids=T(ids), bias_values=T(bias), allowed=T(pack(allowed)))
    assert np.array_equal(tb.process_logits(T(x), **kw).cpu().numpy(), want)
    out = torch.empty(R * V + 1, device=cuda)[1:].view(R, V)
    assert np.array_equal(tb.process_logits(T(x), **kw, out=out).cpu().numpy(), want)
    assert tb.greedy_tokens(T(x), **kw).tolist() == best(want)
    own = dict(bias_ids=T(ids).repeat(R, 1), bias_values=T(bias).repeat(R, 1),
               allowed=T(pack(allowed)))
    assert np.array_equal(tb.process_logits(T(x), **own).cpu().numpy(), want)


def test_long_bias_lists_take_time_in_their_length(cuda):
    """Ten times as many biases for as many tokens take no more than ten times as long (twice,
    measured; 50 times where each entry looked through the whole list)."""
    print("case process_logits long bias lists, time", flush=True)
    g = np.random.default_rng(9)
    x = torch.zeros(1, 2053, device=cuda)

    def time(n):
        kw = dict(bias_ids=torch.from_numpy(g.integers(0, 300, n)).to(cuda),
                  bias_values=torch.zeros(n, device=cuda))
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        least = 1e9
        for _ in range(5):
            a.record()
            for _ in range(20):
                tb.process_logits(x, **kw)
            b.record()
            torch.cuda.synchronize()
            least = min(least, a.elapsed_time(b))
        return least

    few, many = time(400), time(4000)
    print(f"400 biases {few * 50:.1f} us, 4000 {many * 50:.1f} us", flush=True)
    assert many <= 10 * few
