"""verify_tree, accept_tree and tree_step of the GPU decoder against the oracle's
step-by-step decoder: every node's logits equal the oracle's after stepping the
node's own path behind the prefix (within 2e-4, as verify_tokens is held), and the
cache that acceptance leaves drives the following steps like the oracle's."""
import numpy as np
import pytest
import torch

from oracle import oracle as O
from torchburn_amd import synth
from torchburn_amd.decoder import decoder_from_weights
import torchburn_amd as tb

pytestmark = pytest.mark.gpu

V = 1000


def rel(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return float(np.abs(a - b).max() / max(np.abs(b).max(), 1e-30))


def make(wk, lk, max_seq=160, seed=71, **kw):
    cfg = dict(num_layers=2, hidden=256, intermediate=512, num_heads=4, num_kv_heads=2,
               head_dim=64, vocab=V, eps=1e-6, rope_theta=1e6, qkv_bias=True)
    cfg.update(kw)
    w = synth.decoder_weights(cfg, seed, wk, lk, 32)
    ocfg = dict(num_layers=cfg["num_layers"], hidden=cfg["hidden"],
                intermediate=cfg["intermediate"], num_heads=cfg["num_heads"],
                num_kv_heads=cfg["num_kv_heads"], head_dim=cfg["head_dim"], vocab=V,
                group_size=32, max_seq=max_seq, rope_theta=cfg["rope_theta"], eps=cfg["eps"],
                wkind=wk, lmkind=lk)
    return O.Decoder(w, ocfg), decoder_from_weights(w, cfg, group_size=32, max_seq_len=max_seq), cfg


def prefix(ref, dec, g, n):
    toks = [int(t) for t in g.integers(0, V, n)]
    for i, t in enumerate(toks):
        lo = ref.step(t, i)
    dec.prefill_tokens(toks, 0)
    return toks, lo


def branch(par, i):
    p = []
    while i >= 0:
        p.append(i)
        i = par[i]
    return p[::-1]


@pytest.mark.parametrize("wk,lk,n,kw", [
    (4, 4, 1, {}), (4, 4, 7, {}), (4, 32, 12, {}), (8, 8, 9, {}), (4, 4, 40, {}),
    (4, 4, 21, dict(num_heads=8, num_kv_heads=2, head_dim=128, hidden=1024, qkv_bias=False))])
def test_verify_tree(cuda, wk, lk, n, kw):
    print(f"case verify_tree wk={wk} lk={lk} n={n} {kw}", flush=True)
    ref, dec, _ = make(wk, lk, **kw)
    g = np.random.default_rng(n + wk)
    prefix(ref, dec, g, 30)
    par = [-1] + [int(g.integers(0, i)) for i in range(1, n)]
    toks = [int(t) for t in g.integers(0, V, n)]
    rows = dec.verify_tree(30, toks, par).numpy()
    assert rows.shape == (n, V) and dec.kv_len() == 30 + n
    worst = 0.0
    for i in range(n):
        for depth, j in enumerate(branch(par, i)):
            lo = ref.step(toks[j], 30 + depth)
        worst = max(worst, rel(rows[i], lo))
    print(f"verify_tree rel err {worst:.3g}", flush=True)
    assert worst < 2e-4
    # any accepted path continues as the oracle's steps along it
    want = branch(par, n - 1)
    nxt = [V - 1] * n
    for a, b in zip(want, want[1:]):
        nxt[a] = toks[b]
    lowest = [0]      # siblings with the same token: the walk takes the lowest
    while True:
        kids = [j for j in range(lowest[-1] + 1, n)
                if par[j] == lowest[-1] and toks[j] == nxt[lowest[-1]]]
        if not kids:
            break
        lowest.append(kids[0])
    path, tok = dec.accept_tree(30, toks, par, nxt)
    assert path == lowest and tok == nxt[lowest[-1]] and dec.kv_len() == 30 + len(path)
    for depth, j in enumerate(path):
        ref.step(toks[j], 30 + depth)
    pos = 30 + len(path)
    for t in (tok, 5, 17):
        lg, am = dec._step(t, pos, True)
        lo = ref.step(t, pos)
        assert rel(lg, lo) < 2e-4 and am == O.argmax(lo)
        pos += 1
    ref.close()
    dec.close()


def best(lo, hist, path, rep, pres, freq, allowed):
    y = lo.astype(np.float64).copy()
    for t in set(hist) | set(path):
        y[t] = y[t] / rep if y[t] > 0 else y[t] * rep
    c = np.bincount(np.array(list(hist) + list(path), dtype=np.int64), minlength=V)
    y -= freq * c + pres * (c > 0)
    if allowed is not None:
        y[~allowed] = -np.inf
    return int(np.argmax(y))


@pytest.mark.parametrize("wk,rep,freq,mask", [(4, 1.0, 0.0, False), (4, 1.25, 0.0, False),
                                             (8, 1.25, 0.0, True), (4, 1.0, 0.001, True)])
def test_tree_steps_generate_the_oracles_tokens(cuda, wk, rep, freq, mask):
    """Greedy speculative decoding with trees: whatever is drafted, the tokens are those of
    greedy decoding token by token with the same penalties.  Drafts: the right token on a
    random one of a node's children, wrong ones elsewhere."""
    print(f"case tree_step generation wk={wk} rep={rep} freq={freq} mask={mask}", flush=True)
    ref, dec, _ = make(wk, 4, seed=80 + wk)
    g = np.random.default_rng(7)
    hist, lo = prefix(ref, dec, g, 12)
    allowed = g.random(V) < 0.5 if mask else None
    words = None
    if mask:
        bits = np.zeros(((V + 31) // 32) * 32, bool)
        bits[:V] = allowed
        words = np.packbits(bits.reshape(-1, 32), axis=-1, bitorder="little").view(np.uint32) \
            .reshape(-1).astype(np.int32, casting="unsafe")
    # the oracle's tokens
    want, h = [], list(hist)
    for i in range(24):
        t = best(lo, h, [], rep, 0.0, freq, allowed)
        want.append(t)
        h.append(t)
        lo = ref.step(t, 12 + i)
    got, pos, tok, counts = [want[0]], 12, want[0], []
    while len(got) < 20:
        par, toks = [-1], [tok]
        at = 0
        for depth in range(int(g.integers(0, 4))):      # a right chain among wrong siblings
            kids = [int(t) for t in g.integers(0, V, 3)]
            kids[int(g.integers(0, 3))] = want[len(got) + depth]
            nxt = len(par) + kids.index(want[len(got) + depth])
            par += [at] * 3
            toks += kids
            at = nxt
        kw = dict(history=hist + got[:-1], repetition_penalty=rep, frequency_penalty=freq)
        if mask:
            kw["allowed"] = np.tile(words, (len(par), 1))
        path, tok = dec.tree_step(pos, toks, par, **kw)
        counts.append(len(path))
        got += [toks[i] for i in path[1:]] + [tok]
        pos += len(path)
        assert dec.kv_len() == pos
        at = dec.get_logits()      # the row that tok came from
        assert best(np.array(at, np.float32), hist + got[:-1], [], rep, 0.0, freq, allowed) == tok
    print(f"tokens kept a step: {counts}", flush=True)
    assert got[:20] == want[:20] and max(counts) > 1
    ref.close()
    dec.close()


def test_tree_refusals(cuda):
    print("case tree refusals", flush=True)
    ref, dec, _ = make(4, 4, max_seq=20)
    for toks, par in (([1, 2], [-1, 1]), ([1, 2], [0, 0]), ([1, 2], [-1, -2]), ([1, V], [-1, 0]),
                      ([1, -1], [-1, 0]), ([], []), ([1, 2], [-1])):
        with pytest.raises(ValueError):
            dec.verify_tree(0, toks, par)
        with pytest.raises(ValueError):
            dec.accept_tree(0, toks, par, [0] * len(toks))
        with pytest.raises(ValueError):
            dec.tree_step(0, toks, par)
    for start in (-1, 19, 20, 2 ** 63 - 1):
        with pytest.raises(ValueError):
            dec.verify_tree(start, [1, 2], [-1, 0])
        with pytest.raises(ValueError):
            dec.accept_tree(start, [1, 2], [-1, 0], [0, 0])
        with pytest.raises(ValueError):
            dec.tree_step(start, [1, 2], [-1, 0])
    with pytest.raises(ValueError):
        dec.accept_tree(0, [1, 2], [-1, 0], [0])
    with pytest.raises(ValueError):
        dec.tree_step(0, [1], [-1], repetition_penalty=0.0)
    with pytest.raises(tb.UnsupportedOpError):
        dec.tree_step(0, [1], [-1], allowed=np.zeros(5, np.int32))
    with pytest.raises(tb.UnsupportedOpError):
        dec.tree_step(0, [1], [-1], allowed=np.zeros((V + 31) // 32, np.int64))
    dec.set_attention_cap(10)
    with pytest.raises(tb.UnsupportedOpError, match="cap"):
        dec.verify_tree(9, [1, 2], [-1, 0])
    dec.set_attention_cap(0)
    assert dec.verify_tree(18, [1, 2], [-1, 0]).shape == (2, V)
    # two roots: node 1 starts a second sequence behind the same prefix
    rows = dec.verify_tree(0, [3, 4], [-1, -1]).numpy()
    for i, t in enumerate((3, 4)):
        assert rel(rows[i], ref.step(t, 0)) < 2e-4
    # nothing allowed: no token
    none = np.zeros((2, (V + 31) // 32), np.int32)
    assert dec.tree_step(0, [3, 4], [-1, 0], allowed=none) == ([0], -1)
    ref.close()
    dec.close()


def test_accept_tree_takes_the_tree_that_the_cache_holds(cuda):
    """A path is kept once, and only of the tree verified last at that position whose rows
    nothing has been written to since: a second acceptance would move rows that have moved
    already.  A refused call leaves the cache as it was."""
    print("case accept_tree of trees that the cache does not hold", flush=True)
    ref, dec, _ = make(4, 4)
    g = np.random.default_rng(5)
    prefix(ref, dec, g, 10)
    toks, par, nxt = [7, 8, 9, 10, 11], [-1, 0, 0, 2, 3], [9, 0, 10, 11, 3]

    def refused(start=10, t=toks, p=par):
        before = dec.kv_len()
        with pytest.raises(ValueError, match="does not hold"):
            dec.accept_tree(start, t, p, nxt)
        assert dec.kv_len() == before

    refused()                                     # no tree yet
    dec.verify_tree(10, toks, par)
    refused(9)
    refused(10, [7, 8, 9, 10, 12])
    refused(10, toks, [-1, 0, 0, 2, 2])
    with pytest.raises(ValueError, match="does not hold"):
        dec.accept_tree(10, toks[:4], par[:4], nxt[:4])
    assert dec.accept_tree(10, toks, par, nxt) == ([0, 2, 3, 4], 3)
    refused()                                     # accepted already
    for depth, t in enumerate((7, 9, 10, 11)):
        ref.step(t, 10 + depth)
    for i, t in enumerate((3, 5, 17)):            # the refusals moved nothing
        lg, _ = dec._step(t, 14 + i, True)
        assert rel(lg, ref.step(t, 14 + i)) < 2e-4
    dec.tree_step(17, toks, par)
    refused(17)                                   # tree_step has kept its path
    kv = [torch.zeros(2, 18, 64)] * 2
    for write in (lambda: dec._step(1, 21, False), lambda: dec.prefill_tokens([1] * 5, 15),
                  lambda: dec.verify_tokens(21, [1, 2]), lambda: dec.verify_tree(20, [1], [-1]),
                  lambda: dec.generate_loop(1, 19, 2, temperature=0.0),
                  lambda: dec.generate_loop(1, 21, 2, top_k=5), lambda: dec.reset_kv_cache(),
                  lambda: dec.time_greedy(1, 18, 1),
                  lambda: dec.copy_kv_cache_from_tensors(kv, kv, 18),
                  lambda: dec.tree_step(16, [1, 2], [-1, 0])):
        dec.verify_tree(17, toks, par)
        write()
        refused(17)
    # rows before and behind the nodes are not theirs
    dec.verify_tree(17, toks, par)
    dec._step(1, 16, False)
    dec._step(1, 22, False)
    dec.prefill_tokens([1, 2, 3, 4], 13)
    dec.copy_kv_cache_from_tensors(kv, kv, 17)
    assert dec.accept_tree(17, toks, par, nxt) == ([0, 2, 3, 4], 3)
    ref.close()
    dec.close()


def test_verify_tree_of_large_layers_is_no_less_exact(cuda):
    """9 nodes through layers of more than 2^24 weights, as a tree and as the steps that it
    stands for: over all nodes, the tree's error against float64 is not the larger one."""
    H, I, hd, n = 2048, 8320, 128, 9
    cfg = dict(num_layers=1, hidden=H, intermediate=I, num_heads=16, num_kv_heads=4, head_dim=hd,
               vocab=1024, eps=1e-6, rope_theta=1e6, qkv_bias=False)
    w = synth.decoder_weights(cfg, 97, 4, 32, 32)
    y = w["layers"][0]
    y["post_norm"][::128] = 12.0      # large channels, and outputs of about unit size
    for t in ("qkv_s", "o_s", "gate_s", "up_s", "down_s"):
        y[t] *= 0.1
    dec = decoder_from_weights(w, cfg, group_size=32, max_seq_len=32)
    toks = [int(t) for t in np.random.default_rng(97).integers(0, cfg["vocab"], n)]
    par = [-1, 0, 0, 1, 1, 3, 2, 5, 7]
    tree = dec.verify_tree(0, toks, par).numpy()
    steps = np.empty_like(tree)
    for i in range(n):
        for depth, j in enumerate(branch(par, i)):
            steps[i], _ = dec._step(toks[j], depth, True)
    dec.close()

    f = lambda a: np.asarray(a, np.float64)
    deq = lambda p, s: (np.stack((p & 15, p >> 4), -1).reshape(p.shape[0], -1) - 8.0) * \
        np.repeat(f(s), 32, 1)
    lin = lambda a, t: a @ deq(y[t + "_w"], y[t + "_s"]).T
    rms = lambda v, g: v / np.sqrt((v * v).mean(1, keepdims=True) + cfg["eps"]) * f(g)
    x = f(w["embed"])[toks]
    depth = np.array([len(branch(par, i)) - 1 for i in range(n)])
    ang = depth[:, None] / cfg["rope_theta"] ** (np.arange(0, hd, 2) / hd)
    cos, sin = (np.tile(fn(ang), (1, 2))[:, None] for fn in (np.cos, np.sin))
    turn = lambda v: v * cos + np.concatenate((-v[..., hd // 2:], v[..., :hd // 2]), -1) * sin
    q, k, v = (a.reshape(n, -1, hd)
               for a in np.split(lin(rms(x, y["in_norm"]), "qkv"), (H, H + 4 * hd), 1))
    q, k, v = turn(q), np.repeat(turn(k), 4, 1), np.repeat(v, 4, 1)
    see = np.array([[j in branch(par, i) for j in range(n)] for i in range(n)])
    s = np.einsum("ihd,jhd->hij", q, k) / np.sqrt(hd) + np.where(see, 0.0, -np.inf)
    p = np.exp(s - s.max(-1, keepdims=True))
    a = np.einsum("hij,jhd->ihd", p / p.sum(-1, keepdims=True), v).reshape(n, -1)
    x = x + lin(a, "o")
    xn = rms(x, y["post_norm"])
    g, u = lin(xn, "gate"), lin(xn, "up")
    x = x + lin(g / (1 + np.exp(-g)) * u, "down")
    want = rms(x, w["final_norm"]) @ f(w["lm_head_w"]).T
    err = [np.linalg.norm(f(t) - want) / np.linalg.norm(want) for t in (tree, steps)]
    print(f"case verify_tree errors: tree {err[0]:.2e}, steps {err[1]:.2e}", flush=True)
    assert err[0] <= 1.02 * err[1]
