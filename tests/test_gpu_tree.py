"""Draft-tree operators against their definitions in 64 bits.

tree_attention's bound, row by row.  With u = 2^-24, a score is a sum of D
products whose factors are held to 2^-22 (two 11-bit limbs, their smallest
product dropped): ds = scale sum|q k| (3 2^-22 + 4 sqrt(D) u) + 8 u |s|, the
rounding of a D-term sum taken as a random walk with a factor of 4 to spare.  A
softmax weight is then off by a share of 2 ds + 8 u (both the weight and the sum
it is divided by), the weighted sum over T keys by 6 2^-22 + 4 sqrt(T) u more, so
|error| <= sum_p w_p |v_p| (2 ds + 8 u + 6 2^-22 + 4 sqrt(T) u).

Masks, paths, tokens and moved rows have to be equal.
"""
import numpy as np
import pytest
import torch

import torchburn_amd as tb

pytestmark = pytest.mark.gpu


def tree(g, n, used=None, style="mixed"):
    """Parents of a random tree, padded with invalid entries from `used` on."""
    used = n if used is None else used
    par = []
    for i in range(n):
        if i >= used:
            par.append(int(g.choice([-2, -7, i, i + 3])))
        elif i == 0 or (style == "forest" and g.random() < 0.2):
            par.append(-1)
        else:
            par.append(i - 1 if style == "chain" else int(g.integers(0, i)))
    return par


def ancestors(par):
    n = len(par)
    a, depth = np.zeros((n, n), bool), np.zeros(n, np.int32)
    for i, p in enumerate(par):
        if p == -1:
            a[i, i] = True
        elif 0 <= p < i and a[p, p]:
            a[i] = a[p]
            a[i, i] = True
            depth[i] = depth[p] + 1
    return a, depth


def words(bits):
    n = bits.shape[-1]
    w = np.zeros((*bits.shape[:-1], (n + 31) // 32 * 32), bool)
    w[..., :n] = bits
    return np.packbits(w.reshape(*bits.shape[:-1], -1, 32), axis=-1, bitorder="little") \
        .view(np.uint32)[..., 0].astype(np.int32, casting="unsafe").reshape(*bits.shape[:-1], -1)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 64, 65, 100, 511, 1024])
@pytest.mark.parametrize("style", ["mixed", "chain", "forest"])
def test_masks(cuda, n, style):
    print(f"case tree_masks n={n} {style}", flush=True)
    g = np.random.default_rng(n)
    par = [tree(g, n, u, style) for u in (n, max(1, n - 3), 1, 0)]
    # an unreachable subtree: children of a padding node
    bad = tree(g, n, None, style)
    bad[n // 2] = -3
    par.append(bad)
    mask, depth = tb.tree_masks(torch.tensor(par, dtype=torch.int32, device=cuda))
    want = [ancestors(p) for p in par]
    assert np.array_equal(mask.cpu().numpy(), words(np.stack([a for a, _ in want])))
    assert np.array_equal(depth.cpu().numpy(), np.stack([d for _, d in want]))
    one, d1 = tb.tree_masks(torch.tensor(par[0], device=cuda))    # int64, one tree
    assert torch.equal(one, mask[0]) and torch.equal(d1, depth[0])


def reference(q, k, v, bits, lens, scale):
    """(out, bound) in float64 from numpy arrays: q [B, N, H, D], k / v [B, KVH, S, D],
    bits [B, N, N] truth values."""
    B, N, H, D = q.shape
    G, S = H // k.shape[1], k.shape[2]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    u = 2.0 ** -24
    for b in range(B):
        ln = min(max(lens[b], 0), S)
        for i in range(N):
            if not bits[b, i].any():
                continue
            at = np.concatenate((np.arange(ln), ln + np.flatnonzero(bits[b, i])))
            at = at[at < S]
            if not len(at):
                continue
            for h in range(H):
                kk, vv = (c[b, h // G, at].astype(np.float64) for c in (k, v))
                x = q[b, i, h].astype(np.float64)
                s = kk @ x * scale
                e = np.exp(s - s.max())
                w = e / e.sum()
                out[b, i, h] = w @ vv
                ds = abs(scale) * (np.abs(kk) @ np.abs(x)).max() * \
                    (3 * 2.0 ** -22 + 4 * D ** 0.5 * u) + 8 * u * np.abs(s).max()
                bound[b, i, h] = w @ np.abs(vv) * (2 * ds + 8 * u + 6 * 2.0 ** -22 +
                                                   4 * len(at) ** 0.5 * u)
    return out, bound


def inputs(seed, B, N, H, KVH, D, S, used=None, style="mixed", kscale=1.0, vscale=1.0):
    g = np.random.default_rng(seed)
    q = g.standard_normal((B, N, H, D)).astype(np.float32) * 2
    k = (g.standard_normal((B, KVH, S, D)) * kscale).astype(np.float32)
    v = (g.standard_normal((B, KVH, S, D)) * vscale).astype(np.float32)
    par = [tree(g, N, used[b] if used else None, style) for b in range(B)]
    return q, k, v, np.stack([ancestors(p)[0] for p in par])


def check(got, want, bound):
    got = got.cpu().numpy().astype(np.float64)
    assert np.isfinite(got).all()
    err = np.abs(got - want)
    worst = float((err / np.maximum(bound, 1e-300))[bound > 0].max()) if (bound > 0).any() else 0.0
    print(f"worst error {worst:.3g} of the bound", flush=True)
    assert (err <= bound).all(), worst


CASES = [
    # B, N, H, KVH, D, lens, S
    (1, 1, 1, 1, 32, [0], 1),              # one node, no prefix, a full cache
    (1, 1, 14, 2, 64, [1], 8),
    (1, 5, 14, 2, 64, [61], 128),
    (1, 7, 8, 8, 128, [31], 64),           # one head a group
    (1, 16, 8, 2, 128, [32], 48),          # the prefix ends with a tile
    (1, 17, 8, 2, 128, [33], 50),
    (1, 33, 7, 1, 64, [300], 333),
    (1, 64, 8, 2, 128, [1000], 1100),
    (1, 100, 4, 1, 96, [257], 400),
    (1, 3, 5, 5, 160, [129], 200),
    (1, 40, 8, 1, 192, [70], 128),
    (1, 20, 6, 2, 224, [95], 128),
    (1, 65, 4, 2, 256, [511], 600),
    (2, 9, 4, 2, 32, [0, 77], 100),
    (3, 21, 28, 4, 128, [500, 3, 0], 640),
    (5, 4, 4, 2, 64, [10, 0, 63, 64, 65], 80),
    (1, 256, 8, 8, 64, [40], 300),
    (1, 130, 16, 2, 128, [2500], 2700),    # more rows than one tile, a long prefix
    (1, 2, 32, 8, 128, [9000], 9100),
    (1, 50, 8, 2, 64, [1500], 1600),       # two and four row tiles
    (1, 50, 16, 2, 64, [1500], 1600),
    (1, 30, 8, 2, 128, [700], 800),
    (1, 70, 16, 4, 128, [700], 800),
    (2, 30, 8, 2, 256, [700, 90], 800),
    (1, 17, 16, 2, 160, [300], 400),
]


@pytest.mark.parametrize("B,N,H,KVH,D,lens,S", CASES)
def test_attention(cuda, B, N, H, KVH, D, lens, S):
    print(f"case tree_attention B={B} N={N} H={H}/{KVH} D={D} lens={lens} S={S}", flush=True)
    used = [max(0, N - 2 * b) for b in range(B)]
    q, k, v, bits = inputs(N * D + S, B, N, H, KVH, D, S, used)
    T = lambda a: torch.from_numpy(a).to(cuda)
    out = tb.tree_attention(T(q), T(k), T(v), T(words(bits)),
                            torch.tensor(lens, dtype=torch.int32, device=cuda))
    want, bound = reference(q, k, v, bits, lens, D ** -0.5)
    check(out, want, bound)
    if B == 1:      # the forms without a batch, with a number, with a given scale
        a = [T(q[0]), T(k[0]), T(v[0]), T(words(bits[0]))]
        assert torch.equal(tb.tree_attention(*a, lens[0]), out[0])
        assert torch.equal(tb.tree_attention(*a, torch.tensor(lens, device=cuda)), out[0])
        assert torch.equal(tb.tree_attention(*a, lens[0], scale=D ** -0.5), out[0])


@pytest.mark.parametrize("N,H,KVH,D,lens,S", [
    (70, 16, 2, 64, [1000], 131072),
    (40, 16, 4, 64, [0, 2100, 63, 1, 9], 13120),
    (19, 16, 2, 128, [700], 65600),
    (70, 8, 2, 96, [31, 129], 32800),
    # blocks of eight waves (the ones above are of four: too many of 256 rows would be empty)
    (28, 16, 2, 64, [1000], 131072),
    (60, 16, 4, 64, [0, 2100, 63, 1, 9], 13120),
    (25, 16, 2, 128, [700], 65600),        # 200 rows: some waves have few or none
    (120, 8, 2, 96, [31, 129], 32800),     # two tiles of rows
])
def test_attention_of_many_rows_over_a_large_cache(cuda, N, H, KVH, D, lens, S):
    """Blocks of four and of eight waves.  The first K and V rows of every other 4 positions are larger,
    so that the parts of a tile have scales of their own; one node has infinities."""
    B = len(lens)
    print(f"case tree_attention large cache N={N} H={H}/{KVH} D={D} lens={lens} S={S}", flush=True)
    q, k, v, bits = inputs(N + D, B, N, H, KVH, D, max(lens) + N, [N - 3] * B)
    at = np.arange(k.shape[2])
    k[:, :, at % 8 < 4] *= 1.5
    v[:, :, at % 8 >= 4] *= 300.0
    want, bound = reference(q, k, v, bits, lens, D ** -0.5)
    T = lambda a: torch.from_numpy(a).to(cuda)
    kc, vc = (torch.full((B, KVH, S, D), float("nan"), device=cuda) for _ in range(2))
    kc[:, :, :k.shape[2]], vc[:, :, :k.shape[2]] = T(k), T(v)
    a = (T(q), kc, vc, T(words(bits)), torch.tensor(lens, device=cuda))
    check(tb.tree_attention(*a), want, bound)
    node = 2
    for b, ln in enumerate(lens):
        kc[b, :, ln + node] = float("inf")
        vc[b, :, ln + node] = float("nan")
    got = tb.tree_attention(*a).cpu().numpy()
    on = bits[:, :, node]
    assert np.isnan(got[on]).all() and np.isfinite(got[~on]).all()
    assert (np.abs(got - want)[~on] <= bound[~on]).all()


@pytest.mark.parametrize("D,N,kv", [(64, 6, 40), (128, 70, 300), (96, 33, 1000)])
def test_attention_unseen_positions(cuda, D, N, kv):
    """NaN, infinities and the largest values in positions that a row does not see: behind
    the tree, in nodes off its path, and (a padding row) in the prefix."""
    print(f"case tree_attention unseen D={D} N={N} kv={kv}", flush=True)
    H, KVH, S = 8, 2, kv + N + 50
    q, k, v, bits = inputs(D + N, 1, N, H, KVH, D, S, [N - 2])
    want, bound = reference(q, k, v, bits, [kv], D ** -0.5)
    bad = [np.nan, np.inf, -np.inf, 3.4e38, -3.4e38]
    for i, j in enumerate(list(range(kv + N, S)) + [kv + N - 1, kv + N - 2]):
        k[:, :, j], v[:, :, j] = bad[i % 5], bad[(i + 1) % 5]
    T = lambda a: torch.from_numpy(a).to(cuda)
    mask = T(words(bits))
    check(tb.tree_attention(T(q), T(k), T(v), mask, kv), want, bound)
    # a node's own values are bad: its descendants see them, the others do not
    node = 1
    for x, y in ((np.nan, 1.0), (1.0, np.inf), (np.inf, 1.0), (1.0, np.nan)):
        k2, v2 = k.copy(), v.copy()
        k2[:, :, kv + node] *= x
        v2[:, :, kv + node] *= y
        got = tb.tree_attention(T(q), T(k2), T(v2), mask, kv).cpu().numpy()
        off = ~bits[0, :, node]
        assert off.any() and np.isfinite(got[0, off]).all()
        assert (np.abs(got[0, off] - want[0, off]) <= bound[0, off]).all()
        on = np.abs(got[0, bits[0, :, node]])
        if np.isnan(x) or np.isnan(y):
            assert np.isnan(on).all(-1).all()
        elif np.isinf(y):
            assert not np.isfinite(on).any()


@pytest.mark.parametrize("D,N,kv,S", [(64, 6, 40, 46), (128, 7, 0, 7), (128, 25, 90, 115),
                                      (96, 60, 200, 260), (256, 33, 65, 98), (64, 80, 30, 131072), (64, 60, 30, 131072)])
@pytest.mark.parametrize("big", [1e6, 3e38])
def test_attention_large_values_beside_the_path(cuda, D, N, kv, S, big):
    """Nodes whose K and V are very large cost the rows that do not see them no bits, and the
    rows that see one get its V."""
    print(f"case tree_attention large nodes D={D} N={N} kv={kv} big={big}", flush=True)
    H, KVH = 8, 2
    q, k, v, bits = inputs(D + N, 1, N, H, KVH, D, kv + N, [N - 1])
    nodes = [2, N - 1] if N < 10 else [2, 5, N // 2, N - 1]   # the last one is padding
    small = v.copy()
    for j in nodes:
        k[:, :, kv + j] = np.clip(k[:, :, kv + j], -1, 1) * np.float32(big)
        v[:, :, kv + j] = np.clip(v[:, :, kv + j], -1, 1) * np.float32(big)
    v[:, :, kv + N // 3] = 0.0       # scales of their own in both directions
    v[:, :, kv + N // 4] *= 1e-30
    want, bound = reference(q, k, v, bits, [kv], D ** -0.5)
    T = lambda a: torch.from_numpy(a).to(cuda)
    kc, vc = (torch.zeros((1, KVH, S, D), device=cuda) for _ in range(2))
    kc[:, :, :kv + N], vc[:, :, :kv + N] = T(k), T(v)
    ln = torch.tensor([kv], device=cuda)
    got = tb.tree_attention(T(q), kc, vc, T(words(bits)), ln).cpu().numpy()
    on = bits[0][:, nodes].any(-1)
    assert on.any() and not on.all()
    assert (np.abs(got - want)[0, ~on] <= bound[0, ~on]).all()
    # only V: the scores of the rows that see it are ordinary
    k[:, :, [kv + j for j in nodes]] = small[:, :, [kv + j for j in nodes]]
    kc[:, :, :kv + N] = T(k)
    want, bound = reference(q, k, v, bits, [kv], D ** -0.5)
    got = tb.tree_attention(T(q), kc, vc, T(words(bits)), ln)
    # 2^-32 of the largest V seen, for every position
    top = np.where(on, np.float64(big), 0.0)[None, :, None, None] * (kv + N) * 2.0 ** -32
    check(got, want, bound + top)


def test_attention_weights_of_zero_values(cuda):
    """Positions whose V is zero count in the sum, however large other positions' V is."""
    print("case tree_attention zero values", flush=True)
    for N, H, D in ((2, 4, 128), (40, 8, 64), (60, 16, 128)):
        KVH, kv, S = 2, 4000, 4100
        q, k, v, bits = inputs(31, 1, N, H, KVH, D, S)
        v[:, :, :kv] = 0.0
        v[:, :, 3900:3904] = 1e7
        want, bound = reference(q, k, v, bits, [kv], D ** -0.5)
        T = lambda a: torch.from_numpy(a).to(cuda)
        got = tb.tree_attention(T(q), T(k), T(v), T(words(bits)), kv)
        check(got, want, bound + 1e7 * 2.0 ** -32 * (kv + N))


@pytest.mark.parametrize("kscale,vscale", [(1e-20, 1e-30), (1e18, 1e30), (1e-38, 1e-38), (30.0, 1.0)])
def test_attention_ranges(cuda, kscale, vscale):
    print(f"case tree_attention ranges k={kscale} v={vscale}", flush=True)
    N, H, KVH, D, kv, S = 19, 8, 2, 128, 200, 230
    q, k, v, bits = inputs(5, 1, N, H, KVH, D, S, kscale=kscale, vscale=vscale)
    scale = D ** -0.5 / (kscale if kscale > 1e3 or kscale < 1 else 1.0)
    if kscale < 1e-30:
        scale = 1.0
    want, bound = reference(q, k, v, bits, [kv], scale)
    # results of 1e-38 have spacing 2^-149: half of it for every key's product
    tiny = 2.0 ** -149 * (kv + N) if vscale < 1e-30 else 0.0
    T = lambda a: torch.from_numpy(a).to(cuda)
    check(tb.tree_attention(T(q), T(k), T(v), T(words(bits)), kv, scale=scale), want, bound + tiny)


def test_attention_mixed_magnitudes(cuda):
    """Positions of very different magnitude side by side: none may cost another its bits."""
    print("case tree_attention mixed magnitudes", flush=True)
    N, H, KVH, D, kv, S = 9, 4, 1, 64, 150, 170
    q, k, v, bits = inputs(6, 1, N, H, KVH, D, S)
    g = np.random.default_rng(8)
    k *= 2.0 ** g.integers(-6, 1, (1, KVH, S, 1)).astype(np.float32)
    v *= 2.0 ** g.integers(-12, 1, (1, KVH, S, 1)).astype(np.float32)
    want, bound = reference(q, k, v, bits, [kv], D ** -0.5)
    T = lambda a: torch.from_numpy(a).to(cuda)
    check(tb.tree_attention(T(q), T(k), T(v), T(words(bits)), kv), want, bound)


def test_attention_any_mask_and_strides(cuda):
    """A mask that is no tree's (later nodes, rows without bits), one mask for the batch,
    caches as [batch, position, head, dim] and as halves of one buffer, q as a view."""
    print("case tree_attention any mask, strides", flush=True)
    B, N, H, KVH, D, S = 3, 37, 12, 4, 64, 260
    q, k, v, _ = inputs(3, B, N, H, KVH, D, S)
    g = np.random.default_rng(4)
    bits = g.random((N, N)) < 0.1
    bits[5] = bits[36] = False
    lens = [0, 100, 222]
    want, bound = reference(q, k, v, np.broadcast_to(bits, (B, N, N)), lens, D ** -0.5)
    T = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)
    ln = torch.tensor(lens, device=cuda)
    plain = tb.tree_attention(T(q), T(k), T(v), T(words(bits)), ln)
    check(plain, want, bound)
    assert (plain[:, 5] == 0).all() and (plain[:, 36] == 0).all()
    both = torch.empty((B, S, 2, KVH, D), device=cuda)
    both[:, :, 0], both[:, :, 1] = T(k).transpose(1, 2), T(v).transpose(1, 2)
    kc, vc = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    qv = T(q).permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    three = T(words(bits)).expand(B, -1, -1)
    assert torch.equal(tb.tree_attention(qv, kc, vc, three, ln), plain)
    assert torch.equal(tb.tree_attention(T(q).double(), T(k), T(v), T(words(bits)), ln), plain)
    # rows that are not 16-byte aligned are copied
    odd = torch.empty((B, KVH, S, D + 1), device=cuda)
    odd[..., 1:] = T(k)
    assert torch.equal(tb.tree_attention(T(q), odd[..., 1:], T(v), T(words(bits)), ln), plain)
    host = tb.tree_attention(torch.from_numpy(q), torch.from_numpy(k), torch.from_numpy(v),
                             torch.from_numpy(words(bits)), torch.tensor(lens))
    assert not host.is_cuda and torch.equal(host, plain.cpu())


def test_attention_lengths_are_clamped(cuda):
    """Lengths on the device past the cache's end: the nodes that do not fit do not exist."""
    print("case tree_attention clamped lengths", flush=True)
    B, N, H, KVH, D, S = 4, 6, 4, 2, 64, 50
    q, k, v, bits = inputs(9, B, N, H, KVH, D, S, style="chain")
    lens = [47, 50, 1000, -5]
    want, bound = reference(q, k, v, bits, lens, D ** -0.5)
    T = lambda a: torch.from_numpy(a).to(cuda)
    check(tb.tree_attention(T(q), T(k), T(v), T(words(bits)), torch.tensor(lens, device=cuda)),
          want, bound)
    with pytest.raises(ValueError, match="exceed"):
        tb.tree_attention(T(q), T(k), T(v), T(words(bits)), 45)


def test_indices_past_32_bits(cuda):
    """int64 parents and lengths that int32 does not hold are padding and clamped lengths."""
    print("case int64 parents and lengths", flush=True)
    par = torch.tensor([-1, 0, 1 << 32, (1 << 32) - 1, 2, -(1 << 40), 1], device=cuda)
    mask, depth = tb.tree_masks(par)
    assert mask[:, 0].tolist() == [1, 3, 0, 0, 0, 0, 67] and depth.tolist() == [0, 1, 0, 0, 0, 0, 2]
    q, k, v, bits = inputs(2, 2, 5, 4, 2, 64, 20)
    T = lambda a: torch.from_numpy(a).to(cuda)
    a = [T(q), T(k), T(v), T(words(bits))]
    far = tb.tree_attention(*a, torch.tensor([(1 << 32) + 3, -(1 << 33)], device=cuda))
    assert torch.equal(far, tb.tree_attention(*a, torch.tensor([20, 0], device=cuda)))


def test_attention_empty(cuda):
    print("case tree_attention empty", flush=True)
    z = lambda *s: torch.zeros(s, device=cuda)
    m = lambda *s: torch.zeros(s, dtype=torch.int32, device=cuda)
    assert tb.tree_attention(z(0, 4, 64), z(2, 8, 64), z(2, 8, 64), m(0, 0), 3).shape == (0, 4, 64)
    out = tb.tree_attention(z(0, 3, 4, 64), z(0, 2, 8, 64), z(0, 2, 8, 64), m(3, 1), m(0))
    assert out.shape == (0, 3, 4, 64)
    out = tb.tree_attention(z(3, 4, 64) + 1, z(2, 8, 64) + 1, z(2, 8, 64) + 1, m(3, 1), 3)
    assert (out == 0).all()


@pytest.mark.parametrize("N,kv", [(4, 40), (4, 3000), (20, 3000), (60, 3000), (90, 1000)])
def test_attention_not_finite_queries(cuda, N, kv):
    """A NaN in a query makes its row NaN and no other, with one block and with many."""
    print(f"case tree_attention NaN query N={N} kv={kv}", flush=True)
    H, KVH, D, S = 8, 2, 64, kv + N
    q, k, v, bits = inputs(N, 1, N, H, KVH, D, S)
    q[0, N // 2, 3, 5] = np.nan
    T = lambda a: torch.from_numpy(a).to(cuda)
    out = tb.tree_attention(T(q), T(k), T(v), T(words(bits)), kv).cpu().numpy()
    nan = np.zeros(out.shape, bool)
    nan[0, N // 2, 3] = True
    assert np.array_equal(np.isnan(out), nan)


def test_attention_past_32_bits(cuda):
    """Positions and heads further than 2^31 elements into the cache."""
    print("case tree_attention 64-bit offsets", flush=True)
    N, H, KVH, D, S, kv = 5, 4, 2, 64, 40, 33
    q, k, v, bits = inputs(12, 1, N, H, KVH, D, S)
    ss, sh = 60_000_000, 30_000_000
    buf = torch.empty(S * ss, device=cuda)      # 9.6 GB
    kc = buf.as_strided((KVH, S, D), (sh, ss, 1))
    vc = buf.as_strided((KVH, S, D), (sh, ss, 1), storage_offset=1_000_000)
    T = lambda a: torch.from_numpy(a).to(cuda)
    kc.copy_(T(k[0]))
    vc.copy_(T(v[0]))
    want, bound = reference(q, k, v, bits, [kv], D ** -0.5)
    check(tb.tree_attention(T(q[0]), kc, vc, T(words(bits[0])), kv)[None], want, bound)
    # ... and rows moved there
    par = torch.tensor([-1, 0, 0, 0, 2], dtype=torch.int32, device=cuda)
    draft = torch.tensor([9, 5, 6, 7, 8], device=cuda)
    nxt = torch.tensor([6, 0, 8, 0, 3], device=cuda)
    path, n, tok = tb.tree_accept(par, draft, nxt, kv, [kc], [vc])
    assert path.tolist() == [0, 2, 4, -1, -1] and int(n) == 3 and int(tok) == 3
    for c, w in ((kc, k[0]), (vc, v[0])):
        w = T(w)
        assert torch.equal(c[:, kv + 1], w[:, kv + 2]) and torch.equal(c[:, kv + 2], w[:, kv + 4])
        assert torch.equal(c[:, kv + 3:], w[:, kv + 3:]) and torch.equal(c[:, :kv + 1], w[:, :kv + 1])
    del buf, kc, vc
    torch.cuda.empty_cache()


# ---- acceptance ---------------------------------------------------------------


def walk(par, draft, nxt):
    path = [0] if par[0] == -1 else []
    while path:
        kids = [c for c in range(path[-1] + 1, len(par))
                if par[c] == path[-1] and draft[c] == nxt[path[-1]] and draft[c] >= 0]
        if not kids:
            break
        path.append(kids[0])
    return path, (nxt[path[-1]] if path else -1)


@pytest.mark.parametrize("B,N,L,KVH,D,V", [(1, 1, 1, 1, 32, 3), (1, 26, 3, 2, 64, 2),
                                           (4, 64, 2, 8, 128, 2), (3, 200, 1, 5, 96, 1),
                                           (2, 1024, 1, 1, 256, 2), (1, 40, 70, 2, 64, 2),
                                           (2, 33, 0, 1, 64, 2)])
def test_accept(cuda, B, N, L, KVH, D, V):
    """Few token values, so that paths are long and several children match."""
    print(f"case tree_accept B={B} N={N} L={L} KVH={KVH} D={D}", flush=True)
    g = np.random.default_rng(B + N)
    for trial in range(4):
        par = np.array([tree(g, N, N if b == 0 else max(0, N - 5 * trial), "chain" if trial == 3
                             else "mixed") for b in range(B)], np.int32)
        draft, nxt = g.integers(0, V, (B, N)), g.integers(0, V, (B, N))
        draft[g.random((B, N)) < 0.1] = -1
        nxt[g.random((B, N)) < 0.05] = -1
        lens = g.integers(0, 20, B)
        S = 20 + N
        kc = [torch.from_numpy(g.standard_normal((B, KVH, S, D)).astype(np.float32)).to(cuda)
              for _ in range(2 * L)]
        was = [c.clone() for c in kc]
        T = lambda a: torch.from_numpy(a).to(cuda)
        path, n, tok = tb.tree_accept(T(par), T(draft), T(nxt), T(lens), kc[:L], kc[L:])
        for b in range(B):
            want, last = walk(par[b].tolist(), draft[b].tolist(), nxt[b].tolist())
            assert path[b].tolist() == want + [-1] * (N - len(want))
            assert int(n[b]) == len(want) and int(tok[b]) == last
            for w in was:
                src = w[b].clone()
                for j, p in enumerate(want):
                    w[b][:, lens[b] + j] = src[:, lens[b] + p]
        for c, w in zip(kc, was):
            assert torch.equal(c, w)


def test_accept_cache_end_and_host(cuda):
    """Rows past the cache's end do not exist; host caches are written back."""
    print("case tree_accept cache end, host tensors", flush=True)
    par = torch.tensor([-1, 0, 0, 2, 3], dtype=torch.int32)
    draft, nxt = torch.tensor([0, 1, 2, 3, 4]), torch.tensor([2, 0, 3, 4, 9])
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn((2, 10, 32), generator=g) for _ in range(2))
    k0, v0 = k.clone(), v.clone()
    path, n, tok = tb.tree_accept(par, draft, nxt, torch.tensor([7]), [k], [v])
    assert path.tolist() == [0, 2, 3, 4, -1] and int(n) == 4 and int(tok) == 9
    for c, w in ((k, k0), (v, v0)):      # 7 <- 7, 8 <- 9; rows 10 and 11 are not there
        assert torch.equal(c[:, 8], w[:, 9])
        assert torch.equal(c[:, :8], w[:, :8]) and torch.equal(c[:, 9], w[:, 9])
    with pytest.raises(ValueError, match="exceed"):
        tb.tree_accept(par, draft, nxt, 6, [k], [v])
    # the layers' caches stacked in one tensor
    ks, vs = torch.stack((k0, v0)).to(cuda), torch.stack((v0, k0)).to(cuda)
    tb.tree_accept(par.to(cuda), draft.to(cuda), nxt.to(cuda), torch.tensor([7], device=cuda), ks, vs)
    assert torch.equal(ks.cpu(), torch.stack((k, v))) and torch.equal(vs.cpu(), torch.stack((v, k)))


# ---- streams, graphs -------------------------------------------------------------


def step(st):
    mask, depth = tb.tree_masks(st["par"])
    a = tb.tree_attention(st["q"], st["k"][0], st["v"][0], mask, st["len"])
    lg = a.reshape(a.shape[0], a.shape[1], -1) @ st["head"]
    y = tb.process_logits(lg, st["hist"], repetition_penalty=1.25, frequency_penalty=0.5,
                          draft_tokens=st["draft"], tree_mask=mask)
    t = tb.greedy_tokens(lg, st["hist"], repetition_penalty=1.25, frequency_penalty=0.5,
                         draft_tokens=st["draft"], tree_mask=mask)
    return (depth, a, y, t, *tb.tree_accept(st["par"], st["draft"], t, st["len"], st["k"], st["v"]))


def state(dev, seed, B=2, N=12, H=8, KVH=2, D=64, S=700, V=40):
    g = np.random.default_rng(seed)
    T = lambda a: torch.from_numpy(a).to(dev)
    f = lambda *s: T(g.standard_normal(s).astype(np.float32))
    return dict(par=T(np.array([tree(g, N) for _ in range(B)], np.int32)), q=f(B, N, H, D),
                k=[f(B, KVH, S, D) for _ in range(2)], v=[f(B, KVH, S, D) for _ in range(2)],
                len=T(g.integers(1, S - N, B)), head=f(H * D, V), hist=T(g.integers(0, V, (B, 9))),
                draft=T(g.integers(0, V, (B, N))))


def test_step_on_streams(cuda):
    """The run of all of them, as a decoder makes it: on two streams at once, the results
    and the moved caches equal to the default stream's."""
    print("case tree step on two streams", flush=True)
    want, caches = [], []
    for seed in range(2):
        st = state(cuda, seed)
        want.append(step(st))
        caches.append(st["k"] + st["v"])
    torch.cuda.synchronize()
    for _ in range(3):
        sts = [state(cuda, seed) for seed in range(2)]
        torch.cuda.synchronize()
        outs = []
        for st in sts:
            with torch.cuda.stream(torch.cuda.Stream()):
                outs.append(step(st))
        torch.cuda.synchronize()
        for st, out, w, c in zip(sts, outs, want, caches):
            assert all(torch.equal(a, b) for a, b in zip(out, w))
            assert all(torch.equal(a, b) for a, b in zip(st["k"] + st["v"], c))


def test_step_in_graphs(cuda):
    """Two graphs captured on one stream and replayed side by side with new inputs, eager
    work between the replays: equal to eager calls each time."""
    print("case tree step in two graphs", flush=True)
    s = torch.cuda.Stream()
    sts = [state(cuda, 10 + i) for i in range(2)]
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(state(cuda, 9))      # warm-up
    torch.cuda.synchronize()
    graphs, outs = [], []
    for st in sts:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            outs.append(step(st))
        graphs.append(gr)
    sides = [torch.cuda.Stream() for _ in range(2)]
    for rnd in range(4):
        new = [state(cuda, 20 + 2 * rnd + i) for i in range(2)]
        for st, n in zip(sts, new):
            for key in st:
                if isinstance(st[key], list):
                    for a, b in zip(st[key], n[key]):
                        a.copy_(b)
                else:
                    st[key].copy_(n[key])
        torch.cuda.synchronize()
        for gr, side in zip(graphs, sides):
            with torch.cuda.stream(side):
                gr.replay()
        torch.cuda.synchronize()
        for st, n, out in zip(sts, new, outs):
            want = step(n)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), rnd
            assert all(torch.equal(a, b) for a, b in zip(st["k"] + st["v"], n["k"] + n["v"]))


def test_attention_of_misaligned_queries(cuda):
    """A contiguous q that does not start at a multiple of 16 bytes is copied, as misaligned
    caches are."""
    print("case tree_attention misaligned q", flush=True)
    N, H, KVH, D, S, kv = 5, 4, 2, 64, 60, 40
    q, k, v, bits = inputs(21, 1, N, H, KVH, D, S)
    T = lambda a: torch.from_numpy(a).to(cuda)
    a = (T(k[0]), T(v[0]), T(words(bits[0])), kv)
    want = tb.tree_attention(T(q[0]), *a)
    for off in (1, 2, 3):
        buf = torch.empty(N * H * D + 4, device=cuda)
        x = buf[off:off + N * H * D].view(N, H, D)
        x.copy_(T(q[0]))
        assert x.is_contiguous() and x.data_ptr() % 16
        assert torch.equal(tb.tree_attention(x, *a), want)


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("bad", [0, 1, 2, 3])
def test_accept_of_misaligned_caches(cuda, bad, strided):
    """One cache among the layers' that does not start at a multiple of 16 bytes, the first or
    a later one, contiguous or not: copied and written back."""
    print(f"case tree_accept misaligned cache {bad} strided={strided}", flush=True)
    KVH, S, D = 2, 12, 32
    g = torch.Generator().manual_seed(3)
    was = [torch.randn((KVH, S, D), generator=g) for _ in range(4)]
    caches = []
    for i, w in enumerate(was):
        at = int(i == bad)
        c = torch.empty(KVH * S * D + 4, device=cuda)[at:at + KVH * S * D]
        caches.append(c.view(S, KVH, D).transpose(0, 1) if strided else c.view(KVH, S, D))
        caches[i].copy_(w)
    T = lambda a: torch.tensor(a, device=cuda)
    path, n, tok = tb.tree_accept(T([-1, 0, 0, 2]), T([0, 1, 2, 3]), T([2, 0, 3, 9]), 6, caches[:2],
                                  caches[2:])
    assert path.tolist() == [0, 2, 3, -1] and int(n) == 3 and int(tok) == 9
    for c, w in zip(caches, was):
        w[:, 7:9] = w[:, 8:10].clone()
        assert torch.equal(c.cpu(), w)


def weight_floor(q, k, v, bits, lens, scale, slack):
    """What the bound leaves to weights that are small beside their tile's reference, row by
    row.  A weight's two limbs have 22 bits down to 2^-21 of the reference and an error of
    2^-43 of it below; times the largest V of the 64 positions and 2^slack, where the outputs'
    scale is up to that far above it.  The reference is at most the row's largest score, and
    at most 2^24 above the tile's largest one while that is 2^-36 of the largest or more."""
    out = np.zeros((*q.shape[:3], 1))
    G = q.shape[2] // k.shape[1]
    for b, i, h in np.ndindex(*q.shape[:3]):
        if not bits[b, i].any():
            continue
        n = bits.shape[1]
        s = k[b, h // G, :lens[b] + n].astype(np.float64) @ q[b, i, h].astype(np.float64) * scale
        s[lens[b]:][~bits[b, i]] = -np.inf
        w = np.exp(s - s.max())
        big = np.abs(v[b, h // G, :lens[b] + n]).max(-1)
        for t in range(0, len(w), 64):
            top = w[t:t + 64].max()
            out[b, i, h] += 64 * 2.0 ** (slack - 43) * big[t:t + 64].max() * \
                min(1.0, max(2.0 ** 24 * top, 2.0 ** -36))
    return out


@pytest.mark.parametrize("N,H,KVH,D,kv,S", [
    (2, 4, 2, 128, 9000, 9100), (8, 8, 2, 64, 3000, 3100),          # few rows
    (40, 8, 2, 64, 5000, 5100), (49, 8, 2, 128, 2000, 2100), (17, 4, 1, 224, 1500, 1600),
    (64, 8, 2, 64, 3000, 131072), (64, 4, 1, 128, 1500, 131200),    # blocks of eight waves
])
@pytest.mark.parametrize("gap", [8.0, 14.0, 21.1, 39.0])
def test_attention_of_small_weights(cuda, N, H, KVH, D, kv, S, gap):
    """One position whose V is zero takes nearly all of the weight; the result is that of the
    others, each with e^-gap of it, all of them alike, so that their errors add up."""
    print(f"case tree_attention small weights N={N} H={H}/{KVH} D={D} kv={kv} gap={gap}", flush=True)
    g = np.random.default_rng(N)
    bits = ancestors(tree(g, N))[0][None]
    q = np.zeros((1, N, H, D), np.float32)
    k, v = np.zeros((1, KVH, kv + N, D), np.float32), np.ones((1, KVH, kv + N, D), np.float32)
    q[..., 0] = 1.0
    for at in (0, kv // 2 + 5):      # in the first split and in another
        k[..., 0] = 0.0
        k[:, :, at, 0] = gap
        v[:] = 1.0
        v[:, :, at] = 0.0
        want, bound = reference(q, k, v, bits, [kv], 1.0)
        bound += weight_floor(q, k, v, bits, [kv], 1.0, 1)
        # sharp: 2 ds is 3.4e-4 at most, and the tile of the large weight leaves 64 2^-42
        assert (bound < 1e-3 * want + 2e-11).all()
        T = lambda a: torch.from_numpy(a).to(cuda)
        kc, vc = (torch.zeros((1, KVH, S, D), device=cuda) for _ in range(2))
        kc[:, :, :kv + N], vc[:, :, :kv + N] = T(k), T(v)
        got = tb.tree_attention(T(q), kc, vc, T(words(bits)), torch.tensor([kv], device=cuda), 1.0)
        check(got, want, bound)


@pytest.mark.parametrize("N,H,KVH,D,kv,S", [
    (2, 4, 2, 128, 700, 800), (8, 8, 2, 64, 700, 800), (40, 8, 2, 64, 700, 800),
    (49, 8, 2, 128, 700, 800), (17, 4, 1, 224, 700, 800), (64, 8, 2, 64, 700, 131072),
])
@pytest.mark.parametrize("fall,rise", [(30.0, 0.0), (60.0, 50.0), (100.0, 90.0), (40.0, -80.0),
                                       (-80.0, 60.0), (-60.0, -60.0)])
def test_attention_of_falling_scores(cuda, N, H, KVH, D, kv, S, fall, rise):
    """Scores that fall by `fall` powers of two over the cache (or rise, up and down again in
    every fourth position), V that grows or shrinks by `rise` of them: small weights of large
    V, and references and scales that follow both."""
    print(f"case tree_attention falling scores N={N} H={H}/{KVH} D={D} {fall} {rise}", flush=True)
    q, k, v, bits = inputs(N + D, 1, N, H, KVH, D, kv + N)
    x = np.arange(kv + N) / (kv + N)
    k *= 0.05
    q[..., 0] = 1.0
    k[..., 0] = (-fall * np.log(2) * x)[None, None]
    k[:, :, 3::4, 0] *= 0.5
    v *= (2.0 ** (rise * x))[None, None, :, None].astype(np.float32)
    want, bound = reference(q, k, v, bits, [kv], 1.0)
    bound += weight_floor(q, k, v, bits, [kv], 1.0, 8)
    T = lambda a: torch.from_numpy(a).to(cuda)
    kc, vc = (torch.zeros((1, KVH, S, D), device=cuda) for _ in range(2))
    kc[:, :, :kv + N], vc[:, :, :kv + N] = T(k), T(v)
    got = tb.tree_attention(T(q), kc, vc, T(words(bits)), torch.tensor([kv], device=cuda), 1.0)
    check(got, want, bound)


def test_attention_sums_of_zero_values(cuda):
    """As test_attention_weights_of_zero_values, with an allowance for the positions whose V is
    large alone: what is lost from the sum of weights would show."""
    print("case tree_attention sums of zero values", flush=True)
    for N, H, D in ((2, 4, 128), (40, 8, 64), (60, 16, 128)):
        KVH, kv, S = 2, 4000, 4100
        q, k, v, bits = inputs(31, 1, N, H, KVH, D, S)
        v[:, :, :kv] = 0.0
        v[:, :, 3900:3904] = 1e7
        want, bound = reference(q, k, v, bits, [kv], D ** -0.5)
        floor = weight_floor(q, k, v, bits, [kv], D ** -0.5, 1)
        assert floor.max() < 1e-3
        T = lambda a: torch.from_numpy(a).to(cuda)
        check(tb.tree_attention(T(q), T(k), T(v), T(words(bits)), kv), want, bound + floor)


@pytest.mark.parametrize("D,N,kv,S", [(64, 6, 40, 46), (128, 25, 90, 115), (96, 60, 200, 260),
                                      (256, 33, 65, 98), (64, 60, 30, 131072)])
@pytest.mark.parametrize("big", [1e6, 3e38])
def test_attention_large_values_seen(cuda, D, N, kv, S, big):
    """Rows that see nodes of very large V, with no allowance beside the bound: those tiles are
    worked in f32."""
    print(f"case tree_attention large values seen D={D} N={N} kv={kv} big={big}", flush=True)
    H, KVH = 8, 2
    q, k, v, bits = inputs(D + N + 1, 1, N, H, KVH, D, kv + N, [N - 1])
    nodes = [0, N // 2, N - 1]
    for j in nodes:
        v[:, :, kv + j] = np.clip(v[:, :, kv + j], -1, 1) * np.float32(big)
    want, bound = reference(q, k, v, bits, [kv], D ** -0.5)
    T = lambda a: torch.from_numpy(a).to(cuda)
    kc, vc = (torch.zeros((1, KVH, S, D), device=cuda) for _ in range(2))
    kc[:, :, :kv + N], vc[:, :, :kv + N] = T(k), T(v)
    check(tb.tree_attention(T(q), kc, vc, T(words(bits)), torch.tensor([kv], device=cuda)), want,
          bound)
