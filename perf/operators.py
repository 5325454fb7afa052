"""Performance cases of the operators of a speculative step over a drafted tree.

A step of tree speculation verifies a tree of drafted tokens in one forward
over the KV cache and keeps the path that the model agrees with:

  masks    the ancestor bit masks and depths of a tree, from its parent list
  attn     attention of the tree's nodes over the cached prefix and their own
           ancestors, whose K / V rows follow the prefix in the cache
  logits   penalties for repeated tokens, biases and grammar masks on the rows
           of logits, and (greedy) each row's best token
  accept   the walk down the tree along the model's own tokens, and the accepted
           rows' move to the end of the prefix in every layer's cache

Sizes are those of the repository's benchmark configurations (Qwen2.5-0.5B and
Llama-3-8B heads and vocabularies) or generic; `draw` spreads more cases over
the same ranges.  Trees hold the drafter's first choices as a chain of nodes
first and its other choices after them; batches of trees are padded to the
largest one's node count.

`own` False computes the operators from elementary torch operations in 32 bits;
`own` True calls torchburn_amd.
"""
import math
import random

import numpy as np
import torch

own = False

QWEN_0_5B = dict(heads=14, kv_heads=2, head_dim=64)
LLAMA3_8B = dict(heads=32, kv_heads=8, head_dim=128)


def _masks(batch, nodes, **kw):
    return dict(op="masks", batch=batch, nodes=nodes, **kw)


def _attn(shape, batch, nodes, kv, **kw):
    return dict(op="attn", batch=batch, nodes=nodes, kv=kv, **shape, **kw)


def _logits(rows, vocab, hist, groups=1, prompt=0, rep=1.0, pres=0.0, freq=0.0, per_row=False,
            bias=0, allow=1.0, tree=False, greedy=False, **kw):
    return dict(op="logits", rows=rows, vocab=vocab, hist=hist, groups=groups, prompt=prompt,
                rep=rep, pres=pres, freq=freq, per_row=per_row, bias=bias, allow=allow, tree=tree,
                greedy=greedy, **kw)


def _accept(layers, kv_heads, head_dim, nodes, keep, side, kv, batch=1, **kw):
    return dict(op="accept", layers=layers, kv_heads=kv_heads, head_dim=head_dim, nodes=nodes,
                keep=keep, side=side, kv=kv, batch=batch, **kw)


def listed():
    return [
        # One sequence's draft tree; launch and host latency.
        _masks(1, 26, name="masks_one"),
        # The trees of a batch of sequences, large ones.
        _masks(64, 512, name="masks_batch"),
        # The smallest attention call: a few drafted tokens of a 0.5B model on a short prompt.
        _attn(QWEN_0_5B, 1, 7, 61, name="attn_small"),
        # One layer of an 8B model: a usual draft tree over 4096 cached positions.
        _attn(LLAMA3_8B, 1, 49, 4096, name="attn_tree_8b"),
        # A wide draft tree over a long document.
        _attn(LLAMA3_8B, 1, 64, 32767, name="attn_tree_long"),
        # A batch of sequences of different lengths, a small tree each.
        _attn(dict(heads=28, kv_heads=4, head_dim=128), 12, 21, 6000, name="attn_batch_ragged"),
        # One row: the next token of a 0.5B model with a repetition penalty.
        _logits(1, 151936, 300, rep=1.125, name="logits_token"),
        # Every node of a draft tree: one shared history, the node's own path, a grammar mask.
        _logits(64, 128256, 2048, prompt=1500, rep=1.125, pres=0.25, freq=0.125, allow=0.6,
                tree=True, name="logits_tree"),
        # A batch of requests, each with its own history, penalties, biases and mask.
        _logits(192, 128256, 1500, groups=192, prompt=400, rep=1.25, pres=0.5, freq=0.25,
                per_row=True, bias=64, allow=0.9, name="logits_batch"),
        # The greedy tokens of four draft trees under a strict grammar; an odd vocabulary.
        _logits(100, 32003, 500, groups=4, rep=1.125, allow=0.02, tree=True, greedy=True,
                name="greedy_trees"),
        # Acceptance in a 0.5B model's cache: a short tree, two side tokens.
        _accept(24, 2, 64, 15, 2, 2, 200, name="accept_small"),
        # Acceptance in an 8B model's cache: a usual tree, a path off the first choices.
        _accept(32, 8, 128, 49, 2, 5, 900, name="accept_8b"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """One more case of the listed ones' ranges."""
    op = rng.choice(("masks", "attn", "attn", "attn", "logits", "logits", "accept"))
    if op == "masks":
        nodes = _log(rng, 1, 512)
        return _masks(_log(rng, 1, 64), nodes)
    if op == "attn":
        kvh = rng.choice((1, 2, 4, 8))
        shape = dict(heads=kvh * rng.choice((1, 2, 4, 5, 7, 8)), kv_heads=kvh,
                     head_dim=rng.choice((32, 64, 64, 96, 128, 128, 128, 160, 192, 256)))
        nodes, kv, batch = _log(rng, 1, 256), _log(rng, 1, 32767), _log(rng, 1, 12)
        most = 32 * 64 * 32768 * 128      # no more work than the long document's
        while batch * shape["heads"] * nodes * kv * shape["head_dim"] > most:
            nodes, kv, batch = max(1, nodes // 2), max(1, kv * 3 // 4), max(1, batch - 1)
        while batch * kvh * kv * shape["head_dim"] > 8 * 32768 * 128:
            kv = kv * 3 // 4
        return _attn(shape, batch, nodes, kv)
    if op == "logits":
        rows, vocab = _log(rng, 1, 192), _log(rng, 1000, 151936)
        groups = rng.choice((1, rows))
        tree = groups == 1 and rng.random() < 0.6
        hist = _log(rng, 1, 2048)
        return _logits(rows, vocab, hist, groups, rng.choice((0, hist // 2)),
                       rng.choice((1.0, 1.125, 1.5)), rng.choice((0.0, 0.5)),
                       rng.choice((0.0, 0.25)), rng.random() < 0.3, rng.choice((0, 0, 7, 200)),
                       rng.choice((1.0, 0.95, 0.3, 0.01)), tree, rng.random() < 0.4)
    nodes = _log(rng, 4, 256)
    keep = rng.randint(1, max(1, min(8, nodes // 3)))
    side = rng.randint(0, max(0, min(8, nodes // 4)))
    return _accept(rng.randint(1, 32), rng.choice((1, 2, 4, 8)), rng.choice((64, 128)), nodes,
                   keep, side, _log(rng, 1, 900), rng.choice((1, 1, 2)))


# ---- inputs, from the seed alone ------------------------------------------


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


def _lengths(r, batch, most, least=1):
    """Ragged lengths up to `most`, the first one `most`."""
    return [most] + [r.randint(min(least, most), most) for _ in range(batch - 1)]


def _tree(r, nodes, used, chain=None, keep=0, side=0):
    """Parents of a tree of `used` nodes padded to `nodes` (-2): a chain of first choices, then
    the other choices, off shallow nodes more often than off deep ones.  With `side`, the first
    of them are a chain of `side` nodes off the first chain's node keep - 1."""
    chain = min(used - 1, chain if chain is not None else max(1, min(12, used // 4)))
    par = [-1] + list(range(chain))[:max(0, used - 1)]
    par = par[:used]
    while len(par) < used:
        i, j = len(par), len(par) - chain - 1
        par.append((keep - 1 if j == 0 else i - 1) if j < side
                   else int((i - 1) * r.random() ** 2))
    return par + [-2] * (nodes - used)


def _ancestors(parents):
    """[B][N][N] truth values: node j is node i or an ancestor of it (False for padding)."""
    out = []
    for par in parents:
        n = len(par)
        a = np.zeros((n, n), bool)
        for i, p in enumerate(par):
            if p == -1 or (0 <= p < i and a[p, p]):
                if p >= 0:
                    a[i] = a[p]
                a[i, i] = True
        out.append(a)
    return np.stack(out)


def _words(bits):
    """Truth values [..., n] as int32 words [..., ceil(n / 32)], bit k % 32 of word k // 32."""
    n = bits.shape[-1]
    w = (n + 31) // 32
    if isinstance(bits, np.ndarray):
        bits = torch.from_numpy(bits)
    pad = torch.zeros((*bits.shape[:-1], w * 32), dtype=torch.int64, device=bits.device)
    pad[..., :n] = bits
    pad = pad.reshape(*bits.shape[:-1], w, 32) << torch.arange(32, device=bits.device)
    v = pad.sum(-1)
    return torch.where(v >= 1 << 31, v - (1 << 32), v).to(torch.int32)


def _bits(words, n):
    """The inverse of _words: truth values [..., n]."""
    b = (words.unsqueeze(-1) >> torch.arange(32, dtype=torch.int32, device=words.device)) & 1
    return b.reshape(*words.shape[:-1], -1)[..., :n] != 0


def _tokens(g, vocab, *shape):
    """Token ids as text has them: a few of them often, most rarely."""
    return (torch.rand(shape, device="cuda", generator=g) ** 3 * vocab).long().clamp_(max=vocab - 1)


def prepare(case, seed):
    g, r, op = _gen(seed), random.Random(int(seed)), case["op"]
    st = dict(case=case)
    if op == "masks":
        b, n = case["batch"], case["nodes"]
        par = [_tree(r, n, u) for u in _lengths(r, b, n)]
        st["parents"] = torch.tensor(par, dtype=torch.int32, device="cuda")
        return st
    if op == "attn":
        b, n, kv = case["batch"], case["nodes"], case["kv"]
        h, kvh, d = case["heads"], case["kv_heads"], case["head_dim"]
        lens = _lengths(r, b, kv, kv // 8)
        par = [_tree(r, n, u) for u in _lengths(r, b, n)]
        rows = (kv + n + 127) // 64 * 64      # the cache's positions, some of them free
        st["q"] = 2.0 * _normal(g, b, n, h, d)
        st["k"], st["v"] = _normal(g, b, kvh, rows, d), _normal(g, b, kvh, rows, d)
        st["mask"] = _words(_ancestors(par)).cuda()
        st["kv_len"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["longest"] = max(lens)     # the program knows its sequences' lengths
        return st
    if op == "logits":
        rows, v, gr, hist = case["rows"], case["vocab"], case["groups"], case["hist"]
        st["logits"] = 3.0 * _normal(g, rows, v)
        st["history"] = _tokens(g, v, gr, hist)
        lens = _lengths(r, gr, hist, hist // 4)
        st["history_len"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["prompt_len"] = torch.tensor([min(case["prompt"], n) for n in lens], dtype=torch.int32,
                                        device="cuda")
        for f in ("rep", "pres", "freq"):
            st[f] = case[f]
            if case["per_row"]:
                st[f] = case[f] * (0.5 + torch.rand(rows, device="cuda", generator=g))
        if case["bias"]:
            st["bias_ids"] = torch.stack([torch.randperm(v, device="cuda", generator=g)
                                          [:case["bias"]] for _ in range(gr)])
            st["bias_values"] = 4.0 * _normal(g, *st["bias_ids"].shape)
        if case["allow"] < 1.0:
            allowed = torch.rand((rows, v), device="cuda", generator=g) < case["allow"]
            st["allowed"] = torch.cat([_words(allowed[i:i + 16]) for i in range(0, rows, 16)])
        if case["tree"]:
            n = rows // gr
            st["drafts"] = _tokens(g, v, gr, n)
            st["mask"] = _words(_ancestors([_tree(r, n, n) for _ in range(gr)])).cuda()
        return st
    b, n, kv, keep, side = (case[f] for f in ("batch", "nodes", "kv", "keep", "side"))
    vocab, chain = 128256, min(n - 1 - side, max(keep + side, n // 4))
    par = [_tree(r, n, n, chain, keep, side) for _ in range(b)]
    drafts = torch.randint(0, vocab - 1, (b, n), device="cuda", generator=g)
    nxt = torch.randint(0, vocab - 1, (b, n), device="cuda", generator=g)
    path = list(range(keep)) + list(range(chain + 1, chain + 1 + side))
    for a, c in zip(path, path[1:]):
        nxt[:, a] = drafts[:, c]
    nxt[:, path[-1]] = vocab - 1      # no drafted token: the path ends here
    st["parents"] = torch.tensor(par, dtype=torch.int32, device="cuda")
    st["drafts"], st["next"] = drafts, nxt
    st["kv_len"] = torch.tensor(_lengths(r, b, kv), dtype=torch.int32, device="cuda")
    rows = (kv + n + 127) // 64 * 64
    # the layers' caches, each a view of one allocation
    shape = (case["layers"], b, case["kv_heads"], rows, case["head_dim"])
    st["caches"] = _normal(g, *shape), _normal(g, *shape)
    st["k"], st["v"] = (list(c.unbind(0)) for c in st["caches"])
    return st


# ---- the plain forms --------------------------------------------------------


def _plain_masks(parents):
    b, n = parents.shape
    idx = torch.arange(n, device=parents.device)
    root = parents == -1
    child = (parents >= 0) & (parents < idx)
    p = parents.clamp(0, n - 1).long()
    # reach[i, j]: node j is at most 2^k - 1 steps above node i
    step = torch.zeros((b, n, n), device=parents.device)
    step.scatter_(2, p.unsqueeze(-1), child.float().unsqueeze(-1))
    reach = torch.eye(n, device=parents.device).expand(b, n, n)
    reach = (reach + step).clamp(max=1.0)
    k = 1
    while k < n:
        reach = (reach @ reach).clamp(max=1.0)
        k *= 2
    live = (reach * root.float().unsqueeze(1)).sum(-1) > 0      # its topmost ancestor is a root
    anc = (reach > 0) & live.unsqueeze(-1)
    depth = (anc.sum(-1) - 1).clamp(min=0).to(torch.int32)
    return _words(anc), depth


def _plain_attn(q, k, v, mask, kv_len, longest):
    b, n, h, d = q.shape
    kvh = k.shape[1]
    used = min(longest + n, k.shape[2])
    k, v = k[:, :, :used].float(), v[:, :, :used].float()
    x = q.float().reshape(b, n, kvh, h // kvh, d).permute(0, 2, 1, 3, 4).reshape(b, kvh, -1, d)
    s = (x @ k.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    at = torch.arange(used, device=q.device) - kv_len.unsqueeze(-1)      # [b, used]
    anc = _bits(mask, n)                                               # [b, n, n]
    node = at.clamp(0, n - 1).long().unsqueeze(1).expand(b, n, used)
    see = torch.where((at < 0).unsqueeze(1), anc.any(-1, keepdim=True),
                      anc.gather(2, node) & (at < n).unsqueeze(1))
    see = see.unsqueeze(2).expand(b, n, h // kvh, used).reshape(b, 1, -1, used)
    s = s.masked_fill(~see, -math.inf)
    top = s.max(-1, keepdim=True).values
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    o = (e @ v) / e.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.reshape(b, kvh, n, h // kvh, d).permute(0, 2, 1, 3, 4).reshape(b, n, h, d)


def _column(x, rows):
    return x.unsqueeze(-1) if torch.is_tensor(x) else x


def _plain_logits(st):
    c, x = st["case"], st["logits"].float()
    rows, v = x.shape
    gr, dev = c["groups"], x.device
    at = torch.arange(c["hist"], device=dev)
    real = at < st["history_len"].unsqueeze(-1)
    made = real & (at >= st["prompt_len"].unsqueeze(-1))
    count = torch.zeros((gr, v), device=dev).scatter_add_(1, st["history"], made.float())
    seen = torch.zeros((gr, v), device=dev).scatter_add_(1, st["history"], real.float())
    count = count.repeat_interleave(rows // gr, 0)
    seen = seen.repeat_interleave(rows // gr, 0)
    if c["tree"]:
        n = rows // gr
        anc = _bits(st["mask"], n).reshape(rows, n).float()
        ids = st["drafts"].unsqueeze(1).expand(gr, n, n).reshape(rows, n)
        count.scatter_add_(1, ids, anc)
        seen.scatter_add_(1, ids, anc)
    rep, pres, freq = (_column(st[f], rows) for f in ("rep", "pres", "freq"))
    y = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    y = (y - freq * count) - (count > 0) * pres
    if c["bias"]:
        bias = torch.zeros((gr, v), device=dev).scatter_add_(1, st["bias_ids"], st["bias_values"])
        y = y + bias.repeat_interleave(rows // gr, 0)
    if c["allow"] < 1.0:
        y = y.masked_fill(~_bits(st["allowed"], v), -math.inf)
    if not c["greedy"]:
        return y
    y = torch.where(torch.isnan(y), -math.inf, y)
    top = y.max(-1, keepdim=True).values
    first = torch.where((y == top) & (y > -math.inf), torch.arange(v, device=dev), v).min(-1).values
    return torch.where(first == v, -1, first)


def _plain_accept(st):
    par, drafts, nxt = st["parents"].long(), st["drafts"], st["next"]
    b, n = par.shape
    idx = torch.arange(n, device=par.device)
    node = torch.where(par[:, 0] == -1, 0, -1)
    path = torch.full((b, n), -1, device=par.device)
    last = node
    # no path is longer than the trees' first chains, which the program knows
    most = st["case"]["keep"] + st["case"]["side"] + 1
    for j in range(min(most, n)):
        path[:, j] = node
        last = torch.where(node >= 0, node, last)
        want = nxt.gather(1, node.clamp(min=0).unsqueeze(-1))
        kid = (par == node.unsqueeze(-1)) & (drafts == want) & (node >= 0).unsqueeze(-1) & \
            (idx > node.unsqueeze(-1))
        node = torch.where(kid, idx, n).min(-1).values
        node = torch.where(node == n, -1, node)
    count = (path >= 0).sum(-1)
    token = torch.where(last >= 0, nxt.gather(1, last.clamp(min=0).unsqueeze(-1)).squeeze(-1), -1)
    lens = st["kv_len"].long().unsqueeze(-1)
    # every path entry's row moves; entries past the path move nothing (row to itself)
    at = torch.arange(n, device=par.device)
    src = (lens + torch.where(path >= 0, path, at))[:, :most]
    dst = (lens + at)[:, :most]
    for c in (*st["k"], *st["v"]):
        kvh, d = c.shape[1], c.shape[3]
        s = src.view(b, 1, -1, 1).expand(b, kvh, src.shape[1], d)
        t = dst.view(b, 1, -1, 1).expand(b, kvh, dst.shape[1], d)
        c.scatter_(2, t, c.gather(2, s))
    return path.to(torch.int32), count.to(torch.int32), token


# ---- one pass -----------------------------------------------------------------


def run(st):
    op = st["case"]["op"]
    if not own:
        if op == "masks":
            return _plain_masks(st["parents"])
        if op == "attn":
            return _plain_attn(st["q"], st["k"], st["v"], st["mask"], st["kv_len"], st["longest"])
        if op == "logits":
            return _plain_logits(st)
        return (*_plain_accept(st), *st["caches"])
    import torchburn_amd as tb
    if op == "masks":
        return tb.tree_masks(st["parents"])
    if op == "attn":
        return tb.tree_attention(st["q"], st["k"], st["v"], st["mask"], st["kv_len"])
    if op == "logits":
        call = tb.greedy_tokens if st["case"]["greedy"] else tb.process_logits
        return call(st["logits"], st["history"], history_len=st["history_len"],
                    prompt_len=st["prompt_len"], repetition_penalty=st["rep"],
                    presence_penalty=st["pres"], frequency_penalty=st["freq"],
                    bias_ids=st.get("bias_ids"), bias_values=st.get("bias_values"),
                    allowed=st.get("allowed"), draft_tokens=st.get("drafts"),
                    tree_mask=st.get("mask"))
    path, count, token = tb.tree_accept(st["parents"], st["drafts"], st["next"], st["kv_len"],
                                        st["k"], st["v"])
    return path, count, token, *st["caches"]


def work(case):
    op = case["op"]
    if op == "masks":
        b, n = case["batch"], case["nodes"]
        return dict(bytes=4 * b * n * (2 + (n + 31) // 32), flops=b * n * max(1, n // 32))
    if op == "attn":
        b, n, h, kvh, d = (case[f] for f in ("batch", "nodes", "heads", "kv_heads", "head_dim"))
        # lengths are spread evenly from an eighth of the longest on
        mean = (case["kv"] + (b - 1) * case["kv"] * 9 / 16) / b
        return dict(bytes=int(4 * b * d * (2 * n * h + 2 * kvh * (mean + n))),
                    flops=int(4 * b * h * n * (mean + n) * d))
    if op == "logits":
        r, v = case["rows"], case["vocab"]
        nbytes = r * v * (4 if case["greedy"] else 8) + 8 * case["groups"] * case["hist"]
        if case["allow"] < 1.0:
            nbytes += r * ((v + 31) // 32) * 4
        return dict(bytes=nbytes, flops=2 * r * v)
    row = case["layers"] * case["kv_heads"] * case["head_dim"] * 4 * 2      # K and V
    return dict(bytes=case["batch"] * (2 * row * case["side"] + 20 * case["nodes"]),
                flops=case["batch"] * case["nodes"])


# ---- the operators' definitions, in 64 bits ------------------------------------


def exact(case, seed):
    st, op = prepare(case, seed), case["op"]
    if op == "masks":
        anc = _ancestors(st["parents"].tolist())
        depth = np.maximum(anc.sum(-1) - 1, 0)
        return _words(anc), torch.from_numpy(depth.astype(np.int32))
    if op == "attn":
        q, mask = st["q"].double(), st["mask"].cpu().numpy().view(np.uint32)
        b, n, h, d = q.shape
        group = h // case["kv_heads"]
        out = torch.zeros_like(q)
        for i, ln in enumerate(st["kv_len"].tolist()):
            keys = [[j for j in range(n) if mask[i, t, j // 32] >> (j % 32) & 1] for t in range(n)]
            hide = torch.ones((n, n), dtype=torch.bool)
            for t, js in enumerate(keys):
                hide[t, js] = False
            hide = hide.to(q.device)
            for hh in range(h):
                k = st["k"][i, hh // group, :ln + n].double()
                v = st["v"][i, hh // group, :ln + n].double()
                s = q[i, :, hh] @ k.T / d ** 0.5
                s[:, ln:][hide] = -math.inf
                out[i, :, hh] = torch.softmax(s, -1) @ v
            for t, js in enumerate(keys):
                if not js:
                    out[i, t] = 0.0
        return out
    if op == "logits":
        rows, gr, v = case["rows"], case["groups"], case["vocab"]
        x = st["logits"].double()
        lens, prompts = st["history_len"].tolist(), st["prompt_len"].tolist()
        word = None if case["allow"] >= 1.0 else st["allowed"]
        masks = st["mask"].cpu().numpy().view(np.uint32) if case["tree"] else None
        best = []
        for r in range(rows):
            a = r // (rows // gr)
            toks = st["history"][a, :lens[a]]
            path = toks[:0]
            if case["tree"]:
                i = r % (rows // gr)
                path = st["drafts"][a, [j for j in range(rows // gr)
                                        if masks[a, i, j // 32] >> (j % 32) & 1]]
            rep, pres, freq = (float(st[f][r]) if torch.is_tensor(st[f]) else st[f]
                               for f in ("rep", "pres", "freq"))
            y = x[r]
            ids = torch.unique(torch.cat((toks, path)))
            y[ids] = torch.where(y[ids] > 0, y[ids] / rep, y[ids] * rep)
            ids, times = torch.unique(torch.cat((toks[prompts[a]:], path)), return_counts=True)
            y[ids] -= times.double() * freq + pres
            if case["bias"]:
                y[st["bias_ids"][a]] += st["bias_values"][a].double()
            if word is not None:
                t = torch.arange(v, device=y.device)
                y[(word[r][t // 32] >> (t % 32)) & 1 == 0] = -math.inf
            if case["greedy"]:
                j = int(torch.argmax(y))
                j = int((y == y[j]).nonzero()[0])
                best.append(j if y[j] > -math.inf else -1)
        return torch.tensor(best) if case["greedy"] else x
    parents, drafts, nxt = st["parents"].tolist(), st["drafts"].tolist(), st["next"].tolist()
    k, v = (c.double() for c in st["caches"])
    paths, counts, tokens = [], [], []
    for i, (par, dr, nx) in enumerate(zip(parents, drafts, nxt)):
        path = [0]
        while True:
            kids = [c for c in range(path[-1] + 1, len(par))
                    if par[c] == path[-1] and dr[c] == nx[path[-1]]]
            if not kids:
                break
            path.append(kids[0])
        ln = int(st["kv_len"][i])
        for c, was in zip((k, v), st["caches"]):
            for j, p in enumerate(path):
                c[:, i, :, ln + j] = was[:, i, :, ln + p].double()
        paths.append(path + [-1] * (len(par) - len(path)))
        counts.append(len(path))
        tokens.append(nx[path[-1]])
    return (torch.tensor(paths, dtype=torch.int32), torch.tensor(counts, dtype=torch.int32),
            torch.tensor(tokens), k, v)
