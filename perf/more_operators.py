"""Performance cases of decoding many sequences from one shared prompt.

Several continuations of one prompt (samples side by side, or the beams of a
beam search) share the prompt's cache and have a short one each for what they
added.  A step takes each sequence's last token:

  rope     norms of the query and key heads and their position rotation in one
           pass; in a step the key and value rows go to the sequences' caches
  prefix   attention over the shared prompt, read once for all of its sequences,
           and each sequence's own cache
  select   the best continuations of a group of beams, over beams and vocabulary
  reorder  the beams' caches follow the selection, in place, in every layer

Sizes are those of the repository's benchmark configurations (Qwen2.5-0.5B and
Llama-3-8B heads and vocabularies) or generic; `draw` spreads more cases over
the same ranges.

`own` False computes the operators from elementary torch operations in 32 bits
(angles and the selection's values in 64); `own` True calls torchburn_amd.
"""
import math
import random

import torch

own = False

QWEN_0_5B = dict(heads=14, kv_heads=2, head_dim=64)
LLAMA3_8B = dict(heads=32, kv_heads=8, head_dim=128)


def _rope(shape, tokens, rotary, start, append=0, norm=True, interleaved=False, scaled=False, **kw):
    return dict(op="rope", tokens=tokens, rotary=rotary, start=start, append=append, norm=norm,
                interleaved=interleaved, scaled=scaled, **shape, **kw)


def _prefix(shape, groups, rows, prefix, own_len, **kw):
    return dict(op="prefix", groups=groups, rows=rows, prefix=prefix, own_len=own_len, **shape, **kw)


def _select(groups, beams, vocab, k, first=False, ended=False, masked=False, **kw):
    return dict(op="select", groups=groups, beams=beams, vocab=vocab, k=k, first=first,
                ended=ended, masked=masked, **kw)


def _reorder(layers, kv_heads, head_dim, groups, beams, length, **kw):
    return dict(op="reorder", layers=layers, kv_heads=kv_heads, head_dim=head_dim, groups=groups,
                beams=beams, length=length, **kw)


def listed():
    return [
        # One layer's step of four beams of a 0.5B model; launch and host latency.
        _rope(QWEN_0_5B, 4, 64, 200, append=32, name="rope_step_small"),
        # A step of 64 sequences behind a long document, scaled positions.
        _rope(LLAMA3_8B, 64, 128, 100000, append=256, scaled=True, name="rope_step_batch"),
        # The prompt itself, which all of them share.
        _rope(LLAMA3_8B, 4096, 128, 0, name="rope_prompt"),
        # A prompt whose heads rotate in part, in neighbouring pairs, without norms; odd length.
        _rope(dict(heads=28, kv_heads=4, head_dim=96), 1777, 48, 5000, norm=False,
              interleaved=True, name="rope_prompt_part"),
        # The smallest attention call: four beams of a 0.5B model on a short prompt.
        _prefix(QWEN_0_5B, 1, 4, 200, 7, name="prefix_small"),
        # One layer of an 8B model: the beams of one search over 4096 tokens.
        _prefix(LLAMA3_8B, 1, 8, 4096, 64, name="prefix_beams_8b"),
        # A batch of requests behind one long system prompt, each of a length of its own.
        _prefix(LLAMA3_8B, 1, 64, 16384, 256, name="prefix_batch_8b"),
        # Six searches of five beams, each over a prompt of its own; ragged.
        _prefix(dict(heads=28, kv_heads=4, head_dim=128), 6, 5, 2999, 121, name="prefix_groups"),
        # Four beams of a small search; an odd vocabulary, twice as many candidates as beams.
        _select(1, 4, 32003, 8, name="select_small"),
        # A batch of searches over a large vocabulary, some beams ended, a grammar's masks.
        _select(32, 8, 128256, 16, ended=True, masked=True, name="select_batch"),
        # The caches of a 0.5B model's four beams.
        _reorder(24, 2, 64, 1, 4, 50, name="reorder_small"),
        # The caches of an 8B model's four searches of eight beams.
        _reorder(32, 8, 128, 4, 8, 93, name="reorder_8b"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """One more case of the listed ones' ranges."""
    op = rng.choice(("rope", "rope", "prefix", "prefix", "prefix", "select", "select", "reorder"))
    kvh = rng.choice((1, 2, 4, 8))
    heads = kvh * rng.choice((1, 2, 4, 5, 7, 8))
    if op == "rope":
        d = rng.choice((32, 64, 64, 72, 80, 96, 128, 128, 128, 160, 192, 256))
        rotary = max(2, int(d * rng.choice((1.0, 1.0, 0.5, 0.25))) // 2 * 2)
        append = rng.random() < 0.5
        tokens = _log(rng, 1, 256 if append else 4096)
        while tokens * (heads + 2 * kvh) * d > 4096 * 40 * 128:
            tokens = tokens * 3 // 4
        return _rope(dict(heads=heads, kv_heads=kvh, head_dim=d), tokens, rotary,
                     rng.choice((0, _log(rng, 1, 1000000))), _log(rng, 1, 256) if append else 0,
                     rng.random() < 0.6, rng.random() < 0.4, rng.random() < 0.4)
    if op == "prefix":
        shape = dict(heads=heads, kv_heads=kvh,
                     head_dim=rng.choice((32, 64, 64, 96, 128, 128, 128, 160, 192, 256)))
        groups, rows = _log(rng, 1, 8), _log(rng, 1, 128)
        prefix, own_len = _log(rng, 1, 32768), _log(rng, 1, 512)
        d = shape["head_dim"]
        while groups * rows * heads * (prefix + own_len) * d > 64 * 32 * 16640 * 128:
            groups, rows, prefix = max(1, groups - 1), max(1, rows * 3 // 4), max(1, prefix * 3 // 4)
        while groups * kvh * prefix * d > 8 * 16384 * 128:
            prefix = prefix * 3 // 4
        while groups * rows * kvh * own_len * d > 64 * 8 * 256 * 128:
            own_len = own_len * 3 // 4
        return _prefix(shape, groups, rows, prefix, own_len)
    if op == "select":
        groups, beams = _log(rng, 1, 32), _log(rng, 1, 16)
        vocab = _log(rng, 1000, 151936)
        while groups * beams * vocab > 32 * 8 * 128256:
            groups = max(1, groups // 2)
        return _select(groups, beams, vocab, rng.choice((beams, 2 * beams)), rng.random() < 0.2,
                       rng.random() < 0.4, rng.random() < 0.4)
    layers, d = rng.randint(1, 32), rng.choice((64, 128))
    groups, beams, length = _log(rng, 1, 8), rng.randint(2, 16), _log(rng, 1, 256)
    while layers * kvh * d * groups * beams * (length + 64) > 32 * 8 * 128 * 32 * 128:
        layers, groups, length = max(1, layers * 3 // 4), max(1, groups - 1), max(1, length * 3 // 4)
    return _reorder(layers, kvh, d, groups, beams, length)


# ---- inputs, from the seed alone ------------------------------------------


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _lengths(r, n, most, least):
    """Ragged lengths up to `most`, the first one `most`."""
    return [most] + [r.randint(min(least, most), most) for _ in range(n - 1)]


def _frequencies(rotary, scaled):
    """Rotations a position, of a base of 500000; scaled: the long wavelengths by a factor of 8,
    the short ones not at all, those between in part."""
    f = 500000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    if scaled:
        mix = ((8192 * f / (2 * math.pi) - 1.0) / 3.0).clamp(0.0, 1.0)
        f = f * mix + f / 8.0 * (1.0 - mix)
    return f


def _parents(r, beams):
    """Which beam each one continues: two thirds of them go on from another one, and half as
    many are gone on from."""
    out = list(range(beams))
    moved = r.sample(out, max(1, beams - beams // 3))
    best = r.sample(range(beams), max(2, (len(moved) + 1) // 2))
    for i, m in enumerate(moved):
        a, b = best[i % len(best)], best[(i + 1) % len(best)]
        out[m] = b if a == m else a
    return out


def prepare(case, seed):
    g, r, op = _gen(seed), random.Random(int(seed)), case["op"]
    st = dict(case=case)
    if op == "rope":
        n, h, kvh, d = (case[f] for f in ("tokens", "heads", "kv_heads", "head_dim"))
        # the projections' output: queries, keys and values of a token side by side
        st["qkv"] = 1.5 * _normal(g, n, (h + 2 * kvh) * d)
        st["inv_freq"] = _frequencies(case["rotary"], case["scaled"])
        if case["norm"]:
            st["qw"], st["kw"] = (1.0 + 0.2 * _normal(g, d) for _ in range(2))
        if case["append"]:
            lens = _lengths(r, n, case["append"] - 1, 0)
            rows = (case["append"] + 63) // 64 * 64
            st["at"] = _ints(lens)
            st["positions"] = case["start"] + st["at"].long()
            st["k"], st["v"] = (_normal(g, n, kvh, rows, d) for _ in range(2))
        else:
            st["positions"] = torch.arange(case["start"], case["start"] + n, device="cuda")
        return st
    if op == "prefix":
        s, n, h, kvh, d = (case[f] for f in ("groups", "rows", "heads", "kv_heads", "head_dim"))
        st["q"] = 2.0 * _normal(g, s, n, h, d)
        p = (case["prefix"] + 63) // 64 * 64      # the caches' positions, some of them free
        st["kp"], st["vp"] = (_normal(g, s, kvh, p, d) for _ in range(2))
        p = (case["own_len"] + 63) // 64 * 64
        st["k"], st["v"] = (_normal(g, s, n, kvh, p, d) for _ in range(2))
        lens = _lengths(r, s, case["prefix"], case["prefix"] // 4)
        st["prefix_len"] = _ints(lens) if s > 1 else lens[0]
        st["own_len"] = _ints([_lengths(r, n, case["own_len"], case["own_len"] // 8)
                               for _ in range(s)])
        return st
    if op == "select":
        s, b, v = case["groups"], case["beams"], case["vocab"]
        x = 3.0 * _normal(g, s, b, v)
        # a few tokens stand out, as a model's choices do
        x.scatter_add_(2, torch.randint(0, v, (s, b, 8), device="cuda", generator=g),
                       8.0 * torch.rand((s, b, 8), device="cuda", generator=g))
        st["scores"] = -3.0 * torch.rand((s, b), device="cuda", generator=g).cumsum(-1)
        if case["first"]:      # the prompt's last token, the same for every beam
            x = x[:, :1].expand(s, b, v).contiguous()
            st["scores"][:, 1:] = -math.inf
            st["scores"][:, 0] = 0.0
        if case["masked"]:
            x.masked_fill_(torch.rand((s, 1, v), device="cuda", generator=g) < 0.3, -math.inf)
        st["logits"], st["eos"] = x, v - 3
        if case["ended"]:
            st["ended"] = torch.rand((s, b), device="cuda", generator=g) < 0.2
        return st
    s, b = case["groups"], case["beams"]
    st["beams"] = _ints([_parents(r, b) for _ in range(s)], torch.int64)
    st["length"] = _ints([[n] * b for n in _lengths(r, s, case["length"], case["length"] // 4)])
    rows = (case["length"] + 64) // 64 * 64
    # the layers' caches, each a view of one allocation
    shape = (case["layers"], s, b, case["kv_heads"], rows, case["head_dim"])
    st["caches"] = _normal(g, *shape), _normal(g, *shape)
    st["k"], st["v"] = (list(c.unbind(0)) for c in st["caches"])
    return st


def _split(st):
    """The fused projections' queries, keys and values, as views."""
    c = st["case"]
    n, h, kvh, d = (c[f] for f in ("tokens", "heads", "kv_heads", "head_dim"))
    return (t.view(n, -1, d) for t in st["qkv"].split((h * d, kvh * d, kvh * d), -1))


# ---- the plain forms --------------------------------------------------------


def _plain_rotate(x, weight, cos, sin, interleaved):
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight
    half = cos.shape[-1]
    r, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (r[..., ::2], r[..., 1::2]) if interleaved else (r[..., :half], r[..., half:])
    a, b = a * cos - b * sin, b * cos + a * sin
    r = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((r, rest), -1)


def _plain_rope(st):
    c = st["case"]
    q, k, v = _split(st)
    angle = (st["positions"].double().unsqueeze(-1) * st["inv_freq"]).unsqueeze(1)
    cos, sin = angle.cos().float(), angle.sin().float()
    q = _plain_rotate(q.float(), st.get("qw"), cos, sin, c["interleaved"])
    k = _plain_rotate(k.float(), st.get("kw"), cos, sin, c["interleaved"])
    if not c["append"]:
        return q, k
    row, at = torch.arange(c["tokens"], device=q.device), st["at"].long()
    st["k"][row, :, at] = k
    st["v"][row, :, at] = v
    return q, st["k"], st["v"]


def _plain_prefix(st):
    q, kp, vp, k, v = (st[f].float() for f in ("q", "kp", "vp", "k", "v"))
    s, n, h, d = q.shape
    kvh = kp.shape[1]
    x = q.reshape(s, n, kvh, h // kvh, d).permute(0, 2, 1, 3, 4)         # [s, kvh, n, g, d]
    scale = 1.0 / math.sqrt(d)
    a = (x.reshape(s, kvh, -1, d) @ kp.transpose(-1, -2)).reshape(*x.shape[:-1], -1) * scale
    mine = x.transpose(1, 2)                                             # [s, n, kvh, g, d]
    b = (mine @ k.transpose(-1, -2)).transpose(1, 2) * scale             # [s, kvh, n, g, own]
    at = torch.arange(a.shape[-1], device=q.device)
    if s > 1:
        a = a.masked_fill(at >= st["prefix_len"].view(s, 1, 1, 1, 1), -math.inf)
    else:
        a = a.masked_fill(at >= st["prefix_len"], -math.inf)
    at = torch.arange(b.shape[-1], device=q.device)
    b = b.masked_fill(at >= st["own_len"].view(s, 1, n, 1, 1), -math.inf)
    top = torch.maximum(a.amax(-1, keepdim=True), b.amax(-1, keepdim=True))
    top = torch.where(top == -math.inf, 0.0, top)
    a, b = torch.exp(a - top), torch.exp(b - top)
    total = (a.sum(-1, keepdim=True) + b.sum(-1, keepdim=True)).clamp(min=1e-30)
    o = (a.reshape(s, kvh, -1, a.shape[-1]) @ vp).reshape(x.shape)
    o = (o + (b.transpose(1, 2) @ v).transpose(1, 2)) / total
    return o.permute(0, 2, 1, 3, 4).reshape(s, n, h, d)


def _plain_select(st):
    x, c = st["logits"].double(), st["case"]
    s, b, v = x.shape
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    y = x - (torch.exp(x - top).sum(-1, keepdim=True).log() + top)
    y = y + st["scores"].double().unsqueeze(-1)
    if c["ended"]:
        last = torch.full_like(y, -math.inf)
        last[..., st["eos"]] = st["scores"].double()
        y = torch.where(st["ended"].unsqueeze(-1), last, y)
    y = y.reshape(s, b * v)
    y = torch.where(torch.isnan(y), -math.inf, y)
    at = torch.arange(b * v, device=y.device)
    values, index = [], []
    for _ in range(c["k"]):      # one after the other: ties go to the lowest index
        best = y.amax(-1, keepdim=True)
        i = torch.where(y == best, at, b * v).amin(-1, keepdim=True)
        y = y.scatter(1, i, -math.inf)
        values.append(best)
        index.append(torch.where(best == -math.inf, -1, i))
    values, index = torch.cat(values, -1), torch.cat(index, -1)
    none = index < 0
    return (values.float(), torch.where(none, -1, index % v),
            torch.where(none, -1, torch.div(index, v, rounding_mode="floor")))


def _plain_reorder(st):
    beams, length = st["beams"], st["length"]
    s, b = beams.shape
    n = st["case"]["length"]
    group = torch.arange(s, device=beams.device).unsqueeze(-1)
    at = torch.arange(n, device=beams.device)
    real = (at < length.gather(1, beams).unsqueeze(-1)).view(s, b, 1, n, 1)
    for c in (*st["k"], *st["v"]):
        rows = c[:, :, :, :n]
        c[:, :, :, :n] = torch.where(real, rows[group, beams], rows)


# ---- one pass -----------------------------------------------------------------


def run(st):
    c, op = st["case"], st["case"]["op"]
    if not own:
        if op == "rope":
            return _plain_rope(st)
        if op == "prefix":
            return _plain_prefix(st)
        if op == "select":
            return _plain_select(st)
        _plain_reorder(st)
        return st["caches"]
    import torchburn_amd as tb
    if op == "rope":
        q, k, v = _split(st)
        how = dict(q_weight=st.get("qw"), k_weight=st.get("kw"), eps=1e-6,
                   interleaved=c["interleaved"])
        if not c["append"]:
            return tb.norm_rope(q, k, st["positions"], st["inv_freq"], **how)
        q = tb.norm_rope_append(q, k, v, st["positions"], st["inv_freq"], st["k"], st["v"],
                                st["at"], **how)
        return q, st["k"], st["v"]
    if op == "prefix":
        return tb.prefix_attention(st["q"], st["kp"], st["vp"], st["prefix_len"], st["k"], st["v"],
                                   st["own_len"])
    if op == "select":
        return tb.beam_select(st["logits"], st["scores"], k=c["k"], finished=st.get("ended"),
                              eos=st["eos"])
    tb.beam_reorder(st["beams"], st["k"], st["v"], st["length"])
    return st["caches"]


def work(case):
    op = case["op"]
    if op == "rope":
        n, h, kvh, d = (case[f] for f in ("tokens", "heads", "kv_heads", "head_dim"))
        heads = h + (2 if case["append"] else 1) * kvh
        return dict(bytes=8 * n * heads * d + 8 * n + 4 * case["rotary"],
                    flops=n * (h + kvh) * (3 * case["rotary"] + (4 * d if case["norm"] else 0)))
    if op == "prefix":
        s, n, h, kvh, d = (case[f] for f in ("groups", "rows", "heads", "kv_heads", "head_dim"))
        # lengths are spread evenly from a share of the longest on
        mean = (case["prefix"] + (s - 1) * case["prefix"] * 5 / 8) / s
        mine = (case["own_len"] + (n - 1) * case["own_len"] * 9 / 16) / n
        return dict(bytes=int(8 * s * d * (n * h + kvh * (mean + n * mine))),
                    flops=int(4 * s * n * h * (mean + mine) * d))
    if op == "select":
        n = case["groups"] * case["beams"] * case["vocab"]
        return dict(bytes=4 * n + 20 * case["groups"] * case["k"], flops=3 * n)
    s, b, n = case["groups"], case["beams"], case["length"]
    moved = max(1, b - b // 3)
    row = case["layers"] * case["kv_heads"] * case["head_dim"] * 4 * 2      # K and V
    mean = (n + (s - 1) * n * 5 / 8) / s
    return dict(bytes=int(row * s * mean * (moved + max(2, (moved + 1) // 2))), flops=s * b)


# ---- the operators' definitions, in 64 bits ------------------------------------


def exact(case, seed):
    st, op = prepare(case, seed), case["op"]
    if op == "rope":
        n, h, kvh, d = (case[f] for f in ("tokens", "heads", "kv_heads", "head_dim"))
        x = st["qkv"].double().reshape(n, h + 2 * kvh, d)
        if case["norm"]:
            scale = (x.square().sum(-1, keepdim=True) / d + 1e-6).sqrt()
            w = torch.cat((st["qw"].expand(h, d), st["kw"].expand(kvh, d))).double()
            x[:, :h + kvh] = x[:, :h + kvh] / scale[:, :h + kvh] * w
        half = case["rotary"] // 2
        # a pair is a complex number, turned by its angle
        turn = st["positions"].double().reshape(n, 1, 1) * st["inv_freq"]
        turn = torch.polar(torch.ones_like(turn), turn)
        at = torch.arange(half, device=x.device)
        re, im = (2 * at, 2 * at + 1) if case["interleaved"] else (at, at + half)
        z = torch.complex(x[:, :h + kvh][..., re], x[:, :h + kvh][..., im]) * turn
        x[:, :h + kvh, re], x[:, :h + kvh, im] = z.real, z.imag
        q, k, v = x[:, :h], x[:, h:h + kvh], x[:, h + kvh:]
        if not case["append"]:
            return q, k
        kc, vc = st["k"].double(), st["v"].double()
        for i, j in enumerate(st["at"].tolist()):
            kc[i, :, j], vc[i, :, j] = k[i], v[i]
        return q, kc, vc
    if op == "prefix":
        q = st["q"].double()
        s, n, h, d = q.shape
        group = h // case["kv_heads"]
        lens = st["prefix_len"].tolist() if s > 1 else [st["prefix_len"]]
        mine = st["own_len"].tolist()
        out = torch.zeros_like(q)
        for i in range(s):
            for j in range(case["kv_heads"]):
                heads = slice(j * group, (j + 1) * group)
                kp, vp = (st[f][i, j, :lens[i]].double() for f in ("kp", "vp"))
                shared = q[i, :, heads] @ kp.T / d ** 0.5
                for t in range(n):
                    k, v = (st[f][i, t, j, :mine[i][t]].double() for f in ("k", "v"))
                    w = torch.cat((shared[t], q[i, t, heads] @ k.T / d ** 0.5), -1)
                    w = torch.softmax(w, -1)
                    out[i, t, heads] = w[:, :lens[i]] @ vp + w[:, lens[i]:] @ v
        return out
    if op == "select":
        s, b, v = st["logits"].shape
        scores, tokens, beams = [], [], []
        for i in range(s):
            y = torch.log_softmax(st["logits"][i].double(), -1) + st["scores"][i, :, None].double()
            if case["ended"]:
                for j in st["ended"][i].nonzero().flatten().tolist():
                    y[j] = -math.inf
                    y[j, st["eos"]] = float(st["scores"][i, j])
            y, order = torch.sort(y.flatten(), descending=True, stable=True)
            y, order = y[:case["k"]], order[:case["k"]]
            order = torch.where(y > -math.inf, order, -1)
            scores.append(y)
            tokens.append(torch.where(order < 0, -1, order % v))
            beams.append(torch.where(order < 0, -1, order // v))
        return torch.stack(scores), torch.stack(tokens), torch.stack(beams)
    beams, length = st["beams"].tolist(), st["length"].tolist()
    out = []
    for was in st["caches"]:
        c = was.double()
        for i, group in enumerate(beams):
            for j, p in enumerate(group):
                n = length[i][p]
                c[:, i, j, :, :n] = was[:, i, p, :, :n].double()
        out.append(c)
    return tuple(out)
