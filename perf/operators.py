"""Workloads of speculative decoding with trees of drafted tokens and with sampled requests.

A verify pass scores a tree of drafted tokens behind each of a few running sequences.  Node 0 is the token that was sampled
last, a node comes after its parent, and ``anc`` holds for each node a word whose bit ``i`` says that node ``i`` is one of its
ancestors or itself.  A case names one operator of that pass:

* ``attn``: attention of the nodes over the paged cache of their sequence and their own ancestors, with the output gate;
* ``gdn``: the gated delta rule of the nodes from their sequence's state, along their paths;
* ``tree``: which drafted path a request's own tokens take: every node's token is drawn from the target's probabilities with the
  uniform number of its depth (temperature 0: the arg-max), and the walk goes on while a child carries it;
* ``drafts``: the accepted length of a chain of drafts that were drawn from a draft model's probabilities, and the token after it;
* ``commit``: rows of the accepted path move to their places in the cache, states and convolution rings advance along it.

Weights, cached keys and values, recurrent states and logits are drawn from the seed at the magnitudes that the shapes' random-init
weights produce; the caches' pages are in random order, as in a pool that has been in use.
"""
from __future__ import annotations

import math
import random

import torch
import torch.nn.functional as F

own = False
PAGE = 64
RING = 16
TAPS = 4
DEV = "cuda"
EPS = 1e-6


# ---------------------------------------------------------------------------------------------- the cases
def _attn(rows, nodes, context, longest, heads, kv_heads, dim, pages="bf16"):
    return {"kind": "attn", "rows": rows, "nodes": nodes, "context": context, "longest": longest, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "pages": pages}


def _gdn(rows, nodes, key_heads, value_heads, dim):
    return {"kind": "gdn", "rows": rows, "nodes": nodes, "key_heads": key_heads, "value_heads": value_heads, "dim": dim}


def _tree(rows, nodes, vocab, temperature):
    return {"kind": "tree", "rows": rows, "nodes": nodes, "vocab": vocab, "temperature": temperature}


def _drafts(rows, nodes, vocab, temperature):
    return {"kind": "drafts", "rows": rows, "nodes": nodes, "vocab": vocab, "temperature": temperature}


def _commit(rows, nodes, steps, context, full_layers, linear_layers, kv_heads, dim, key_heads, value_heads, state_dim):
    return {"kind": "commit", "rows": rows, "nodes": nodes, "steps": steps, "context": context, "full_layers": full_layers,
            "linear_layers": linear_layers, "kv_heads": kv_heads, "dim": dim, "key_heads": key_heads, "value_heads": value_heads,
            "state_dim": state_dim}


def listed():
    cases = {
        # one sequence with the default three drafts in a chain, a short conversation: latency
        "attn-chain-4": _attn(1, 4, 517, 517, 16, 4, 256),
        # a full batch of sequences of very different length, small trees
        "attn-tree-16": _attn(8, 16, 517, 16391, 16, 4, 256),
        # int8 pages, six query heads a kv head
        "attn-tree-int8": _attn(4, 23, 1031, 8191, 24, 4, 256, "int8"),
        # the widest tree over long documents
        "attn-tree-64-long": _attn(2, 64, 65473, 65536, 16, 4, 256),
        # one sequence, three drafts
        "gdn-chain-4": _gdn(1, 4, 16, 32, 128),
        # a full batch of small trees
        "gdn-tree-16": _gdn(8, 16, 16, 32, 128),
        # the widest tree, the larger model's heads
        "gdn-tree-64": _gdn(4, 64, 16, 48, 128),
        # a greedy request with three drafts
        "tree-greedy-4": _tree(1, 4, 151936, 0.0),
        # sampled requests, a full batch of small trees
        "tree-sampled-16": _tree(8, 16, 151936, 0.8),
        # drafts drawn by a draft head
        "drafts-8": _drafts(8, 8, 151936, 1.0),
        # one sequence takes two of three drafts
        "commit-3": _commit(1, 4, 2, 517, 8, 24, 4, 256, 16, 32, 128),
        # every sequence of a full batch takes a path of its tree
        "commit-batch": _commit(8, 16, 5, 261, 8, 24, 4, 256, 16, 32, 128),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("attn", "attn", "gdn", "tree", "drafts", "commit"))
    if kind == "attn":
        heads, kv_heads, dim = rng.choice(((16, 4, 256), (24, 4, 256), (16, 2, 256), (8, 1, 256), (8, 2, 128), (4, 2, 64), (6, 6, 64)))
        longest = _log(rng, 1, 65536)
        nodes = _log(rng, 1, 64)
        rows = min(_log(rng, 1, 16), max(1, min(131072 // longest, (1 << 35) // (longest * nodes * heads * dim))))
        return _attn(rows, nodes, max(0, longest - _log(rng, 1, longest)) if rows > 1 else longest, longest, heads, kv_heads, dim,
                     rng.choice(("bf16", "bf16", "int8")))
    if kind == "gdn":
        key_heads, value_heads, dim = rng.choice(((16, 32, 128), (16, 48, 128), (8, 8, 128), (2, 4, 64)))
        nodes = _log(rng, 1, 64)
        return _gdn(min(_log(rng, 1, 16), max(1, 256 // nodes)), nodes, key_heads, value_heads, dim)
    if kind in ("tree", "drafts"):
        vocab = _log(rng, 300, 151936)
        nodes = _log(rng, 1 if kind == "tree" else 2, 64)
        rows = min(_log(rng, 1, 16), max(1, 128 // nodes if kind == "tree" else 64 // nodes))
        return (_tree if kind == "tree" else _drafts)(rows, nodes, vocab, rng.choice((0.0, 0.6, 1.0, 1.3)))
    nodes = _log(rng, 2, 24)
    return _commit(_log(rng, 1, 8), nodes, rng.randint(1, (nodes + 1) // 2), _log(rng, 1, 400), rng.randint(1, 8), rng.randint(1, 24),
                   *rng.choice(((4, 256, 16, 32, 128), (2, 256, 16, 32, 128), (2, 64, 2, 4, 64))))


def work(case):
    k, R, C = case["kind"], case["rows"], case["nodes"]
    if k == "attn":
        nh, nkv, hd = case["heads"], case["kv_heads"], case["dim"]
        keys = sum(_contexts(case))
        row = hd + 4 if case["pages"] == "int8" else 2 * hd
        return {"bytes": 2 * (keys + R * C) * nkv * row + 3 * R * C * nh * hd * 2, "flops": 4.0 * C * nh * hd * keys}
    if k == "gdn":
        nk, nv, d = case["key_heads"], case["value_heads"], case["dim"]
        wide = 2 * nk * d + 2 * nv * d + 2 * nv
        return {"bytes": R * nv * d * d * 4 + R * C * (wide * 2 + nv * d * 2 + nv * (2 * d + 1) * 4 + (2 * nk * d + nv * d) * 2),
                "flops": 4.0 * R * C * nv * d * d}
    if k == "tree":
        return {"bytes": R * C * case["vocab"] * 4, "flops": 2.0 * R * C * case["vocab"]}
    if k == "drafts":
        return {"bytes": R * (C + 2) * case["vocab"] * 4, "flops": 2.0 * R * (C + 2) * case["vocab"]}
    nv, d, n = case["value_heads"], case["state_dim"], case["steps"]
    conv = 2 * case["key_heads"] * d + nv * d
    return {"bytes": R * (case["linear_layers"] * (2 * nv * d * d * 4 + n * nv * (2 * d + 1) * 4 + 2 * RING * conv * 2)
                          + case["full_layers"] * (n - 1) * 4 * case["kv_heads"] * case["dim"] * 2),
            "flops": 2.0 * R * case["linear_layers"] * n * nv * d * d}


# ---------------------------------------------------------------------------------------------- inputs
def _contexts(case):
    """Tokens cached before the tree, a sequence: spread evenly over the case's range."""
    R, lo, hi = case["rows"], case["context"], case.get("longest", case["context"])
    return [hi if R == 1 else lo + (hi - lo) * r // (R - 1) for r in range(R)]


def _parents(rng, C):
    """A drafted tree: most nodes go on from a recent one, some branch off further up."""
    return [-1] + [rng.randint(max(0, j - 4), j - 1) for j in range(1, C)]


def _masks(parents):
    anc = []
    for j, p in enumerate(parents):
        anc.append((anc[p] if p >= 0 else 0) | 1 << j)
    return [a - (1 << 64) if a >> 63 else a for a in anc]


def _tables(rng, counts, extra=3):
    """Page tables of sequences whose pages lie anywhere in a pool, and the pool's pages."""
    total = sum(counts) + extra
    ids = list(range(total))
    rng.shuffle(ids)
    wide, out = max(counts), []
    for n in counts:
        out.append([ids.pop() for _ in range(n)] + [0] * (wide - n))
    return torch.tensor(out, dtype=torch.int32, device=DEV), total


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _bf(g, *shape, scale=1.0):
    return torch.empty(shape, dtype=torch.bfloat16, device=DEV).normal_(0.0, scale, generator=g)


def _f32(g, *shape, scale=1.0):
    return torch.empty(shape, dtype=torch.float32, device=DEV).normal_(0.0, scale, generator=g)


def _int8_rows(x):
    s = (x.float().abs().amax(-1) / 127).clamp_min(1e-8)
    return (x.float() / s.unsqueeze(-1)).round_().clamp_(-127, 127).to(torch.int8), s


def prepare(case, seed):
    rng, g, k = random.Random(seed), _gen(seed), case["kind"]
    R, C = case["rows"], case["nodes"]
    s = {"case": case}
    parents = [_parents(rng, C) for _ in range(R)]
    if k == "drafts":
        parents = [list(range(-1, C - 1))] * R
    s["anc"] = torch.tensor([_masks(p) for p in parents], dtype=torch.int64, device=DEV)
    if k == "attn":
        nh, nkv, hd = case["heads"], case["kv_heads"], case["dim"]
        ctx = _contexts(case)
        s["tables"], pages = _tables(rng, [-(-(n + C) // PAGE) for n in ctx])
        s["positions"] = torch.tensor(ctx, dtype=torch.int32, device=DEV)
        s["kpool"], s["vpool"] = _bf(g, pages * PAGE, nkv, hd), _bf(g, pages * PAGE, nkv, hd)
        s["kscale"] = s["vscale"] = None
        if case["pages"] == "int8":
            s["kpool"], s["kscale"] = _int8_rows(s["kpool"])
            s["vpool"], s["vscale"] = _int8_rows(s["vpool"])
        s["q"] = _bf(g, R * C, nh, hd)
        s["proj"] = _bf(g, R * C, nh * 2 * hd + 2 * nkv * hd)              # (q | gate) of each head, then k, then v
        s["out"] = torch.zeros(R * C, nh * hd, dtype=torch.bfloat16, device=DEV)
    elif k == "gdn":
        nk, nv, d = case["key_heads"], case["value_heads"], case["dim"]
        conv = 2 * nk * d + nv * d
        s["proj"] = _bf(g, R * C, conv + nv * d + 2 * nv)                 # q | k | v | z | b | a
        s["conv_w"] = _f32(g, conv, TAPS, scale=0.5)
        s["A_log"] = torch.empty(nv, device=DEV).uniform_(0.0, 2.0, generator=g)
        s["dt_bias"] = _f32(g, nv, scale=0.5) - 2.0
        s["norm_w"] = 1.0 + _f32(g, d, scale=0.1)
        s["ring"] = _bf(g, R + 1, RING, conv)
        s["state"] = _f32(g, R + 1, nv, d, d, scale=0.1)
        s["slots"] = torch.tensor(rng.sample(range(R + 1), R), dtype=torch.int32, device=DEV)
        s["positions"] = torch.tensor([rng.choice((0, 1, 2, 517, 2111, 16391)) for _ in range(R)], dtype=torch.int32, device=DEV)
        s["out"] = torch.zeros(R * C, nv * d, dtype=torch.bfloat16, device=DEV)
        s["record"] = torch.zeros(R, C, nv, 2 * d + 1, device=DEV)
        s["raw"] = torch.zeros(R, C, conv, dtype=torch.bfloat16, device=DEV)
    elif k in ("tree", "drafts"):
        V, T = case["vocab"], case["temperature"]
        s["logits"] = _f32(g, R, C, V, scale=3.0)
        s["temperature"] = torch.full((R,), T, device=DEV)
        s["u"] = torch.rand(R, C, generator=g, device=DEV)
        if k == "tree":
            # most of the drafts are what the target goes on with
            picks, depth = _draws(s), _depths(s["anc"])[0]
            par = torch.tensor([[0] + p[1:] for p in parents], device=DEV)
            right = torch.rand(R, C, generator=g, device=DEV) < 0.8
            s["tokens"] = torch.where(right & (depth > 0), picks.gather(1, par), torch.randint(V, (R, C), generator=g, device=DEV))
        else:
            heat = T if T > 0 else 1.0
            s["q"] = torch.softmax((s["logits"][:, :-1] + _f32(g, R, C - 1, V, scale=0.7)) / heat, -1)
            drawn = torch.multinomial(s["q"].reshape(-1, V), 1, generator=g).reshape(R, C - 1)
            if T <= 0:
                best = s["logits"][:, :-1].argmax(-1)
                drawn = torch.where(torch.rand(R, C - 1, generator=g, device=DEV) < 0.8, best, drawn)
            s["tokens"] = torch.cat([torch.randint(V, (R, 1), generator=g, device=DEV), drawn], 1)
            s["lengths"] = torch.tensor([rng.randint(max(1, C // 2), C) for _ in range(R)], dtype=torch.int32, device=DEV)
            s["u_draw"] = torch.rand(R, generator=g, device=DEV)
    else:
        nkv, hd, nk, nv, d = (case[n] for n in ("kv_heads", "dim", "key_heads", "value_heads", "state_dim"))
        Lf, Ll, n, conv = case["full_layers"], case["linear_layers"], case["steps"], 2 * nk * d + nv * d
        ctx = [max(0, case["context"] - 7 * r) for r in range(R)]
        s["tables"], pages = _tables(rng, [-(-(c + C) // PAGE) for c in ctx])
        s["positions"] = torch.tensor(ctx, dtype=torch.int32, device=DEV)
        s["kpool"], s["vpool"] = _bf(g, Lf, pages * PAGE, nkv, hd), _bf(g, Lf, pages * PAGE, nkv, hd)
        # the accepted nodes come late among their alternatives, so that a second pass finds what the first one found
        path = [[0] + sorted(rng.sample(range(n, C), n - 1)) + [-1] * (C - n) for _ in range(R)]
        s["path"] = torch.tensor(path, dtype=torch.int32, device=DEV)
        s["steps"] = torch.full((R,), n, dtype=torch.int32, device=DEV)
        s["state"] = _f32(g, Ll, 2 * R, nv, d, d, scale=0.1)
        s["ring"] = _bf(g, Ll, 2 * R, RING, conv)
        rec = _f32(g, Ll, R, C, nv, 2 * d + 1)
        rec[..., :d] = F.normalize(rec[..., :d], dim=-1)
        rec[..., 2 * d] = torch.sigmoid(rec[..., 2 * d] + 2.0)
        s["record"] = rec
        s["raw"] = _bf(g, Ll, R, C, conv)
        ids = rng.sample(range(2 * R), 2 * R)                             # a fork: the state advances into a slot of its own
        s["slots"], s["to"] = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in (ids[:R], ids[R:]))
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _visible(anc):
    """[R, C, C] truth values: node i on the path to node j."""
    bits = torch.arange(anc.shape[1], device=anc.device)
    return (anc.unsqueeze(-1) >> bits & 1).bool()


def _depths(anc):
    on = _visible(anc)
    return on.sum(-1) - 1, on


def _rows(tables, count, start=None):
    """Pool rows of the positions ``start .. start + count`` of each sequence."""
    pos = torch.arange(count, device=tables.device).unsqueeze(0)
    if start is not None:
        pos = pos + start.long().unsqueeze(1)
    page = (pos // PAGE).clamp(max=tables.shape[1] - 1).expand(tables.shape[0], -1)
    return tables.long().gather(1, page) * PAGE + pos % PAGE


def _plain_attn(s):
    c = s["case"]
    R, C, nh, nkv, hd = c["rows"], c["nodes"], c["heads"], c["kv_heads"], c["dim"]
    rows = _rows(s["tables"], c["longest"] + C)                                              # [R, S]
    k, v = s["kpool"][rows].float(), s["vpool"][rows].float()
    if s["kscale"] is not None:
        k, v = k * s["kscale"][rows].unsqueeze(-1), v * s["vscale"][rows].unsqueeze(-1)
    S = rows.shape[1]
    node = torch.arange(S, device=DEV) - s["positions"].long().unsqueeze(1)                  # [R, S]: < 0 cached, >= C behind the tree
    on = _visible(s["anc"]).gather(2, node.clamp(0, C - 1).unsqueeze(1).expand(-1, C, -1))
    on = (node < 0).unsqueeze(1) | on & (node < C).unsqueeze(1)                              # [R, C, S]
    q = s["q"].float().reshape(R, C, nkv, nh // nkv, hd)
    x = torch.einsum("rcgmd,rsgd->rgmcs", q, k) * hd ** -0.5
    x.masked_fill_(~on.unsqueeze(1).unsqueeze(1), -math.inf)
    x = (x - x.amax(-1, keepdim=True)).exp_()
    x /= x.sum(-1, keepdim=True)
    o = torch.einsum("rgmcs,rsgd->rcgmd", x, v).reshape(R * C, nh, hd)
    gate = s["proj"][:, :nh * 2 * hd].reshape(R * C, nh, 2, hd)[:, :, 1].float()
    return (o / (1 + (-gate).exp())).reshape(R * C, nh * hd).to(torch.bfloat16)


def _tap(anc, positions, proj, ring, slots, back, conv):
    """The projection row ``back`` positions before each node on its path: a node's, an older one from the ring, or nothing."""
    R, C = anc.shape
    depth, on = _depths(anc)
    want = depth - back
    node = (on & (depth.unsqueeze(1) == want.unsqueeze(2))).long().argmax(-1)                # [R, C]
    mine = proj[:, :conv].reshape(R, C, conv).float().gather(1, node.unsqueeze(-1).expand(-1, -1, conv))
    pos = positions.long().unsqueeze(1) + want
    old = ring[slots.long().unsqueeze(1), pos % RING].float() * (pos >= 0).unsqueeze(-1)
    return torch.where((want >= 0).unsqueeze(-1), mine, old)


def _plain_gdn(s):
    c = s["case"]
    R, C, nk, nv, d = c["rows"], c["nodes"], c["key_heads"], c["value_heads"], c["dim"]
    conv = 2 * nk * d + nv * d
    anc, proj = s["anc"], s["proj"]
    depth, on = _depths(anc)
    y = sum(_tap(anc, s["positions"], proj, s["ring"], s["slots"], b, conv) * s["conv_w"][:, TAPS - 1 - b] for b in range(TAPS))
    y = y / (1 + (-y).exp())
    q, k, v = y[..., :nk * d].reshape(R, C, nk, d), y[..., nk * d:2 * nk * d].reshape(R, C, nk, d), y[..., 2 * nk * d:].reshape(R, C, nv, d)
    norm = lambda t: t / (t.square().sum(-1, keepdim=True) + 1e-6).sqrt()  # noqa: E731
    rep = nv // nk
    q, k = (norm(q) * d ** -0.5).repeat_interleave(rep, 2).transpose(1, 2), norm(k).repeat_interleave(rep, 2).transpose(1, 2)  # [R, nv, C, d]
    v = v.transpose(1, 2)
    rest = proj[:, conv:].float().reshape(R, C, -1)
    z, b, a = rest[..., :nv * d].reshape(R, C, nv, d), rest[..., nv * d:nv * d + nv], rest[..., nv * d + nv:]
    beta = (1 / (1 + (-b).exp())).transpose(1, 2).unsqueeze(-1)                              # [R, nv, C, 1]
    g = -(s["A_log"].exp() * F.softplus(a + s["dt_bias"])).transpose(1, 2)                    # [R, nv, C]
    cum = (on.unsqueeze(1) * g.unsqueeze(2)).sum(-1)                                          # log decay from the state to each node
    strict = on & ~torch.eye(C, dtype=torch.bool, device=DEV)
    fade = lambda m: torch.where(m.unsqueeze(1), cum.unsqueeze(-1) - cum.unsqueeze(-2), -math.inf).exp()  # noqa: E731
    S = s["state"][s["slots"].long()]
    t = -beta * (k @ k.transpose(-1, -2)) * fade(strict)                                      # d = t d + w
    w = beta * (v - cum.exp().unsqueeze(-1) * (k @ S))
    inv = torch.eye(C, device=DEV) + t
    for _ in range(max(0, (C - 1).bit_length() - 1)):                                        # (1 - t)^-1 = (1 + t)(1 + t^2)(1 + t^4)..
        t = t @ t
        inv = inv + inv @ t
    dl = inv @ w
    o = cum.exp().unsqueeze(-1) * (q @ S) + (q @ k.transpose(-1, -2) * fade(on)) @ dl
    o = o.transpose(1, 2)
    o = o / (o.square().mean(-1, keepdim=True) + EPS).sqrt() * s["norm_w"] * (z / (1 + (-z).exp()))
    record = torch.cat([k, dl, g.exp().unsqueeze(-1)], -1).transpose(1, 2)
    return {"out": o.reshape(R * C, nv * d).to(torch.bfloat16), "record": record, "raw": proj[:, :conv].reshape(R, C, conv).clone()}


def _weights(logits, temperature):
    """exp((logit - largest) / temperature) in 64 bits; at temperature 0 the first largest one alone."""
    x = logits.double()
    T = temperature.double()
    w = ((x - x.amax(-1, keepdim=True)) / T.where(T > 0, 1.0)).exp_()
    first = torch.zeros_like(w).scatter_(-1, logits.argmax(-1, keepdim=True), 1.0)
    return torch.where(T > 0, w, first)


def _pick(w, u):
    """First index whose running sum of ``w`` exceeds ``u`` times the whole; the last one with any weight where none does."""
    run = w.cumsum(-1)
    at = (run <= u.double().unsqueeze(-1) * run[..., -1:]).sum(-1)
    last = w.shape[-1] - 1 - (w.flip(-1) > 0).long().argmax(-1)
    return torch.minimum(at, last)


def _draws(s):
    depth = _depths(s["anc"])[0]
    return _pick(_weights(s["logits"], s["temperature"].view(-1, 1, 1)), s["u"].gather(1, depth))


def _plain_tree(s):
    anc, tokens = s["anc"], s["tokens"]
    C = anc.shape[1]
    depth, on = _depths(anc)
    picks = _draws(s)
    parent = (on & (depth.unsqueeze(1) == depth.unsqueeze(2) - 1)).long().argmax(-1)         # [R, C]
    hit = (tokens == picks.gather(1, parent)) & (depth > 0)
    twin = hit.unsqueeze(1) & hit.unsqueeze(2) & (parent.unsqueeze(1) == parent.unsqueeze(2))
    first = ~torch.tril(twin, -1).any(-1)                                                    # of equal siblings the first
    good = (hit & first) | (depth == 0)
    taken = ~(on & ~good.unsqueeze(1)).any(-1)                                               # the whole path holds
    steps = taken.sum(-1)
    order = torch.where(taken, depth, C)
    path = torch.full_like(order, -1).scatter_(1, order.argsort(1).argsort(1), torch.arange(C, device=DEV).expand_as(order))
    path = path.where(torch.arange(C, device=DEV) < steps.unsqueeze(1), -1)
    last = path.gather(1, (steps - 1).unsqueeze(1))
    return {"path": path.int(), "steps": steps.int(), "next": picks.gather(1, last).squeeze(1)}


def _plain_drafts(s):
    tokens, q, n = s["tokens"], s["q"], s["lengths"].long()
    R, C, V = s["logits"].shape
    w = _weights(s["logits"], s["temperature"].view(-1, 1, 1))
    p = w / w.sum(-1, keepdim=True)
    x = tokens[:, 1:].unsqueeze(-1)
    ok = s["u"][:, 1:].double() * q.gather(2, x).squeeze(-1).double() < p[:, :-1].gather(2, x).squeeze(-1)
    ok &= torch.arange(1, C, device=DEV) < n.unsqueeze(1)
    taken = ok.long().cumprod(1).sum(1)                                                       # drafts accepted
    row = torch.arange(R, device=DEV)
    at = p[row, taken]
    rest = (at - q[row, taken.clamp(max=C - 2)].double()).clamp_min(0.0)
    rest = torch.where(((taken < n - 1) & (rest.sum(-1) > 0)).unsqueeze(1), rest, at)
    return {"steps": (taken + 1).int(), "next": _pick(rest, s["u_draw"])}


def _plain_commit(s):
    R, n = s["path"].shape[0], s["case"]["steps"]
    path, pos = s["path"][:, :n].long(), s["positions"]
    C = s["path"].shape[1]
    rows = _rows(s["tables"], C, pos)                                                         # [R, C]
    src, dst = rows.gather(1, path), rows[:, :n]
    for pool in (s["kpool"], s["vpool"]):
        pool[:, dst] = pool[:, src]
    L, d = s["state"].shape[0], s["state"].shape[-1]
    rec = s["record"].gather(2, path.view(1, R, n, 1, 1).expand(L, -1, -1, *s["record"].shape[3:]))       # [L, R, n, nv, 2d + 1]
    alpha = rec[..., 2 * d].log()
    later = (alpha.sum(2, keepdim=True) - alpha.cumsum(2)).exp()
    new = s["state"][:, s["slots"].long()] * alpha.sum(2).exp().unsqueeze(-1).unsqueeze(-1)
    new += torch.einsum("lrnhk,lrnhv->lrhkv", rec[..., :d] * later.unsqueeze(-1), rec[..., d:2 * d])
    s["state"][:, s["to"].long()] = new
    ring = s["ring"][:, s["slots"].long()]
    last = pos.long() + n - 1
    place = last.unsqueeze(1) - (last.unsqueeze(1) - torch.arange(RING, device=DEV)) % RING     # position behind each entry
    step = place - pos.long().unsqueeze(1)                                                     # [R, RING]
    node = path.gather(1, step.clamp(0, n - 1))
    fresh = s["raw"].gather(2, node.view(1, R, RING, 1).expand(L, -1, -1, ring.shape[-1]))
    s["ring"][:, s["to"].long()] = torch.where((step >= 0).view(1, R, RING, 1), fresh, ring)
    return {"k": s["kpool"], "v": s["vpool"], "state": s["state"], "ring": s["ring"]}


def run(state):
    s, c = state, state["case"]
    k = c["kind"]
    if not own:
        return {"attn": _plain_attn, "gdn": _plain_gdn, "tree": _plain_tree, "drafts": _plain_drafts, "commit": _plain_commit}[k](s)
    from coffin_b200.ops import tree
    if k == "attn":
        return tree.attn_tree(s["q"], s["proj"], s["kpool"], s["vpool"], s["tables"], s["positions"], s["anc"], s["out"], nh=c["heads"],
                              nkv=c["kv_heads"], hd=c["dim"], kscale=s["kscale"], vscale=s["vscale"])
    if k == "gdn":
        tree.gdn_tree(s["proj"], s["conv_w"], s["A_log"], s["dt_bias"], s["norm_w"], s["ring"], s["state"], s["slots"], s["positions"],
                      s["anc"], s["out"], s["record"], s["raw"], nk=c["key_heads"], nv=c["value_heads"], dk=c["dim"], dv=c["dim"], eps=EPS)
        return {"out": s["out"], "record": s["record"], "raw": s["raw"]}
    if k == "tree":
        path, steps, nxt = tree.verify_tree(s["logits"], s["tokens"], s["anc"], s["temperature"], s["u"])
        return {"path": path, "steps": steps, "next": nxt}
    if k == "drafts":
        steps, nxt = tree.verify_drafts(s["logits"], s["tokens"], s["lengths"], s["q"], s["temperature"], s["u"], s["u_draw"])
        return {"steps": steps, "next": nxt}
    tree.kv_tree_commit(s["kpool"], s["vpool"], s["tables"], s["positions"], s["path"], s["steps"])
    tree.gdn_tree_commit(s["state"], s["ring"], s["record"], s["raw"], s["slots"], s["positions"], s["path"], s["steps"], to_slots=s["to"])
    return {"k": s["kpool"], "v": s["vpool"], "state": s["state"], "ring": s["ring"]}


# ---------------------------------------------------------------------------------------------- the definitions, in 64 bits
def _nodes_above(word, j):
    """Nodes on the path to node j, the root first."""
    return [i for i in range(j + 1) if word >> i & 1]


def _exact_attn(s):
    c = s["case"]
    R, C, nh, nkv, hd = c["rows"], c["nodes"], c["heads"], c["kv_heads"], c["dim"]
    out = torch.empty(R, C, nh, hd, dtype=torch.float64, device=DEV)
    gate = s["proj"].double()[:, :nh * 2 * hd].reshape(R, C, nh, 2 * hd)[..., hd:]
    for r, n in enumerate(_contexts(c)):
        at = torch.arange(n + C, device=DEV)
        rows = s["tables"][r].long()[at // PAGE] * PAGE + at % PAGE
        words = s["anc"][r].tolist()
        hide = torch.zeros(C, n + C, dtype=torch.bool)
        for j in range(C):
            hide[j, n:] = True
            hide[j, [n + i for i in _nodes_above(words[j], j)]] = False
        hide = hide.to(DEV)
        for h in range(nh):
            g = h * nkv // nh
            k, v = s["kpool"][rows, g].double(), s["vpool"][rows, g].double()
            if s["kscale"] is not None:
                k, v = k * s["kscale"][rows, g].double()[:, None], v * s["vscale"][rows, g].double()[:, None]
            x = s["q"].reshape(R, C, nh, hd)[r, :, h].double() @ k.T / math.sqrt(hd)
            out[r, :, h] = torch.softmax(x.masked_fill(hide, -math.inf), -1) @ v
    return (out * torch.sigmoid(gate)).reshape(R * C, nh * hd)


def _exact_gdn(s):
    c = s["case"]
    R, C, nk, nv, d = c["rows"], c["nodes"], c["key_heads"], c["value_heads"], c["dim"]
    conv = 2 * nk * d + nv * d
    proj = s["proj"].double().reshape(R, C, -1)
    out = torch.empty(R, C, nv, d, dtype=torch.float64, device=DEV)
    rec = torch.empty(R, C, nv, 2 * d + 1, dtype=torch.float64, device=DEV)
    for r in range(R):
        slot, pos = int(s["slots"][r]), int(s["positions"][r])
        past = {p: s["ring"][slot, p % RING].double() for p in range(max(0, pos - TAPS + 1), pos)}
        states, words = {}, s["anc"][r].tolist()
        for j in range(C):
            up = _nodes_above(words[j], j)
            line = {**past, **{pos + i: proj[r, m, :conv] for i, m in enumerate(up)}}
            at = pos + len(up) - 1
            x = sum(line[at - b] * s["conv_w"][:, TAPS - 1 - b].double() for b in range(TAPS) if at - b in line)
            x = x * torch.sigmoid(x)
            q, k, v = x[:nk * d].view(nk, d), x[nk * d:2 * nk * d].view(nk, d), x[2 * nk * d:].view(nv, d)
            q = (q / torch.sqrt((q * q).sum(-1, keepdim=True) + 1e-6) / math.sqrt(d)).repeat_interleave(nv // nk, 0)
            k = (k / torch.sqrt((k * k).sum(-1, keepdim=True) + 1e-6)).repeat_interleave(nv // nk, 0)
            z, b, a = proj[r, j, conv:conv + nv * d].view(nv, d), proj[r, j, conv + nv * d:conv + nv * d + nv], proj[r, j, conv + nv * d + nv:]
            t = a + s["dt_bias"].double()
            alpha = torch.exp(-torch.exp(s["A_log"].double()) * torch.logaddexp(t, torch.zeros_like(t)))
            S = (states[up[-2]] if len(up) > 1 else s["state"][slot].double()) * alpha[:, None, None]
            delta = torch.sigmoid(b)[:, None] * (v - torch.einsum("hkv,hk->hv", S, k))
            S = states[j] = S + k[:, :, None] * delta[:, None, :]
            o = torch.einsum("hkv,hk->hv", S, q)
            o = o / torch.sqrt((o * o).mean(-1, keepdim=True) + EPS) * s["norm_w"].double()
            out[r, j] = o * z * torch.sigmoid(z)
            rec[r, j] = torch.cat([k, delta, alpha[:, None]], -1)
    return {"out": out.reshape(R * C, nv * d), "record": rec, "raw": proj[:, :, :conv]}


def _prob(logits, T):
    if T <= 0:
        p = torch.zeros(logits.shape[0], dtype=torch.float64, device=DEV)
        p[int((logits == logits.max()).nonzero()[0])] = 1.0
        return p
    return torch.softmax(logits.double() / T, 0)


def _choose(p, u):
    run = torch.cumsum(p, 0)
    at = int(torch.searchsorted(run, u * run[-1], right=True))
    return min(at, int(p.nonzero()[-1]))


def _exact_tree(s):
    T, C = float(s["temperature"][0]), s["anc"].shape[1]
    paths, steps, nxt = [], [], []
    for r in range(s["anc"].shape[0]):
        words, toks = s["anc"][r].tolist(), s["tokens"][r].tolist()
        above = [_nodes_above(w, j) for j, w in enumerate(words)]
        path = [0]
        while True:
            t = _choose(_prob(s["logits"][r, path[-1]], T), s["u"][r, len(path) - 1].double())
            on = [j for j in range(C) if len(above[j]) == len(path) + 1 and above[j][-2] == path[-1] and toks[j] == t]
            if not on:
                break
            path.append(on[0])
        paths.append(path + [-1] * (C - len(path)))
        steps.append(len(path))
        nxt.append(t)
    return {"path": torch.tensor(paths, dtype=torch.int32), "steps": torch.tensor(steps, dtype=torch.int32), "next": torch.tensor(nxt)}


def _exact_drafts(s):
    T, steps, nxt = float(s["temperature"][0]), [], []
    for r in range(s["tokens"].shape[0]):
        n, i, toks = int(s["lengths"][r]), 0, s["tokens"][r].tolist()
        while True:
            p = _prob(s["logits"][r, i], T)
            if i == n - 1:
                break
            q, x = s["q"][r, i].double(), toks[i + 1]
            if float(s["u"][r, i + 1]) * float(q[x]) < float(p[x]):
                i += 1
                continue
            left = torch.clamp(p - q, min=0)
            p = left if float(left.sum()) > 0 else p
            break
        steps.append(i + 1)
        nxt.append(_choose(p, s["u_draw"][r].double()))
    return {"steps": torch.tensor(steps, dtype=torch.int32), "next": torch.tensor(nxt)}


def _exact_commit(s):
    k, v, state, ring = s["kpool"].clone(), s["vpool"].clone(), s["state"].double(), s["ring"].clone()
    d = state.shape[-1]
    for r in range(s["path"].shape[0]):
        pos, n, a, b = (int(s[m][r]) for m in ("positions", "steps", "slots", "to"))
        table, path = s["tables"][r].tolist(), s["path"][r].tolist()
        row = lambda p: table[p // PAGE] * PAGE + p % PAGE  # noqa: E731
        S = state[:, a].clone()
        ring[:, b] = s["ring"][:, a]
        for i in range(n):
            k[:, row(pos + i)], v[:, row(pos + i)] = s["kpool"][:, row(pos + path[i])], s["vpool"][:, row(pos + path[i])]
            rec = s["record"][:, r, path[i]].double()
            S = S * rec[..., 2 * d, None, None] + rec[..., :d, None] * rec[..., None, d:2 * d]
            ring[:, b, (pos + i) % RING] = s["raw"][:, r, path[i]]
        state[:, b] = S
    return {"k": k, "v": v, "state": state, "ring": ring}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "gdn": _exact_gdn, "tree": _exact_tree, "drafts": _exact_drafts, "commit": _exact_commit}[case["kind"]](s)
