"""Plain 64-bit forms of the tree operators, node by node, and first-order bounds of what 32-bit arithmetic may be off by."""
import math

import torch

PAGE, RING = 64, 16
U32 = 2.0 ** -24          # half a step of fp32
UBF = 2.0 ** -8           # half a step of bf16


def random_parents(rng, C, kind="tree"):
    if kind == "chain":
        return list(range(-1, C - 1))
    if kind == "star":
        return [-1] + [0] * (C - 1)
    return [-1] + [rng.randint(max(0, j - 4), j - 1) for j in range(1, C)]


def path_of(parents, j):
    out = []
    while j >= 0:
        out.append(j)
        j = parents[j]
    return out[::-1]


def slots_of(table, positions):
    return [int(table[p // PAGE]) * PAGE + p % PAGE for p in positions]


def attn(q, gate, kpool, vpool, kscale, vscale, tables, positions, parents, nkv):
    """(outputs, bound): ``q [R, C, nh, hd]``, ``gate`` the same or None, ``parents`` a list a sequence (None: unused; entry None: no node).
    Weights are rounded to bf16 (half a step each, against their exact sum), and the result once more."""
    R, C, nh, hd = q.shape
    out = torch.zeros(R, C, nh, hd, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for r in range(R):
        if parents[r] is None:
            continue
        pos0 = int(positions[r])
        for j in range(C):
            if parents[r][j] is None:
                continue
            rows = slots_of(tables[r], list(range(pos0)) + [pos0 + i for i in path_of(parents[r], j)])
            rows = torch.tensor(rows, device=q.device)
            k, v = kpool[rows].double(), vpool[rows].double()
            if kscale is not None:
                k, v = k * kscale[rows].double().unsqueeze(-1), v * vscale[rows].double().unsqueeze(-1)
            k, v = (t.repeat_interleave(nh // nkv, 1) for t in (k, v))
            s = torch.einsum("hd,shd->hs", q[r, j].double(), k) / math.sqrt(hd)
            p = torch.softmax(s, -1)
            out[r, j] = torch.einsum("hs,shd->hd", p, v)
            mean_abs = torch.einsum("hs,shd->hd", p, v.abs())
            # scores: products of hd terms in fp32, |ds| <= hd 2^-24 sum |q k|; a weight moves by as much relatively
            ds = (hd + 8) * U32 * torch.einsum("hd,shd->hs", q[r, j].double().abs(), k.abs()).amax(-1) / math.sqrt(hd)
            bound[r, j] = mean_abs * (UBF + 2 * ds.unsqueeze(-1) + (len(rows) + 64) * U32)
    if gate is not None:
        g = torch.sigmoid(gate.double())
        out, bound = out * g, bound * g + out.abs() * g * 2.0 ** -20
    return out, bound + out.abs() * UBF


def gdn(proj, conv_w, A_log, dt_bias, norm_w, ring, state, slots, positions, parents, nk, nv, dk, dv, eps, gate_sigmoid=False):
    """dict of 64-bit results and bounds; ``proj [R, C, width]``."""
    R, C, _ = proj.shape
    conv, dev = 2 * nk * dk + nv * dv, proj.device
    f64 = dict(dtype=torch.float64, device=dev)
    res = {"out": torch.zeros(R, C, nv, dv, **f64), "record": torch.zeros(R, C, nv, dk + dv + 1, **f64), "raw": proj[..., :conv].clone()}
    res["out_bound"], res["record_bound"] = torch.zeros_like(res["out"]), torch.zeros_like(res["record"])
    n_eps = (2 * dk + C + 64) * U32                  # conv, SiLU, norm and the products: at most so many roundings a term
    for r in range(R):
        if parents[r] is None:
            continue
        slot, pos0 = int(slots[r]), int(positions[r])
        S0 = state[slot].double()
        nodes = {}
        for j in range(C):
            if parents[r][j] is None:
                continue
            path = path_of(parents[r], j)
            lines = [ring[slot, p % RING].double() for p in range(max(0, pos0 - 3), pos0)] + [proj[r, i, :conv].double() for i in path]
            lines = [torch.zeros(conv, **f64)] * max(0, 4 - len(lines)) + lines[-4:]
            x = sum(lines[t] * conv_w[:, t].double() for t in range(4))
            # a channel where its four terms cancel is off by as much as they are large; SiLU's slope is at most 1.1
            xe = 1.1 * sum(lines[t].abs() * conv_w[:, t].double().abs() for t in range(4)) * 8 * U32
            x = x * torch.sigmoid(x)
            q, k, v = x[:nk * dk].view(nk, dk), x[nk * dk:2 * nk * dk].view(nk, dk), x[2 * nk * dk:].view(nv, dv)
            qe, ke, ve = xe[:nk * dk].view(nk, dk), xe[nk * dk:2 * nk * dk].view(nk, dk), xe[2 * nk * dk:].view(nv, dv)
            rep = nv // nk

            def unit(t, e, scale):
                n = torch.sqrt((t * t).sum(-1, keepdim=True) + 1e-6)
                err = e / n + t.abs() / n * ((t.abs() * e).sum(-1, keepdim=True) / n ** 2 + (dk + 8) * U32)
                return (t / n * scale).repeat_interleave(rep, 0), (err * scale).repeat_interleave(rep, 0)

            q, qe = unit(q, qe, dk ** -0.5)
            k, ke = unit(k, ke, 1.0)
            rest = proj[r, j, conv:].double()
            z, b, a = rest[:nv * dv].view(nv, dv), rest[nv * dv:nv * dv + nv], rest[nv * dv + nv:nv * dv + 2 * nv]
            beta = torch.sigmoid(b)
            g = -torch.exp(A_log.double()) * torch.nn.functional.softplus(a + dt_bias.double(), threshold=1e9)
            up = [nodes[i] for i in path[:-1]]
            c = g + (up[-1]["c"] if up else 0)
            dec = torch.exp(c)
            slack = lambda cc: n_eps + 8 * U32 * cc.abs()          # noqa: E731  a decay exp(c) is off by the roundings of its exponent

            def from_state(x_, e_):
                val = dec[:, None] * torch.einsum("hk,hkv->hv", x_, S0)
                mag = dec[:, None] * torch.einsum("hk,hkv->hv", x_.abs(), S0.abs())
                return val, mag * slack(c)[:, None] + dec[:, None] * torch.einsum("hk,hkv->hv", e_, S0.abs())

            def from_node(m, x_, e_):
                f = torch.exp(c - m["c"])
                dot = f * (x_ * m["k"]).sum(-1)
                de = f * ((x_.abs() * m["k"].abs()).sum(-1) * slack(c - m["c"]) + (e_ * m["k"].abs()).sum(-1) + (x_.abs() * m["ke"]).sum(-1))
                return dot[:, None] * m["d"], de[:, None] * m["d"].abs() + dot.abs()[:, None] * m["de"]

            w, we = from_state(k, ke)
            d, de = v - w, ve + we + (v.abs() + w.abs()) * n_eps
            for m in up:
                t, te = from_node(m, k, ke)
                d, de = d - t, de + te + t.abs() * n_eps
            d, de = beta[:, None] * d, beta[:, None] * (de + d.abs() * n_eps)
            me = nodes[j] = {"c": c, "k": k, "ke": ke, "d": d, "de": de}
            o, oe = from_state(q, qe)
            for m in up + [me]:
                t, te = from_node(m, q, qe)
                o, oe = o + t, oe + te + t.abs() * n_eps
            rms = torch.sqrt((o * o).mean(-1, keepdim=True) + eps)
            gate = torch.sigmoid(z) if gate_sigmoid else z * torch.sigmoid(z)
            f = norm_w.double() * gate / rms
            out = o * f
            res["out"][r, j] = out
            res["out_bound"][r, j] = oe * f.abs() + out.abs() * ((o.abs() * oe).mean(-1, keepdim=True) / rms ** 2 + (dv + 64) * U32) + out.abs() * UBF
            res["record"][r, j] = torch.cat([k, d, torch.exp(g)[:, None]], -1)
            res["record_bound"][r, j] = torch.cat([ke, de, (torch.exp(g) * (8 * g.abs() + 4) * U32)[:, None]], -1)
    for key in ("out_bound", "record_bound"):
        res[key] = res[key] * 1.01 + 1e-30           # second-order terms
    return res


def probs(logits, T):
    x = logits.double()
    if T <= 0:
        p = torch.zeros_like(x)
        p[int((logits == logits.max()).nonzero()[0])] = 1.0
        return p
    w = torch.where(logits == logits.max(), torch.zeros_like(x), x - x.max())
    return torch.softmax(w / T, 0)


def choose(p, u):
    """(first index with a running sum above u, how near the border is)."""
    run = torch.cumsum(p, 0)
    at = int(torch.searchsorted(run, torch.tensor(float(u), dtype=torch.float64, device=p.device) * run[-1], right=True))
    at = min(at, int(p.nonzero()[-1]))
    near = float((run - u * run[-1]).abs().min())
    return at, near


def walk(logits, tokens, parents, T, u):
    """(path, next, nearest border) of one tree: ``logits [C, V]``."""
    path, near = [0], 1.0
    while True:
        t, e = choose(probs(logits[path[-1]], T), float(u[len(path) - 1]))
        near = min(near, e) if T > 0 else near
        on = [j for j, p in enumerate(parents) if p == path[-1] and int(tokens[j]) == t]
        if not on:
            return path, t, near
        path.append(on[0])


def chain(logits, tokens, n, q, T, u, u_draw):
    """(tokens kept, next, nearest border) of one chain."""
    i, near = 0, 1.0
    while i < n - 1:
        p = probs(logits[i], T)
        x = int(tokens[i + 1])
        px, qx = float(p[x]), float(q[i, x])
        if T > 0:
            near = min(near, abs(float(u[i + 1]) * qx - px))
        if float(u[i + 1]) * qx < px:
            i += 1
            continue
        left = torch.clamp(p - q[i].double(), min=0)
        p = left if float(left.sum()) > 0 else p
        t, e = choose(p, float(u_draw))
        return i + 1, t, min(near, e) if T > 0 else near
    t, e = choose(probs(logits[n - 1], T), float(u_draw))
    return n, t, min(near, e) if T > 0 else near


def advance(state, record, path, dk, dv):
    """(state after the recorded updates of ``path``, bound): ``state [nv, dk, dv]``, ``record [C, nv, dk + dv + 1]``."""
    S, e = state.double(), torch.zeros_like(state, dtype=torch.float64)
    for i in path:
        rec = record[i].double()
        k, d, alpha = rec[:, :dk, None], rec[:, None, dk:dk + dv], rec[:, dk + dv, None, None]
        e = alpha.abs() * e + ((alpha * S).abs() + (k * d).abs()) * 3 * U32
        S = alpha * S + k * d
        e = e + S.abs() * U32
    return S, e * 1.01 + 1e-30
