"""Tree verification operators against 64-bit forms, node by node, with bounds from the roundings they make."""
import random

import pytest
import torch

import plain_tree as P

pytestmark = pytest.mark.gpu
BF, F32, F64, I32, I64 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.int64


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _words(parents, C):
    """``anc`` of a list of trees; an entry None is no node (its tree None: no sequence)."""
    from coffin_b200.ops import tree
    rows = []
    for p in parents:
        if p is None:
            rows.append([0] * C)
            continue
        w = tree.path_words([-1 if q is None else q for q in p])
        rows.append([0 if q is None else x for q, x in zip(p, w)])
    return torch.tensor(rows, dtype=I64, device="cuda")


def _i32(v):
    return torch.tensor(v, dtype=I32, device="cuda")


# ------------------------------------------------------------------ attention
class Attn:
    def __init__(self, R, C, contexts, nh, nkv, hd, q8=False, kind="tree", gate=True, seed=0, parents=None, pages=None):
        rng, g = random.Random(seed), _gen(seed)
        self.R, self.C, self.nh, self.nkv, self.hd, self.contexts = R, C, nh, nkv, hd, contexts
        self.parents = parents or [P.random_parents(rng, C, kind) if c >= 0 else None for c in contexts]
        counts = [-(-(max(c, 0) + C) // 64) for c in contexts]
        pages = pages or sum(counts) + 3
        ids = rng.sample(range(pages), sum(counts))
        wide = max(counts)
        self.tables = _i32([[ids.pop() for _ in range(n)] + [0] * (wide - n) for n in counts])
        self.positions = _i32(contexts)
        n = lambda *s: torch.empty(s, dtype=BF, device="cuda").normal_(generator=g)  # noqa: E731
        self.kpool, self.vpool = n(pages * 64, nkv, hd), n(pages * 64, nkv, hd)
        self.kscale = self.vscale = None
        if q8:
            self.kpool, self.kscale = self._int8(self.kpool)
            self.vpool, self.vscale = self._int8(self.vpool)
        self.q = n(R * C, nh, hd)
        self.proj = n(R * C, nh * 2 * hd + 2 * nkv * hd) if gate else None
        self.out = torch.full((R * C, nh * hd), 7.0, dtype=BF, device="cuda")
        self.anc = _words(self.parents, C)

    @staticmethod
    def _int8(x):
        s = (x.float().abs().amax(-1) / 127).clamp_min(1e-8)
        return (x.float() / s.unsqueeze(-1)).round().clamp(-127, 127).to(torch.int8), s

    def run(self):
        from coffin_b200.ops import tree
        return tree.attn_tree(self.q, self.proj, self.kpool, self.vpool, self.tables, self.positions, self.anc, self.out, nh=self.nh, nkv=self.nkv,
                              hd=self.hd, kscale=self.kscale, vscale=self.vscale)

    def check(self, out=None):
        from coffin_b200.ops import kernels as K
        K.check_status()                                   # no bounded wait ran out
        R, C, nh, hd = self.R, self.C, self.nh, self.hd
        gate = self.proj[:, :nh * 2 * hd].reshape(R, C, nh, 2, hd)[:, :, :, 1] if self.proj is not None else None
        ref, bound = P.attn(self.q.view(R, C, nh, hd), gate, self.kpool, self.vpool, self.kscale, self.vscale, self.tables.tolist(), self.contexts,
                            self.parents, self.nkv)
        got = (self.out if out is None else out).view(R, C, nh, hd).double()
        used = (self.anc != 0).view(R, C, 1, 1).expand_as(got)
        off = ((got - ref).abs() / bound.clamp_min(1e-30))[used]
        assert off.numel() and float(off.max()) <= 1.0, f"{float(off.max()):.3g} times the bound"
        assert (got[~used] == 7.0).all(), "a row without a node was written"


@pytest.mark.parametrize("q8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("nh,nkv,hd", [(16, 4, 256), (24, 4, 256), (8, 1, 256), (8, 2, 128), (4, 2, 64), (3, 3, 64)])
@pytest.mark.parametrize("C,contexts,kind", [(1, [0, 1, 63, 64], "chain"), (4, [517], "chain"), (7, [65, 0, 127], "tree"), (16, [130, 700, 64, 5], "tree"),
                                             (33, [200], "star"), (64, [190, 3], "tree"), (64, [61], "chain")])
def test_attention_of_trees(nh, nkv, hd, C, contexts, kind, q8):
    a = Attn(len(contexts), C, contexts, nh, nkv, hd, q8, kind, gate=C % 2 == 1 or hd == 256, seed=C + hd)
    a.run()
    a.check()


@pytest.mark.parametrize("q8", [False, True], ids=["bf16", "int8"])
def test_attention_over_long_caches_of_uneven_length(q8):
    a = Attn(3, 5, [9001, 40, 2048], 16, 4, 256, q8, seed=3)
    a.run()
    a.check()
    again = a.out.clone()
    a.run()
    assert torch.equal(again, a.out), "the same inputs give the same bits"


@pytest.mark.parametrize("q8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("R,C,nh,nkv,hd,longest", [(20, 33, 16, 4, 256, 900), (12, 64, 21, 7, 128, 1500), (43, 3, 16, 4, 256, 1200), (3, 64, 32, 4, 256, 3000),
                                                   (150, 2, 4, 1, 64, 400), (2, 64, 16, 4, 256, 9000), (1, 43, 24, 4, 256, 5000)])
def test_attention_of_pieces_that_hold_several_items_and_of_items_in_several_pieces(R, C, nh, nkv, hd, longest, q8):
    """Many short sequences: pieces go on from one item to the next, with odd and even numbers of pages; few long ones: pieces end with them."""
    rng = random.Random(R + C)
    contexts = [rng.choice((0, 1, 64, rng.randrange(longest), rng.randrange(longest))) for _ in range(R - 1)] + [longest]
    a = Attn(R, C, contexts, nh, nkv, hd, q8, "tree", seed=R + hd)
    a.run()
    a.check()


def test_attention_skips_unused_rows_and_places():
    parents = [[-1, 0, None, 1, None], None, [-1, 0, 1, 2, 3]]
    a = Attn(3, 5, [100, -1, 31], 8, 2, 128, parents=parents, seed=5)
    a.run()
    a.check()


@pytest.mark.parametrize("q8", [False, True], ids=["bf16", "int8"])
def test_attention_does_not_read_what_is_masked(q8):
    """NaN and infinities behind the tree, in the pool's other pages and in other branches' rows."""
    a = Attn(2, 6, [70, 128], 8, 2, 64, q8, parents=[[-1, 0, 0, 1, 2, 3], [-1, 0, 1, 0, 3, 4]], seed=8)
    sick = {0: 2, 1: 1}                                    # a node of each tree and what hangs on it
    a.run()
    healthy = a.out.clone()
    seen = torch.zeros(a.kpool.shape[0], dtype=torch.bool)
    for r, ctx in enumerate(a.contexts):
        rows = P.slots_of(a.tables[r].tolist(), range(ctx + 6))
        keep = [row for i, row in enumerate(rows) if i - ctx != sick[r]]
        seen[keep] = True
    bad = (~seen).nonzero().flatten().cuda()
    if q8:
        a.kscale[bad], a.vscale[bad] = float("nan"), float("inf")
    else:
        a.kpool[bad], a.vpool[bad] = float("nan"), float("inf")
    a.run()
    for r in range(2):
        for j in range(6):
            row = r * 6 + j
            if sick[r] not in P.path_of(a.parents[r], j):
                assert torch.equal(a.out[row], healthy[row]), f"sequence {r} node {j} read a row that is not on its path"


@pytest.mark.parametrize("q8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("hd", [128, 256])
def test_attention_of_many_rows_does_not_read_what_is_masked(hd, q8):
    """The same with more than 128 rows a kv head: behind a last page that is short, alone or the second of two, and of no tokens at all."""
    contexts = [70, 128, 129, 0, 63]
    a = Attn(5, 48, contexts, 8, 2, hd, q8, seed=9)
    a.run()
    a.check()
    healthy = a.out.clone()
    seen = torch.zeros(a.kpool.shape[0], dtype=torch.bool)
    for r, ctx in enumerate(contexts):
        seen[P.slots_of(a.tables[r].tolist(), range(ctx + 48))] = True
    bad = (~seen).nonzero().flatten().cuda()
    if q8:
        a.kscale[bad], a.vscale[bad] = float("nan"), float("inf")
    else:
        a.kpool[bad], a.vpool[bad] = float("nan"), float("inf")
    a.run()
    assert torch.equal(a.out, healthy)


def test_attention_of_many_rows_in_two_graphs_that_run_at_once():
    a, b = (Attn(2, 64, [300, 1000], 16, 4, 256, seed=s) for s in (25, 26))
    graphs = [_captured(x.run)[0] for x in (a, b)]
    a.out.fill_(7.0), b.out.fill_(7.0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    a.check(), b.check()


def test_attention_with_strides_and_views():
    a = Attn(2, 9, [77, 300], 16, 4, 256, seed=11)
    tables = torch.full((2, a.tables.shape[1] + 5), -9, dtype=I32, device="cuda")
    tables[:, :a.tables.shape[1]] = a.tables
    a.tables = tables[:, :a.tables.shape[1]]
    proj = torch.zeros(18, a.proj.shape[1] + 64, dtype=BF, device="cuda")
    proj[:, :a.proj.shape[1]] = a.proj
    a.proj = proj[:, :a.proj.shape[1]]
    wide = torch.full((20, a.out.shape[1] + 8), 7.0, dtype=BF, device="cuda")
    a.out = wide[:18, :a.out.shape[1]]
    a.run()
    a.check(a.out.contiguous())
    assert (wide[18:] == 7.0).all() and (wide[:, a.out.shape[1]:] == 7.0).all()


def test_attention_of_pages_outside_the_pool_reads_nothing():
    a = Attn(1, 3, [150], 4, 2, 64, seed=2)
    a.tables[0, 1] = 1 << 24                               # no such page: its keys are no keys
    a.run()
    short = Attn(1, 3, [150], 4, 2, 64, seed=2)
    slots = P.slots_of(short.tables[0].tolist(), [p for p in range(153) if not 64 <= p < 128])
    k, v = short.kpool[slots].double(), short.vpool[slots].double()
    s = torch.einsum("hd,shd->hs", short.q[0].double(), k.repeat_interleave(2, 1)) / 8
    s[:, 150 - 64 + 1:] = float("-inf")                    # node 0 sees itself alone among the nodes
    ref = torch.einsum("hs,shd->hd", torch.softmax(s, -1), v.repeat_interleave(2, 1))
    gate = torch.sigmoid(short.proj[0, :512].view(4, 2, 64)[:, 1].double())
    assert ((a.out[0].view(4, 64).double() - ref * gate).abs() <= 3 * P.UBF * (ref.abs() + v.abs().amax()) * gate).all()
    a.tables[0, 1] = -5
    a.run()
    torch.cuda.synchronize()


def test_attention_passes_32_bits_of_offset():
    """Pages whose first element lies behind 2^31 elements of the pool."""
    pages = (1 << 31) // (64 * 4 * 256) + 40
    if torch.cuda.mem_get_info()[0] < 4 * pages * 64 * 4 * 256 * 2:
        pytest.skip("no room for two pools of more than 2^31 elements")
    a = Attn(1, 3, [100], 16, 4, 256, pages=1000, seed=4)
    small_k, small_v, ids = a.kpool, a.vpool, a.tables[0].tolist()
    a.kpool = torch.zeros(pages * 64, 4, 256, dtype=BF, device="cuda")
    a.vpool = torch.zeros_like(a.kpool)
    far = [pages - 1 - i for i in range(len(ids))]
    for f, i in zip(far, ids):
        a.kpool[f * 64:f * 64 + 64], a.vpool[f * 64:f * 64 + 64] = small_k[i * 64:i * 64 + 64], small_v[i * 64:i * 64 + 64]
    a.tables = _i32([far])
    a.run()
    a.check()


def _captured(fn):
    """``fn`` once eagerly on a side stream, then captured; returns the graph and what the captured call returned."""
    from coffin_b200.ops import kernels as K
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with K.capture_graph(graph):
        got = fn()
    return graph, got


def test_attention_in_two_graphs_that_run_at_once():
    a, b = (Attn(2, 8, [300, 1000], 16, 4, 256, seed=s) for s in (21, 22))
    graphs = [_captured(x.run)[0] for x in (a, b)]
    a.out.fill_(7.0), b.out.fill_(7.0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    a.check(), b.check()


# ------------------------------------------------------------------ delta net
class Gdn:
    def __init__(self, R, C, nk, nv, d, positions, kind="tree", seed=0, parents=None, pad=0):
        rng, g = random.Random(seed), _gen(seed)
        self.R, self.C, self.dims, self.pos = R, C, (nk, nv, d, d), positions
        conv = 2 * nk * d + nv * d
        n = lambda *s, scale=1.0, dtype=F32: torch.empty(s, dtype=dtype, device="cuda").normal_(0, scale, generator=g)  # noqa: E731
        self.parents = parents or [P.random_parents(rng, C, kind) for _ in range(R)]
        self.anc = _words(self.parents, C)
        self.width = conv + nv * d + 2 * nv
        self.proj = n(R * C, (self.width + 7) // 8 * 8 + pad, dtype=BF)
        self.conv_w, self.A_log = n(conv, 4, scale=0.5), torch.empty(nv, device="cuda").uniform_(0, 2, generator=g)
        self.dt_bias, self.norm_w = n(nv, scale=0.5) - 2, 1 + n(d, scale=0.1)
        self.ring, self.state = n(R + 2, 16, conv, dtype=BF), n(R + 2, nv, d, d, scale=0.1)
        self.slots = [-1 if p is None else s for p, s in zip(self.parents, rng.sample(range(R + 2), R))]
        self.out = torch.full((R * C, nv * d), 7.0, dtype=BF, device="cuda")
        self.record = torch.full((R, C, nv, 2 * d + 1), 7.0, device="cuda")
        self.raw = torch.full((R, C, conv), 7.0, dtype=BF, device="cuda")

    def run(self, **kw):
        from coffin_b200.ops import tree
        nk, nv, dk, dv = self.dims
        return tree.gdn_tree(self.proj, self.conv_w, self.A_log, self.dt_bias, self.norm_w, self.ring, self.state, _i32(self.slots) if not hasattr(self, "dslots") else self.dslots,
                             _i32(self.pos) if not hasattr(self, "dpos") else self.dpos, self.anc, self.out, self.record, self.raw,
                             nk=nk, nv=nv, dk=dk, dv=dv, eps=1e-6, **kw)

    def check(self, gate_sigmoid=False):
        nk, nv, dk, dv = self.dims
        R, C = self.R, self.C
        ref = P.gdn(self.proj.view(R, C, -1)[..., :self.width], self.conv_w, self.A_log, self.dt_bias, self.norm_w, self.ring, self.state, self.slots, self.pos,
                    self.parents, nk, nv, dk, dv, 1e-6, gate_sigmoid)
        used = (self.anc != 0)
        for name, got in (("out", self.out.view(R, C, nv, dv)), ("record", self.record)):
            off = ((got.double() - ref[name]).abs() / ref[name + "_bound"])[used]
            assert float(off.max()) <= 1.0, f"{name}: {float(off.max()):.3g} times the bound"
            assert (got[~used] == 7.0).all(), f"{name}: a place without a node was written"
        assert torch.equal(self.raw[used], ref["raw"][used]) and (self.raw[~used] == 7.0).all()


@pytest.mark.parametrize("nk,nv,d", [(16, 32, 128), (2, 6, 128), (2, 4, 64), (3, 3, 64)])
@pytest.mark.parametrize("C,positions,kind", [(1, [0], "chain"), (2, [1, 2, 3], "chain"), (5, [0, 517], "tree"), (8, [2], "star"), (16, [31, 1, 0], "tree"),
                                              (23, [100], "tree"), (64, [15], "tree"), (64, [16], "chain"), (41, [3], "star")])
def test_delta_net_of_trees(nk, nv, d, C, positions, kind):
    a = Gdn(len(positions), C, nk, nv, d, positions, kind, seed=C + nv)
    keep = a.state.clone(), a.ring.clone()
    a.run()
    a.check()
    assert torch.equal(keep[0], a.state) and torch.equal(keep[1], a.ring), "state and ring are read only"


@pytest.mark.parametrize("R,C,nk,nv,kind", [(3, 64, 16, 32, "tree"), (5, 49, 4, 16, "tree"), (1, 57, 8, 96, "star"), (2, 63, 38, 38, "chain"),      # a CTA a head
                                            (2, 33, 8, 24, "tree"), (1, 64, 19, 38, "chain")])                                               # two CTAs a head
def test_delta_net_of_trees_of_many_heads(R, C, nk, nv, kind):
    a = Gdn(R, C, nk, nv, 128, list(range(3, 3 + R)), kind, seed=C + nv)
    a.run()
    a.check()


def test_delta_net_with_sigmoid_gates_wide_rows_and_unused_places():
    a = Gdn(3, 9, 2, 4, 64, [4, 9, 40], parents=[[-1, 0, 1, None, 0, 4, None, 5, None], None, [-1] + list(range(8))], seed=6, pad=24)
    a.run(gate_sigmoid=True)
    a.check(gate_sigmoid=True)


def test_delta_net_of_a_chain_is_that_of_the_decode_kernel():
    """Same layer, chain of four: the kernel for chains uses approximate exponentials, so the two agree to their roundings only."""
    from coffin_b200.ops import kernels as K
    a = Gdn(2, 4, 16, 32, 128, [20, 700], "chain", seed=9)
    a.run()
    nk, nv, dk, dv = a.dims
    out, record = torch.zeros_like(a.out), torch.zeros_like(a.record)
    K.gdn_decode(a.proj, a.conv_w, a.A_log, a.dt_bias, a.norm_w, a.ring.clone(), a.state, _i32(a.slots), _i32(a.pos), out, nk=nk, nv=nv, dk=dk, dv=dv,
                 eps=1e-6, ntok=4, record=record, write_state=False)
    assert (record - a.record).abs().max() <= 2e-4 * record.abs().max()
    assert (out.float() - a.out.float()).norm() <= 2 * P.UBF * out.float().norm()


def test_delta_net_keeps_what_is_sick_on_its_path():
    a = Gdn(1, 7, 2, 4, 64, [12], parents=[[-1, 0, 0, 1, 2, 3, 4]], seed=12)
    a.run()
    healthy = a.out.clone(), a.record.clone()
    a.proj[2] = float("nan")
    a.run()
    for j in range(7):
        if 2 not in P.path_of(a.parents[0], j):
            assert torch.equal(a.out[j], healthy[0][j]) and torch.equal(a.record[0, j], healthy[1][0, j]), f"node {j}"
        else:
            assert not torch.isfinite(a.out[j].float()).any()


@pytest.mark.parametrize("C, kind", [(7, "tree"), (64, "tree")])
def test_delta_net_keeps_a_sick_gate_on_its_path(C, kind):
    """A decay that is no number is not taken for some decay: its node and the nodes behind it are none either, the others are what they were."""
    nv, d = 96, 128
    a = Gdn(1, C, 2, nv, d, [12], kind, seed=15)
    a.run()
    healthy = a.out.clone()
    a.proj[2, 2 * 2 * d + 2 * nv * d + nv:2 * 2 * d + 2 * nv * d + 2 * nv] = float("nan")
    a.run()
    for j in range(C):
        if 2 in P.path_of(a.parents[0], j):
            assert not torch.isfinite(a.out[j].float()).any()
        else:
            assert torch.equal(a.out[j], healthy[j]), f"node {j}"


def test_delta_net_with_decays_of_every_strength():
    a = Gdn(1, 32, 2, 4, 64, [50], "chain", seed=13)
    a.A_log.copy_(torch.tensor([-8.0, 0.0, 4.0, 12.0]))       # from almost none to everything at once
    a.dt_bias.copy_(torch.tensor([-4.0, 0.0, 4.0, 30.0]))
    a.run()
    assert torch.isfinite(a.out.float()).all() and torch.isfinite(a.record).all()
    a.check()


def test_delta_net_in_a_graph():
    a = Gdn(2, 16, 16, 32, 128, [7, 300], seed=14)
    a.dslots, a.dpos = _i32(a.slots), _i32(a.pos)
    graph, _ = _captured(a.run)
    a.out.fill_(7.0), a.record.fill_(7.0), a.raw.fill_(7.0)
    a.state.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    a.check()


# ------------------------------------------------------------------ verification
def _trees(R, C, V, T, seed, kind="tree", scale=3.0):
    """Logits, trees whose drafts are mostly what the target goes on with, and uniforms."""
    rng, g = random.Random(seed), _gen(seed)
    logits = torch.empty(R, C, V, device="cuda").normal_(0, scale, generator=g)
    u = torch.rand(R, C, generator=g, device="cuda")
    parents = [P.random_parents(rng, C, kind) for _ in range(R)]
    tokens = torch.randint(V, (R, C), generator=g, device="cuda")
    temps = [T] * R if not isinstance(T, (list, tuple)) else [T[r % len(T)] for r in range(R)]
    for r in range(R):
        for j in range(1, C):
            if rng.random() < 0.8:
                p = parents[r][j]
                tokens[r, j] = P.choose(P.probs(logits[r, p], temps[r]), float(u[r, len(P.path_of(parents[r], p)) - 1]))[0]
    return logits, parents, tokens, torch.tensor(temps, dtype=F32, device="cuda"), u


def _check_tree(logits, parents, tokens, temps, u, got):
    path, steps, nxt = (t.tolist() for t in got)
    for r in range(logits.shape[0]):
        want, t, near = P.walk(logits[r], tokens[r], parents[r], float(temps[r]), u[r])
        assert near > 1e-11, "the inputs put a draw on a border"
        n = len(want)
        assert steps[r] == n and path[r][:n] == want and all(x == -1 for x in path[r][n:]) and nxt[r] == t, (r, path[r], steps[r], nxt[r], want, t)


@pytest.mark.parametrize("R,C,V,T,kind", [(1, 1, 1, 1.0, "chain"), (1, 4, 512, 0.0, "chain"), (3, 5, 515, (0.0, 0.7, 1.5), "tree"), (2, 64, 4097, 1.0, "tree"),
                                          (2, 64, 100, 0.9, "chain"), (4, 16, 32003, (0.5, 0.0), "tree"), (1, 9, 151936, 0.8, "star"), (8, 8, 151936, (1.0, 0.0), "tree"),
                                          (1, 2, 1 << 20, 1.0, "chain"), (1, 3, (1 << 20) + 77, 1.3, "star")])
def test_verification_of_trees(R, C, V, T, kind):
    from coffin_b200.ops import tree
    logits, parents, tokens, temps, u = _trees(R, C, V, T, R * C + V % 97, kind)
    _check_tree(logits, parents, tokens, temps, u, tree.verify_tree(logits, tokens, _words(parents, C), temps, u))


def test_verification_takes_the_first_of_equal_siblings_and_of_equal_logits():
    from coffin_b200.ops import tree
    logits = torch.zeros(1, 4, 5000, device="cuda")
    logits[0, 0, [17, 4100, 4999]] = 3.0                       # ties: the lowest index
    logits[0, 2, 4999] = 1.0
    tokens = torch.tensor([[0, 4100, 17, 17]], device="cuda")
    path, steps, nxt = tree.verify_tree(logits, tokens, _words([[-1, 0, 0, 0]], 4), torch.zeros(1, device="cuda"), torch.zeros(1, 4, device="cuda"))
    assert path.tolist() == [[0, 2, -1, -1]] and steps.tolist() == [2] and nxt.tolist() == [4999]


def test_verification_with_masked_vocabularies_and_uniforms_at_the_ends():
    """Logits of -inf are never drawn, +inf is certain, NaN weighs nothing; u = 0 is the first token with weight, u = 1 the last one."""
    from coffin_b200.ops import tree
    V = 9001
    logits = torch.full((4, 1, V), float("-inf"), device="cuda")
    logits[0, 0, 5:8000] = torch.randn(7995, generator=_gen(1), device="cuda")
    logits[1] = logits[0]
    logits[2, 0, :] = 0.0
    logits[2, 0, 8191] = float("inf")
    logits[3, 0, 77:79] = torch.tensor([1.0, 1.0])
    logits[3, 0, 90:] = float("nan")
    one = torch.ones(4, device="cuda")
    u = torch.tensor([[0.0], [1.0], [0.3], [0.75]], device="cuda")
    got = tree.verify_tree(logits, torch.zeros(4, 1, dtype=I64, device="cuda"), torch.ones(4, 1, dtype=I64, device="cuda"), one, u)[2].tolist()
    assert got == [5, 7999, 8191, 78]
    masked = torch.full((1, 1, V), float("-inf"), device="cuda")
    t = int(tree.verify_tree(masked, torch.zeros(1, 1, dtype=I64, device="cuda"), torch.ones(1, 1, dtype=I64, device="cuda"), one[:1], u[2:3])[2])
    assert 0 <= t < V


@pytest.mark.parametrize("T", [1e-30, 1e-9, 3e-5, 0.02, 50.0, 1e30])
def test_verification_at_every_temperature(T):
    """Very cold rows are the arg-max (or one of its equals), very hot ones uniform over what is not masked."""
    from coffin_b200.ops import tree
    R, V = 6, 5001
    logits = torch.randn(R, 1, V, generator=_gen(11), device="cuda") * 4 + 31.0
    logits[1] -= 62.0
    logits[2, 0, [7, 4500]] = logits[2].max() + 1
    logits[3, 0, ::3] = float("-inf")
    temps = torch.full((R,), T, device="cuda")
    u = torch.rand(R, 1, generator=_gen(12), device="cuda")
    one = torch.ones(R, 1, dtype=I64, device="cuda")
    got = tree.verify_tree(logits, one, one, temps, u)[2].tolist()
    for r in range(R):
        want, near = P.choose(P.probs(logits[r, 0], float(temps[r])), float(u[r, 0]))
        assert near > 1e-11 and got[r] == want, r


@pytest.mark.parametrize("T", [3e31, 2e36, 3e38])
def test_masked_tokens_weigh_nothing_at_the_highest_temperatures(T):
    """At these all weights are 1 or 0 (exp of at most 40 / T); a floor of the type's lowest value over T would have weight."""
    from coffin_b200.ops import tree
    V = 5001
    logits = torch.randn(4, 1, V, generator=_gen(21), device="cuda")
    keep = torch.arange(0, V, 7, device="cuda")
    masked = torch.full_like(logits, float("-inf"))
    masked[:, :, keep] = logits[:, :, keep]
    one, u = torch.ones(4, 1, dtype=I64, device="cuda"), torch.tensor([[0.01], [0.37], [0.62], [0.99]], device="cuda")
    got = tree.verify_tree(masked, one, one, torch.full((4,), T, device="cuda"), u)[2].tolist()
    n = torch.full((4,), 1, dtype=I32, device="cuda")
    again = tree.verify_drafts(masked, one, n, None, torch.full((4,), T, device="cuda"), u, u[:, 0].contiguous())[1].tolist()
    for r in range(4):
        want, near = P.choose(P.probs(masked[r, 0], T), float(u[r, 0]))
        assert near > 1e-11 and got[r] == want and again[r] == want, r


def test_verification_skips_unused_sequences_and_reads_strided_logits():
    from coffin_b200.ops import tree
    logits, parents, tokens, temps, u = _trees(3, 6, 1003, 0.8, 5)
    wide = torch.full((3, 8, 1010), 50.0, device="cuda")
    wide[:, :6, 3:1006] = logits
    anc = _words(parents, 6)
    anc[1] = 0
    path, steps, nxt = tree.verify_tree(wide[:, :6, 3:1006], tokens, anc, temps, u)
    assert int(steps[1]) == 0 and int(nxt[1]) == -1 and (path[1] == -1).all()
    keep = torch.tensor([0, 2], device="cuda")
    _check_tree(logits[keep], [parents[0], parents[2]], tokens[keep], temps[keep], u[keep], (path[keep], steps[keep], nxt[keep]))


def test_sampled_tokens_follow_the_probabilities():
    """20,000 draws of a small vocabulary: each count within five standard deviations of its binomial."""
    from coffin_b200.ops import tree
    V, R, C = 50, 1000, 20
    row = torch.randn(V, generator=_gen(2), device="cuda") * 2
    p = P.probs(row, 0.9)
    draws = tree.verify_tree(row.view(1, 1, V).expand(R * C, 1, V), torch.zeros(R * C, 1, dtype=I64, device="cuda"), torch.ones(R * C, 1, dtype=I64, device="cuda"),
                             torch.full((R * C,), 0.9, device="cuda"), torch.rand(R * C, 1, generator=_gen(3), device="cuda"))[2]
    n = R * C
    count = torch.bincount(draws, minlength=V).double()
    assert ((count - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt() + 1).all()


def _chains(R, C, V, T, seed):
    rng, g = random.Random(seed), _gen(seed)
    logits = torch.empty(R, C, V, device="cuda").normal_(0, 3, generator=g)
    temps = [T] * R if not isinstance(T, (list, tuple)) else [T[r % len(T)] for r in range(R)]
    q = torch.softmax(logits[:, :-1] + torch.empty(R, C - 1, V, device="cuda").normal_(0, 0.5, generator=g), -1)
    tokens = torch.randint(V, (R, C), generator=g, device="cuda")
    for r in range(R):
        for i in range(C - 1):
            tokens[r, i + 1] = int(logits[r, i].argmax()) if temps[r] <= 0 and rng.random() < 0.8 else int(torch.multinomial(q[r, i], 1, generator=g))
    return (logits, tokens, _i32([rng.randint(1, C) for _ in range(R)]), q, torch.tensor(temps, dtype=F32, device="cuda"),
            torch.rand(R, C, generator=g, device="cuda"), torch.rand(R, generator=g, device="cuda"))


@pytest.mark.parametrize("R,C,V,T", [(1, 1, 77, 1.0), (2, 2, 1, 1.0), (6, 4, 515, (0.0, 1.0, 0.7)), (3, 64, 4097, 1.0), (8, 8, 32003, (1.0, 0.8)), (4, 5, 151936, (1.0, 0.0))])
def test_verification_of_chains_against_draft_probabilities(R, C, V, T):
    from coffin_b200.ops import tree
    args = _chains(R, C, V, T, R + C + V)
    steps, nxt = (t.tolist() for t in tree.verify_drafts(*args))
    logits, tokens, n, q, temps, u, ud = args
    for r in range(R):
        want, t, near = P.chain(logits[r], tokens[r], int(n[r]), q[r], float(temps[r]), u[r], ud[r])
        assert near > 1e-11 or V == 1
        assert (steps[r], nxt[r]) == (want, t), r


def test_drafts_of_unused_rows_and_of_tokens_outside_the_vocabulary():
    from coffin_b200.ops import tree
    logits, tokens, n, q, temps, u, ud = _chains(3, 4, 600, 1.0, 4)
    n.copy_(_i32([0, 4, 9]))
    tokens[1, 1], tokens[2, 2] = 600, -1                       # no token: not kept
    u[2, 1] = 0.0                                              # kept whatever it is
    steps, nxt = (t.tolist() for t in tree.verify_drafts(logits, tokens, n, q, temps, u, ud))
    assert steps == [0, 1, 2] and nxt[0] == -1 and all(0 <= t < 600 for t in nxt[1:])


def test_tokens_behind_drafts_are_distributed_as_the_targets():
    """One draft from a wrong distribution: the first new token (kept draft or its replacement) follows the target's probabilities."""
    from coffin_b200.ops import tree
    V, R, g = 30, 20000, _gen(7)
    p_l, q_l = torch.randn(V, generator=g, device="cuda") * 2, torch.randn(V, generator=g, device="cuda") * 2
    q = torch.softmax(q_l, -1)
    drafts = torch.multinomial(q, R, replacement=True, generator=g)
    tokens = torch.stack([torch.zeros_like(drafts), drafts], 1)
    steps, nxt = tree.verify_drafts(p_l.view(1, 1, V).expand(R, 2, V), tokens, torch.full((R,), 2, dtype=I32, device="cuda"), q.view(1, 1, V).expand(R, 1, V),
                                    torch.ones(R, device="cuda"), torch.rand(R, 2, generator=g, device="cuda"), torch.rand(R, generator=g, device="cuda"))
    first = torch.where(steps == 2, drafts, nxt)
    p = P.probs(p_l, 1.0)
    count = torch.bincount(first, minlength=V).double()
    assert ((count - R * p).abs() <= 5 * (R * p * (1 - p)).sqrt() + 1).all()
    kept = float((steps == 2).double().mean())
    want = float(torch.minimum(p, q.double()).sum())           # the share of drafts that can be kept at all
    assert abs(kept - want) <= 5 * (want * (1 - want) / R) ** 0.5


def test_verification_in_two_graphs_that_run_at_once():
    from coffin_b200.ops import tree
    sets = [_trees(4, 8, 32003, 0.9, s) for s in (31, 32)]
    calls = [lambda s=s, w=_words(s[1], 8): tree.verify_tree(s[0], s[2], w, s[3], s[4]) for s in sets]
    graphs = [_captured(c) for c in calls]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for s, (_, got) in zip(sets, graphs):
        _check_tree(*s, got)


# ------------------------------------------------------------------ commit
@pytest.mark.parametrize("q8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("C,L,nkv,hd", [(4, 2, 4, 256), (16, 1, 2, 64), (64, 3, 1, 128)])
def test_cache_rows_of_a_path_move_to_their_places(C, L, nkv, hd, q8):
    from coffin_b200.ops import tree
    rng, g, R = random.Random(C), _gen(C), 5
    contexts = [0, 63, 100, 61, -1]
    counts = [(max(c, 0) + C + 63) // 64 for c in contexts]
    pages = sum(counts) + 2
    ids = rng.sample(range(pages), sum(counts))
    tables = _i32([[ids.pop() for _ in range(n)] + [0] * (max(counts) - n) for n in counts])
    paths = [[0] + sorted(rng.sample(range(1, C), min(C - 1, k))) for k in (C - 1, 2, 0, 9, 3)]
    path = _i32([p + [-1] * (C - len(p)) for p in paths])
    steps = [len(p) for p in paths]
    n = lambda *s: torch.empty(s, device="cuda").normal_(generator=g)  # noqa: E731
    if q8:
        pools = [(n(L, pages * 64, nkv, hd) * 40).clamp(-127, 127).to(torch.int8) for _ in range(2)]
        scales = [n(L, pages * 64, nkv) for _ in range(2)]
    else:
        pools, scales = [n(L, pages * 64, nkv, hd).to(BF) for _ in range(2)], [None, None]
    want = [t.clone() if t is not None else None for t in pools + scales]
    for r, ctx in enumerate(contexts):
        if ctx < 0:
            continue
        src = P.slots_of(tables[r].tolist(), [ctx + i for i in paths[r]])
        dst = P.slots_of(tables[r].tolist(), [ctx + i for i in range(steps[r])])
        for t, w in zip(pools + scales, want):
            if t is not None:
                w[:, dst] = t[:, src]
    tree.kv_tree_commit(*pools, tables, _i32(contexts), path, _i32(steps), *scales)
    for t, w in zip(pools + scales, want):
        assert t is None or torch.equal(t, w)


@pytest.mark.parametrize("fork", [False, True], ids=["in place", "into other slots"])
@pytest.mark.parametrize("nk,nv,d,C,positions", [(16, 32, 128, 5, [0, 517]), (2, 4, 64, 64, [3, 16, 40, 0]), (2, 6, 128, 20, [1, 15])])
def test_states_advance_along_a_path(nk, nv, d, C, positions, fork):
    from coffin_b200.ops import tree
    rng, g, R, L, conv = random.Random(C), _gen(C), len(positions), 2, 2 * nk * d + nv * d
    n = lambda *s, scale=1.0: torch.empty(s, device="cuda").normal_(0, scale, generator=g)  # noqa: E731
    slots = rng.sample(range(2 * R + 1), 2 * R)
    src, dst = slots[:R], slots[R:] if fork else slots[:R]
    state, ring = n(L, 2 * R + 1, nv, d, d), n(L, 2 * R + 1, 16, conv).to(BF)
    record, raw = n(L, R, C, nv, 2 * d + 1, scale=0.2), n(L, R, C, conv).to(BF)
    lengths = [C, min(C, 3), 0, 1][:R]
    paths = [sorted(rng.sample(range(C), k)) for k in lengths]
    if R > 2:
        src[1] = -1 if not fork else src[1]
    before = state.clone(), ring.clone()
    tree.gdn_tree_commit(state, ring, record, raw, _i32(src), _i32(positions), _i32([p + [-1] * (C - len(p)) for p in paths]), _i32(lengths),
                         to_slots=_i32(dst) if fork else None)
    untouched = set(range(2 * R + 1))
    for r in range(R):
        if src[r] < 0:
            continue
        untouched.discard(dst[r])
        for l in range(L):
            ref, bound = P.advance(before[0][l, src[r]], record[l, r], paths[r], d, d)
            assert ((state[l, dst[r]].double() - ref).abs() <= bound).all(), (r, l)
            rows = before[1][l, src[r]].clone()
            for i, node in enumerate(paths[r]):
                rows[(positions[r] + i) % 16] = raw[l, r, node]
            assert torch.equal(ring[l, dst[r]], rows), (r, l)
    keep = torch.tensor(sorted(untouched), device="cuda")
    assert torch.equal(state[:, keep], before[0][:, keep]) and torch.equal(ring[:, keep], before[1][:, keep])


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("kind", ["tree", "chain"])
def test_a_verify_pass_of_trees_and_its_commit_equal_stepping_the_tokens(kind):
    """One attention and one delta-net layer: nodes of a tree, the path that is taken, the commit; then the same tokens one after the
    other.  What the next token finds (pages, state, ring) is the same up to the roundings of the two ways."""
    from coffin_b200.ops import tree
    nk, nv, d, nh, nkv, hd, C, pos0 = 2, 4, 64, 4, 2, 64, 12, 70
    a = Attn(1, C, [pos0], nh, nkv, hd, kind=kind, seed=40)
    s = Gdn(1, C, nk, nv, d, [pos0], seed=41, parents=a.parents)
    a.run(), s.run()
    logits = torch.randn(1, C, 300, generator=_gen(42), device="cuda") * 4
    tokens = torch.randint(300, (1, C), generator=_gen(43), device="cuda")
    u = torch.rand(1, C, generator=_gen(44), device="cuda")
    temps = torch.full((1,), 0.7, device="cuda")
    for j in range(1, C):
        p = a.parents[0][j]
        tokens[0, j] = P.choose(P.probs(logits[0, p], 0.7), float(u[0, len(P.path_of(a.parents[0], p)) - 1]))[0]
    path, steps, nxt = tree.verify_tree(logits, tokens, a.anc, temps, u)
    n, nodes = int(steps), path[0, :int(steps)].tolist()
    assert n == (C if kind == "chain" else 2) and nodes == P.walk(logits[0], tokens[0], a.parents[0], 0.7, u[0])[0]
    table = a.tables[0].tolist()
    rows = P.slots_of(table, [pos0 + i for i in nodes])
    want_k, want_v = a.kpool[rows].clone(), a.vpool[rows].clone()
    state, ring = s.state.clone(), s.ring.clone()
    kp, vp = a.kpool.unsqueeze(0), a.vpool.unsqueeze(0)
    tree.kv_tree_commit(kp, vp, a.tables, a.positions, path, steps)
    tree.gdn_tree_commit(state.unsqueeze(0), ring.unsqueeze(0), s.record.unsqueeze(0), s.raw.unsqueeze(0), _i32(s.slots), _i32([pos0]), path, steps)
    now = P.slots_of(table, [pos0 + i for i in range(n)])
    assert torch.equal(a.kpool[now], want_k) and torch.equal(a.vpool[now], want_v)
    # the same rows stepped as a chain from the old state
    chain = Gdn(1, n, nk, nv, d, [pos0], "chain", seed=41)
    for name in ("conv_w", "A_log", "dt_bias", "norm_w", "state", "ring"):
        setattr(chain, name, getattr(s, name))
    chain.slots, chain.proj = s.slots, s.proj[nodes].contiguous()
    chain.run()
    chain.check()
    assert (chain.out.float() - s.out[nodes].float()).norm() <= 2 * P.UBF * chain.out.float().norm()
    st = s.state.clone()
    rg = s.ring.clone()
    tree.gdn_tree_commit(st.unsqueeze(0), rg.unsqueeze(0), chain.record.unsqueeze(0), chain.raw.unsqueeze(0), _i32(s.slots), _i32([pos0]),
                         _i32([list(range(n))]), _i32([n]))
    assert torch.equal(rg, ring) and (st - state).abs().max() <= 64 * n * P.U32 * state.abs().max()


def test_calls_from_two_threads_on_streams_of_their_own():
    """Launches that want different amounts of shared memory, from threads that do not wait for one another."""
    import threading
    jobs = [[Gdn(1, C, 4, 8, 128, [9], "tree", seed=40 + C) for C in (12, 40, 64)], [Attn(2, C, [300, 77], 8, 2, 128, C == 33, seed=50 + C) for C in (5, 33, 64)]]
    failed = []

    def work(mine):
        try:
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.default_stream())
            with torch.cuda.stream(s):
                for i in range(60):
                    mine[i % len(mine)].run()
            s.synchronize()
        except Exception as e:          # noqa: BLE001
            failed.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(m,)) for m in (jobs[0], jobs[0][::-1], jobs[1])]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for x in jobs[0] + jobs[1]:
        x.check()
