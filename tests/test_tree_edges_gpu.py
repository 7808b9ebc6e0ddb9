"""Tree operators where numbers end: scores that are infinite or none, keys that are nearly equal, positions at the end of their type."""
import pytest
import torch

import plain_tree as P
import plain_tree_matrix as M
from test_tree_gpu import Attn, Gdn

pytestmark = pytest.mark.gpu
BF, F32, F64, I32, I64 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.int64
NAN, INF = float("nan"), float("inf")

# (contexts, nodes, heads, kv heads, head width): a page a piece, pieces of several pages, pairs of CTAs
SHAPES = [([200, 100], 3, 8, 2, 64), ([20000, 70], 4, 16, 4, 256), ([900, 300], 48, 8, 2, 128)]


def _page_rows(a, r, pages):
    """Pool rows of the cached tokens in these pages of sequence r."""
    return torch.tensor([s for s in P.slots_of(a.tables[r].tolist(), range(a.contexts[r]))], device="cuda").split(64)[pages[0]:pages[1]]


@pytest.mark.parametrize("q8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("shape", SHAPES, ids=["page", "pages", "pairs"])
@pytest.mark.parametrize("pages", [(1, 2), (0, 1), (0, 10000)], ids=["second", "first", "all"])
def test_scores_that_are_no_numbers_reach_the_output(shape, pages, q8):
    """Whole pages of keys that are NaN, alone or with the rest of the cache: the sequence's rows are NaN, the other's stay as they were."""
    contexts, C, nh, nkv, hd = shape
    a = Attn(2, C, contexts, nh, nkv, hd, q8, seed=31)
    a.run()
    healthy = a.out.clone()
    rows = torch.cat(_page_rows(a, 0, pages))
    if q8:
        a.kscale[rows] = NAN
    else:
        a.kpool[rows] = NAN
    a.run()
    assert a.out[:C].isnan().all()
    assert torch.equal(a.out[C:], healthy[C:])


@pytest.mark.parametrize("shape", SHAPES, ids=["page", "pages", "pairs"])
def test_infinite_scores(shape):
    """A score of -inf is a weight of 0; +inf makes the row NaN, as inf - inf does; a row whose scores are all -inf is 0, like one that
    sees no key."""
    contexts, C, nh, nkv, hd = shape
    a = Attn(2, C, contexts, nh, nkv, hd, seed=32)
    a.q.abs_().clamp_(min=0.01)                            # q.k has the sign of an infinite key
    keys, tables = a.kpool.clone(), a.tables.clone()
    rows = torch.cat(_page_rows(a, 0, (1, 2)))
    a.tables[0, 1] = -1                                    # a page that is none leaves the sum: the same weights
    a.run()
    without = a.out.clone()
    a.tables.copy_(tables)
    a.kpool[rows] = -INF
    a.run()
    assert torch.equal(a.out, without)
    a.kpool[rows[5]] = INF
    a.run()
    assert a.out[:C].isnan().all() and torch.equal(a.out[C:], without[C:])
    a.kpool.copy_(keys)
    a.kpool[P.slots_of(a.tables[0].tolist(), range(contexts[0] + C))] = -INF
    a.run()
    assert (a.out[:C] == 0).all() and torch.equal(a.out[C:], without[C:])


@pytest.mark.parametrize("q8", [False, True], ids=["bf16", "int8"])
def test_positions_at_the_end_of_their_type(q8):
    """Nodes whose positions pass 2^31 have no page, like those behind the table's last one: the row sees the table's pages alone, and a commit
    moves nothing."""
    from coffin_b200.ops import tree
    last = 2 ** 31 - 1
    a = Attn(4, 64, [100, 130, 70, 5], 8, 2, 64, q8, seed=33)
    wide = a.tables.shape[1] * 64
    a.tables[a.tables == 0] = -1                           # places behind a sequence's own pages: none of the pool's
    a.positions.copy_(torch.tensor([wide, wide, wide, 5], dtype=I32))
    a.run()
    at_end = a.out.clone()
    for back in (0, 1, 40, 62, 63, 64):
        a.positions.copy_(torch.tensor([last - back, last, last - 31, 5], dtype=I32))
        a.out.fill_(7.0)
        a.run()
        assert torch.equal(a.out, at_end), back
    path = torch.arange(64, dtype=I32, device="cuda").repeat(4, 1)
    path[:, 1:33] = torch.arange(2, 66, 2, dtype=I32, device="cuda").clamp(max=63)
    steps = torch.tensor([33, 33, 33, 0], dtype=I32, device="cuda")
    pools = [a.kpool[None].clone(), a.vpool[None].clone()]
    scales = [a.kscale[None].clone(), a.vscale[None].clone()] if q8 else [None, None]
    tree.kv_tree_commit(*pools, a.tables, a.positions, path, steps, *scales)
    assert torch.equal(pools[0][0], a.kpool) and torch.equal(pools[1][0], a.vpool)
    if q8:
        assert torch.equal(scales[0][0], a.kscale) and torch.equal(scales[1][0], a.vscale)


@pytest.mark.parametrize("noise", [0.0, 0.02], ids=["equal", "near"])
@pytest.mark.parametrize("C,nk,nv,d,kind", [(8, 2, 4, 128, "chain"), (8, 2, 4, 64, "star"), (24, 8, 32, 128, "chain"), (64, 8, 32, 128, "chain"), (64, 8, 64, 128, "tree"),
                                            (64, 10, 80, 128, "chain"), (33, 10, 160, 128, "chain"), (64, 2, 4, 64, "chain")])
def test_delta_net_of_a_run_of_one_token(C, nk, nv, d, kind, noise):
    """Keys that are equal or nearly so, hardly any decay and every strength of update: the triangular inverse at its worst."""
    a = Gdn(1, C, nk, nv, d, [20], kind, seed=C + nv)
    conv = 2 * nk * d + nv * d
    one = a.proj[:1].clone()
    a.proj.copy_((one.float() * (1 + noise * torch.randn(a.proj.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)))).to(BF))
    a.ring[a.slots[0]] = one[0, :conv]
    a.proj[:, conv + nv * d:conv + nv * d + nv] = torch.linspace(-3, 9, nv, device="cuda").to(BF)
    a.A_log.fill_(-6.0)
    a.run()
    dims = a.dims
    out, bound, D, De = M.gdn(a.proj[:, :a.width], a.conv_w, a.A_log, a.dt_bias, a.norm_w, a.ring[a.slots[0]], a.state[a.slots[0]], 20, a.parents[0], *dims, 1e-6)
    for name, got, want, most in (("update", a.record[0, :, :, d:2 * d], D, De), ("out", a.out.view(C, nv, d), out, bound)):
        off = (got.double() - want).abs()
        assert float((off / most).max()) <= 1.0, name
    # worst-case sums of signs over 64 equal keys; the node-by-node bound is 10^13 times the updates there
    assert float((De / D.abs().amax((0, 2), keepdim=True)).max()) < 0.25
