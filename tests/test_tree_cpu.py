"""What the tree operators refuse and how trees are described; no GPU."""
import pytest
import torch

from coffin_b200.ops import tree

BF, F32, I32, I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64


def test_path_words():
    assert tree.path_words([-1]) == [1]
    assert tree.path_words([-1, 0, 0, 1, 2]) == [1, 0b11, 0b101, 0b1011, 0b10101]
    chain = tree.path_words(list(range(-1, 63)))
    assert chain[62] == (1 << 63) - 1 and chain[63] == -1
    for bad in ([], [-1, 1], [-1, 0, 5], [0], [-2], [-1] + [0] * 64):
        with pytest.raises(ValueError):
            tree.path_words(bad)


def _attn_args(R=2, C=4, nh=4, nkv=2, hd=64, pages=6):
    z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype)  # noqa: E731
    a = [z(R * C, nh, hd), z(R * C, 2 * nh * hd + 2 * nkv * hd), z(pages * 64, nkv, hd), z(pages * 64, nkv, hd), z(R, 3, dtype=I32), z(R, dtype=I32),
         z(R, C, dtype=I64), z(R * C, nh * hd)]
    return a, dict(nh=nh, nkv=nkv, hd=hd)


def _refuse(fn, match, *a, **k):
    with pytest.raises(ValueError, match=match):
        fn(*a, **k)


def test_attention_refuses():
    a, k = _attn_args()

    def swap(i, t, match, **kw):
        _refuse(tree.attn_tree, match, *a[:i], t, *a[i + 1:], **{**k, **kw})

    swap(0, a[0].float(), "q: ")
    swap(0, a[0][:-1], "q: ")
    swap(1, a[1][:, :100], "proj: ")
    swap(1, a[1].half(), "proj: ")
    swap(1, torch.zeros(8, 2 * 4 * 64 + 3, dtype=BF), "proj: ")
    swap(2, a[2].to(torch.int8), "kpool: ")
    swap(2, a[2][:-1], "kpool: ")
    swap(3, a[3][:, :1], "vpool: ")
    swap(4, a[4].long(), "block_tables")
    swap(4, a[4][:1], "block_tables")
    swap(4, a[4][:, :0], "block_tables")
    swap(5, a[5][:1], "positions")
    swap(6, a[6].int(), "anc")
    swap(6, torch.zeros(2, 65, dtype=I64), "1 to 64 nodes")
    swap(6, torch.zeros(2, 0, dtype=I64), "1 to 64 nodes")
    swap(7, a[7].float(), "out: ")
    swap(7, torch.zeros(8, 257, dtype=BF)[:, 1:], "out: ")
    swap(0, a[0], "query heads", hd=96)
    swap(0, a[0], "query heads", nkv=3)
    swap(0, a[0], "kpool: ", kscale=torch.zeros(6 * 64, 2))
    a[2], a[3] = a[2].to(torch.int8), a[3].to(torch.int8)
    swap(0, a[0], "go together", kscale=torch.zeros(6 * 64, 2))
    swap(0, a[0], "scales", kscale=torch.zeros(6 * 64, 2), vscale=torch.zeros(6 * 64))
    swap(0, a[0], "current CUDA device", kscale=torch.zeros(6 * 64, 2), vscale=torch.zeros(6 * 64, 2))


def test_delta_net_refuses():
    R, C, nk, nv, d = 2, 3, 1, 2, 64
    conv = 2 * nk * d + nv * d
    z = lambda *s, dtype=F32: torch.zeros(*s, dtype=dtype)  # noqa: E731
    a = [z(R * C, conv + nv * d + 8, dtype=BF), z(conv, 4), z(nv), z(nv), z(d), z(4, 16, conv, dtype=BF), z(4, nv, d, d), z(R, dtype=I32), z(R, dtype=I32),
         z(R, C, dtype=I64), z(R * C, nv * d, dtype=BF), z(R, C, nv, 2 * d + 1), z(R, C, conv, dtype=BF)]
    k = dict(nk=nk, nv=nv, dk=d, dv=d, eps=1e-6)

    def swap(i, t, match, **kw):
        _refuse(tree.gdn_tree, match, *a[:i], t, *a[i + 1:], **{**k, **kw})

    swap(0, a[0].float(), "proj: ")
    swap(0, torch.zeros(R * C, conv + nv * d + 2 * nv, dtype=BF)[:, :-1], "proj: ")
    swap(0, torch.zeros(R * C, conv + nv * d + 7, dtype=BF), "proj: ")
    swap(1, a[1][:, :3], "conv_w")
    swap(5, a[5][:, :8], "ring")
    swap(6, a[6].double(), "state")
    swap(6, a[6].transpose(2, 3), "state")
    swap(7, a[7].long(), "slots")
    swap(11, a[11][:, :, :, 1:], "record")
    swap(12, a[12].float(), "raw")
    swap(0, a[0], "delta-net heads", dk=32)
    swap(0, a[0], "delta-net heads", nk=3)
    swap(0, a[0], "current CUDA device")


def test_verification_refuses():
    R, C, V = 2, 3, 50
    logits, tokens, anc = torch.zeros(R, C, V), torch.zeros(R, C, dtype=I64), torch.ones(R, C, dtype=I64)
    temp, u, n, q, ud = torch.ones(R), torch.zeros(R, C), torch.ones(R, dtype=I32), torch.zeros(R, C - 1, V), torch.zeros(R)
    for bad, match in (((logits.half(), tokens, anc, temp, u), "logits"), ((logits.transpose(1, 2), tokens, anc, temp, u), "logits"),
                       ((logits[:, :2], tokens, anc, temp, u), "logits"), ((logits[:, :, :0], tokens, anc, temp, u), "logits"),
                       ((logits, tokens.int(), anc, temp, u), "tokens"), ((logits, tokens, anc, temp.double(), u), "temperature"),
                       ((logits, tokens, anc, temp, u[:, :1]), "u: "), ((logits, tokens, anc, temp, u), "current CUDA device")):
        _refuse(tree.verify_tree, match, *bad)
    for bad, match in (((logits, tokens, n.long(), q, temp, u, ud), "lengths"), ((logits, tokens, n, q[:, :1], temp, u, ud), "draft_probs"),
                       ((logits, tokens, n, q.double(), temp, u, ud), "draft_probs"), ((logits, tokens, n, q, temp, u, ud[:1]), "u_draw"),
                       ((logits, torch.zeros(R, 65, dtype=I64), n, q, temp, u, ud), "tokens"), ((logits, tokens, n, q, temp, u, ud), "current CUDA device")):
        _refuse(tree.verify_drafts, match, *bad)


def test_commits_refuse():
    L, slots, nkv, hd, R, C = 2, 128, 2, 64, 2, 4
    pool, tables, pos = torch.zeros(L, slots, nkv, hd, dtype=BF), torch.zeros(R, 2, dtype=I32), torch.zeros(R, dtype=I32)
    path, steps = torch.zeros(R, C, dtype=I32), torch.zeros(R, dtype=I32)
    for bad, match in (((pool[0], pool[0], tables, pos, path, steps), "pools"), ((pool, pool[:1], tables, pos, path, steps), "pools"),
                       ((pool[..., :4].contiguous()[:, :, :1].contiguous(), pool[..., :4].contiguous()[:, :, :1].contiguous(), tables, pos, path, steps), "16 bytes"),
                       ((pool.to(torch.int8), pool.to(torch.int8), tables, pos, path, steps), "int8"), ((pool, pool, tables.long(), pos, path, steps), "block_tables"),
                       ((pool, pool, tables, pos, path.long(), steps), "path"), ((pool, pool, tables, pos, path, steps[:1]), "steps"),
                       ((pool, pool, tables, pos, path, steps), "current CUDA device")):
        _refuse(tree.kv_tree_commit, match, *bad)
    nv, d, conv = 2, 64, 256
    state, ring, rec = torch.zeros(L, 3, nv, d, d), torch.zeros(L, 3, 16, conv, dtype=BF), torch.zeros(L, R, C, nv, 2 * d + 1)
    raw, ids = torch.zeros(L, R, C, conv, dtype=BF), torch.zeros(R, dtype=I32)
    for bad, match in (((state[0], ring, rec, raw, ids, pos, path, steps), "state"), ((state[..., :32].contiguous(), ring, rec, raw, ids, pos, path, steps), "states of"),
                       ((state, ring[:, :2], rec, raw, ids, pos, path, steps), "ring"), ((state, ring, rec[:, :1], raw, ids, pos, path, steps), "record"),
                       ((state, ring, rec, raw.float(), ids, pos, path, steps), "raw"), ((state, ring, rec, raw, ids.long(), pos, path, steps), "slots"),
                       ((state, ring, rec, raw, ids, pos, path, steps), "current CUDA device")):
        _refuse(tree.gdn_tree_commit, match, *bad)
