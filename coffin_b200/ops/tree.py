"""Entry points of speculative verification: trees of drafted tokens and drafts of sampled requests.

A tree has up to ``MAX_NODES`` nodes a sequence, a parent before its children.  Node 0 is the token that was sampled last; its words
``anc [R, C]`` (int64) have bit ``i`` set for every node ``i`` on the path to a node, the node itself included, and are 0 where there is
no node (:func:`path_words` makes them from parents).  Node ``j`` keeps its key and value at position ``positions[r] + j`` of the
sequence's pages (``kernels.attn_prep`` appends them) and is rotated as position ``positions[r] +`` its depth.  Per layer
``attn_tree`` or ``gdn_tree`` takes the place of the prefill and decode kernels; ``verify_tree`` finds the path that the request's own
tokens take, ``kv_tree_commit`` and ``gdn_tree_commit`` make it part of the sequence.  None of them waits for the host, allocates
anything but its own workspace on the current stream, or keeps anything between calls, so all can be captured in a graph.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from . import kernels as K
from ._lib import call

MAX_NODES = 64


def path_words(parents: list[int]) -> list[int]:
    """Words of the nodes whose parents are given (-1: none; a parent before its children), as signed 64-bit numbers."""
    if not 1 <= len(parents) <= MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, not {len(parents)}")
    words: list[int] = []
    for j, p in enumerate(parents):
        if not -1 <= p < j:
            raise ValueError(f"node {j} has parent {p}: a parent comes before its children")
        words.append((words[p] if p >= 0 else 0) | 1 << j)
    return [w - (1 << 64) if w >> 63 else w for w in words]


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _place(anchor: torch.Tensor, **others: torch.Tensor | None) -> None:
    """All tensors on the anchor's device, which has to be the current one (launches go to its current stream)."""
    dev = anchor.device
    _need(dev.type == "cuda" and dev.index == torch.cuda.current_device(), f"tensors have to lie on the current CUDA device, not {dev}")
    for name, t in others.items():
        _need(t is None or t.device == dev, f"{name} lies on another device")


def _rows(anc: torch.Tensor) -> tuple[int, int]:
    _need(anc.dim() == 2 and anc.dtype == torch.int64 and anc.is_contiguous(), "anc: a contiguous int64 [sequences, nodes]")
    R, C = anc.shape
    _need(1 <= C <= MAX_NODES, f"a tree has 1 to {MAX_NODES} nodes, not {C}")
    return R, C


def _vec(t: torch.Tensor, n: int, dtype: torch.dtype, name: str) -> None:
    _need(t.dtype == dtype and t.numel() == n and t.is_contiguous(), f"{name}: {n} contiguous {dtype}")


# ------------------------------------------------------------------ attention
CTAS = 148          # pieces that the pages of all sequences are cut into: one CTA an SM


def attn_tree(q, proj, kpool, vpool, block_tables, positions, anc, out, *, nh: int, nkv: int, hd: int, kscale=None, vscale=None) -> torch.Tensor:
    """Attention of tree nodes over their sequences' pages and their own paths: ``q [R * C, nh, hd]`` normed and rotated, the nodes'
    keys and values in the pools already; ``proj`` supplies the output gate as for ``kernels.attn_prefill`` (``None``: no gate).
    ``block_tables [R, pages]`` and ``positions [R]`` (cached tokens, < 0: unused row) int32; rows without a node stay as they were.
    ``kscale`` / ``vscale``: the pools are int8."""
    R, C = _rows(anc)
    _need(hd in (64, 128, 256) and nkv >= 1 and nh % nkv == 0, f"{nh} query heads of {hd} over {nkv} kv heads")
    _need(q.dtype == torch.bfloat16 and q.is_contiguous() and q.numel() == R * C * nh * hd and q.data_ptr() % 16 == 0, "q: contiguous bf16 [R * C, nh, hd]")
    _need(out.dtype == torch.bfloat16 and out.dim() == 2 and out.shape[0] >= R * C and out.shape[1] >= nh * hd and out.stride(1) == 1
          and out.stride(0) % 8 == 0 and out.data_ptr() % 16 == 0, "out: bf16 [R * C, nh * hd] in 16-byte rows")
    _need(proj is None or (proj.dtype == torch.bfloat16 and proj.dim() == 2 and proj.shape[0] >= R * C and proj.shape[1] >= 2 * nh * hd and proj.stride(1) == 1
                           and proj.stride(0) % 8 == 0 and proj.data_ptr() % 16 == 0), "proj: bf16 rows that begin with (q | gate) of every head")
    kv = torch.int8 if kscale is not None else torch.bfloat16
    slots = kpool.shape[0]
    for t, name in ((kpool, "kpool"), (vpool, "vpool")):
        _need(t.dtype == kv and t.shape == (slots, nkv, hd) and t.is_contiguous() and t.data_ptr() % 16 == 0 and slots % K.BLOCK == 0,
              f"{name}: contiguous {kv} [pages * {K.BLOCK}, {nkv}, {hd}]")
    _need((kscale is None) == (vscale is None), "kscale and vscale go together")
    for t in (kscale, vscale):
        _need(t is None or (t.dtype == torch.float32 and t.is_contiguous() and t.numel() == slots * nkv), "scales: contiguous fp32 [slots, nkv]")
    _need(block_tables.dtype == torch.int32 and block_tables.dim() == 2 and block_tables.shape[0] == R and block_tables.shape[1] >= 1
          and block_tables.stride(1) == 1, "block_tables: int32 [R, pages]")
    _vec(positions, R, torch.int32, "positions")
    _place(q, proj=proj, kpool=kpool, vpool=vpool, block_tables=block_tables, positions=positions, anc=anc, out=out, kscale=kscale, vscale=vscale)
    if R == 0:
        return out
    rows = C * (nh // nkv)
    part = torch.empty((CTAS + R * nkv * -(-rows // 128)) * min(rows, 128) * (hd + 2), dtype=torch.float32, device=q.device)
    call("attn_tree", q, proj, proj.stride(0) if proj is not None else 0, kpool, vpool, slots, kscale, vscale, block_tables, block_tables.stride(0),
         block_tables.shape[1], positions, anc, out, out.stride(0), part, CTAS, R, C, nh, nkv, hd, K.status_word(q.device))
    K._count(2)
    return out


# ------------------------------------------------------------------ gated delta net
def gdn_tree(proj, conv_w, A_log, dt_bias, norm_w, ring, state, slots, positions, anc, out, record, raw, *, nk: int, nv: int, dk: int, dv: int,
             eps: float, gate_sigmoid: bool = False) -> torch.Tensor:
    """The layer of ``kernels.gdn_decode`` over the nodes of trees: ``proj [R * C, ...]`` raw projection rows, ``state [slots, nv, dk, dv]``
    and ``ring [slots, 16, conv]`` of the sequences (read, not written), ``slots [R]`` (< 0: unused row) and ``positions [R]`` int32.
    ``record [R, C, nv, dk + dv + 1]`` (fp32: key, update, decay) and ``raw [R, C, conv]`` are what ``gdn_tree_commit`` replays."""
    R, C = _rows(anc)
    conv, bf, f32 = 2 * nk * dk + nv * dv, torch.bfloat16, torch.float32
    _need((dk, dv) in ((128, 128), (64, 64)) and nk >= 1 and nv % nk == 0, f"delta-net heads {nk} / {nv} of {dk} x {dv}")
    _need(proj.dtype == bf and proj.dim() == 2 and proj.shape[0] >= R * C and proj.shape[1] >= conv + nv * dv + 2 * nv and proj.stride(1) == 1
          and proj.stride(0) % 8 == 0 and proj.data_ptr() % 16 == 0, "proj: bf16 rows q | k | v | z | b | a of a multiple of 16 bytes")
    _need(out.dtype == bf and out.dim() == 2 and out.shape[0] >= R * C and out.shape[1] >= nv * dv and out.stride(1) == 1
          and out.stride(0) % 4 == 0 and out.data_ptr() % 8 == 0, "out: bf16 [R * C, nv * dv] in 8-byte rows")
    n = state.shape[0]
    _need(state.dtype == f32 and state.shape == (n, nv, dk, dv) and state.is_contiguous() and state.data_ptr() % 16 == 0, "state: contiguous fp32 [slots, nv, dk, dv]")
    _need(ring.dtype == bf and ring.shape == (n, K.RING, conv) and ring.is_contiguous() and ring.data_ptr() % 16 == 0, "ring: contiguous bf16 [slots, 16, conv]")
    _vec(conv_w, conv * 4, f32, "conv_w")
    _need(conv_w.data_ptr() % 16 == 0, "conv_w: 16-byte rows")
    _vec(A_log, nv, f32, "A_log"), _vec(dt_bias, nv, f32, "dt_bias"), _vec(norm_w, dv, f32, "norm_w")
    _need(norm_w.data_ptr() % 16 == 0, "norm_w: a 16-byte address")
    _vec(slots, R, torch.int32, "slots"), _vec(positions, R, torch.int32, "positions")
    _vec(record, R * C * nv * (dk + dv + 1), f32, "record"), _vec(raw, R * C * conv, bf, "raw")
    _place(proj, conv_w=conv_w, A_log=A_log, dt_bias=dt_bias, norm_w=norm_w, ring=ring, state=state, slots=slots, positions=positions, anc=anc,
           out=out, record=record, raw=raw)
    if R:
        rows = torch.empty(R * C * conv, dtype=f32, device=proj.device)
        call("gdn_tree", proj, proj.stride(0), conv_w, A_log, dt_bias, norm_w, ring, state, slots, positions, anc, out, out.stride(0), record, raw, rows,
             n, R, C, nk, nv, dk, dv, float(eps), int(gate_sigmoid))
        K._count(2)
    return out


# ------------------------------------------------------------------ verification
def _scratch(R: int, C: int, V: int, device) -> torch.Tensor:
    fn = _lib.lib().cb_verify_scratch
    fn.restype = ctypes.c_int64
    return torch.empty(int(fn(ctypes.c_int64(R), ctypes.c_int64(C), ctypes.c_int64(V))), dtype=torch.uint8, device=device)


def _logits(logits: torch.Tensor, R: int, C: int) -> int:
    _need(logits.dtype == torch.float32 and logits.dim() == 3 and tuple(logits.shape[:2]) == (R, C) and logits.shape[2] >= 1
          and (logits.stride(2) == 1 or logits.shape[2] == 1), "logits: fp32 [R, C, vocabulary]")
    _need(R * C <= 65535, f"{R} x {C} rows of logits")
    return logits.shape[2]


def verify_tree(logits, tokens, anc, temperature, u) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The path that the request's own tokens take through its tree of drafts.

    The token of a node is drawn from ``softmax(logits[r, j] / temperature[r])`` by inverse CDF with ``u[r, depth of j]``, or is the arg-max
    (lowest index) where the temperature is not positive; from node 0 on the first child that carries the token (``tokens [R, C]``
    int64) is next.  Returns ``path`` (int32 ``[R, C]``, -1 behind its end), ``steps`` (int32 ``[R]``, nodes on the path) and ``next``
    (int64 ``[R]``, the token drawn at its end): the new tokens are those of the path behind node 0, then ``next``, the ones that
    sampling one by one with the same uniforms draws.  Draws are 64-bit.  A sequence whose node 0 is none gets 0 steps and token -1."""
    R, C = _rows(anc)
    V = _logits(logits, R, C)
    _vec(tokens, R * C, torch.int64, "tokens"), _vec(temperature, R, torch.float32, "temperature"), _vec(u, R * C, torch.float32, "u")
    dev = logits.device
    _place(logits, tokens=tokens, anc=anc, temperature=temperature, u=u)
    path = torch.empty(R, C, dtype=torch.int32, device=dev)
    steps, nxt = torch.empty(R, dtype=torch.int32, device=dev), torch.empty(R, dtype=torch.int64, device=dev)
    if R:
        call("verify_tree", logits, logits.stride(0), logits.stride(1), tokens, anc, temperature, u, path, steps, nxt, _scratch(R, C, V, dev), R, C, V)
        K._count(3)
    return path, steps, nxt


def verify_drafts(logits, tokens, lengths, draft_probs, temperature, u, u_draw) -> tuple[torch.Tensor, torch.Tensor]:
    """How much of a chain of drafts that were drawn from ``draft_probs`` is kept, and the token after it.

    Row ``r`` is a chain of ``lengths[r]`` (int32; 0: unused row) of the ``C`` tokens ``tokens[r]``: the token that was sampled last,
    then drafts, draft ``i`` drawn from ``draft_probs[r, i - 1]`` (fp32 ``[R, C - 1, vocabulary]``, each summing to one).  With
    ``p = softmax(logits / temperature)`` draft ``i`` is kept while ``u[r, i] q(x) < p(x)``; the next token is drawn with ``u_draw[r]`` from
    ``max(p - q, 0)`` of the first draft that is not, or from ``p`` behind the last one, so that the tokens are distributed as the target's.
    A temperature that is not positive stands for the arg-max.  Returns ``steps`` (int32 ``[R]``, tokens of the chain kept, the first
    one included) and ``next`` (int64 ``[R]``).  Comparisons and draws are 64-bit."""
    _need(tokens.dim() == 2 and 1 <= tokens.shape[1] <= MAX_NODES, f"tokens: [sequences, 1 to {MAX_NODES}]")
    R, C = tokens.shape
    V = _logits(logits, R, C)
    _vec(tokens, R * C, torch.int64, "tokens"), _vec(lengths, R, torch.int32, "lengths"), _vec(temperature, R, torch.float32, "temperature")
    _vec(u, R * C, torch.float32, "u"), _vec(u_draw, R, torch.float32, "u_draw")
    if C > 1:
        _need(draft_probs.dtype == torch.float32 and tuple(draft_probs.shape) == (R, C - 1, V) and (draft_probs.stride(2) == 1 or V == 1),
              "draft_probs: fp32 [R, C - 1, vocabulary]")
    else:
        draft_probs = None
    dev = logits.device
    _place(logits, tokens=tokens, lengths=lengths, draft_probs=draft_probs, temperature=temperature, u=u, u_draw=u_draw)
    steps, nxt = torch.empty(R, dtype=torch.int32, device=dev), torch.empty(R, dtype=torch.int64, device=dev)
    if R:
        call("verify_drafts", logits, logits.stride(0), logits.stride(1), tokens, lengths, draft_probs, draft_probs.stride(0) if C > 1 else 0,
             draft_probs.stride(1) if C > 1 else 0, temperature, u, u_draw, steps, nxt, _scratch(R, C, V, dev), R, C, V)
        K._count(3)
    return steps, nxt


# ------------------------------------------------------------------ commit
def _path(path: torch.Tensor, steps: torch.Tensor, positions: torch.Tensor) -> tuple[int, int]:
    _need(path.dim() == 2 and path.dtype == torch.int32 and path.is_contiguous(), "path: a contiguous int32 [sequences, nodes]")
    R, C = path.shape
    _need(1 <= C <= MAX_NODES, f"a tree has 1 to {MAX_NODES} nodes, not {C}")
    _vec(steps, R, torch.int32, "steps"), _vec(positions, R, torch.int32, "positions")
    return R, C


def kv_tree_commit(kpool, vpool, block_tables, positions, path, steps, kscale=None, vscale=None) -> None:
    """Keys and values of the accepted paths move to consecutive positions, in all layers at once: the row at ``positions[r] + path[r, i]``
    to ``positions[r] + i`` for ``i < steps[r]``.  ``kpool`` / ``vpool [layers, slots, nkv, hd]`` (with ``kscale`` / ``vscale [layers, slots, nkv]``
    int8), ``path`` and ``steps`` as :func:`verify_tree` returns them; a path's nodes are in increasing order."""
    R, C = _path(path, steps, positions)
    _need(kpool.dim() == 4 and kpool.shape == vpool.shape and kpool.dtype == vpool.dtype and kpool.is_contiguous() and vpool.is_contiguous(),
          "pools: two contiguous [layers, slots, nkv, hd]")
    L, slots, nkv, hd = kpool.shape
    row = nkv * hd * kpool.element_size()
    _need(row % 16 == 0 and kpool.data_ptr() % 16 == 0 and vpool.data_ptr() % 16 == 0, "pools: rows of a multiple of 16 bytes")
    _need((kscale is None) == (vscale is None) and (kscale is not None) == (kpool.dtype == torch.int8), "kscale and vscale go with int8 pools")
    for t in (kscale, vscale):
        _need(t is None or (t.dtype == torch.float32 and t.is_contiguous() and t.numel() == L * slots * nkv), "scales: contiguous fp32 [layers, slots, nkv]")
    _need(block_tables.dtype == torch.int32 and block_tables.dim() == 2 and block_tables.shape[0] == R and block_tables.shape[1] >= 1
          and block_tables.stride(1) == 1, "block_tables: int32 [R, pages]")
    _place(kpool, vpool=vpool, block_tables=block_tables, positions=positions, path=path, steps=steps, kscale=kscale, vscale=vscale)
    if R and L and C > 1:
        call("kv_tree_commit", kpool, vpool, kscale, vscale, block_tables, block_tables.stride(0), block_tables.shape[1], positions, path, steps,
             L, slots, row, nkv, R, C)
        K._count()


def gdn_tree_commit(state, ring, record, raw, slots, positions, path, steps, *, to_slots=None) -> None:
    """Delta-net states and convolution rings advance along the accepted paths, in all layers at once: ``state [layers, slots, nv, dk, dv]``,
    ``ring [layers, slots, 16, conv]``, ``record [layers, R, C, nv, dk + dv + 1]`` and ``raw [layers, R, C, conv]`` as ``gdn_tree`` left
    them.  Sequence ``r`` is read in slot ``slots[r]`` (< 0: unused row) and written in ``to_slots[r]`` (the same ones by default; all
    slots that are written are distinct and none of them is read for another sequence)."""
    R, C = _path(path, steps, positions)
    _need(state.dim() == 5 and state.dtype == torch.float32 and state.is_contiguous() and state.data_ptr() % 16 == 0, "state: contiguous fp32 [layers, slots, nv, dk, dv]")
    L, n, nv, dk, dv = state.shape
    _need((dk, dv) in ((128, 128), (64, 64)), f"delta-net states of {dk} x {dv}")
    conv = ring.shape[-1]
    _need(ring.dtype == torch.bfloat16 and ring.shape == (L, n, K.RING, conv) and ring.is_contiguous() and conv % 8 == 0 and ring.data_ptr() % 16 == 0,
          "ring: contiguous bf16 [layers, slots, 16, conv]")
    _need(record.dtype == torch.float32 and record.shape == (L, R, C, nv, dk + dv + 1) and record.is_contiguous(), "record: contiguous fp32 [layers, R, C, nv, dk + dv + 1]")
    _need(raw.dtype == torch.bfloat16 and raw.shape == (L, R, C, conv) and raw.is_contiguous() and raw.data_ptr() % 16 == 0, "raw: contiguous bf16 [layers, R, C, conv]")
    to = slots if to_slots is None else to_slots
    _vec(slots, R, torch.int32, "slots"), _vec(to, R, torch.int32, "to_slots")
    _place(state, ring=ring, record=record, raw=raw, slots=slots, to_slots=to, positions=positions, path=path, steps=steps)
    if R and L:
        call("gdn_tree_commit", state, ring, record, raw, slots, to, positions, path, steps, L, n, R, C, nv, dk, dv, conv)
        K._count()
