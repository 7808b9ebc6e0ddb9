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
import functools

import torch

from . import _lib
from . import kernels as K

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


def _bad(what: str) -> None:
    raise ValueError(what)


_fns: dict[str, object] = {}
_PLAIN = (int, float)
# the current stream's handle without a Stream object around it (3 us less a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def call(name: str, *args) -> None:
    """``_lib.call`` with the argument types declared once per entry point (pointers, 64-bit integers, floats): these calls are a few
    microseconds on the device, and converting thirty arguments one by one takes longer than that."""
    fn = _fns.get(name)
    if fn is None:
        fn = _fns[name] = _lib.lib()["cb_" + name]
        fn.restype = ctypes.c_int
        fn.argtypes = [ctypes.c_float if isinstance(a, float) else ctypes.c_int64 if isinstance(a, int) else ctypes.c_void_p for a in args] + [ctypes.c_void_p]
    rc = fn(*[a if a is None or a.__class__ in _PLAIN else a.data_ptr() for a in args], _raw_stream(torch.cuda.current_device()))
    if rc:
        raise _lib.KernelError(f"cb_{name} failed: {_lib.ERRORS.get(rc, 'CUDA error')} ({rc})")


def _place(anchor: torch.Tensor, *others: torch.Tensor | None) -> None:
    """All tensors on the anchor's device, which has to be the current one (launches go to its current stream)."""
    i = anchor.get_device()
    if i < 0 or i != torch.cuda.current_device():
        _bad(f"tensors have to lie on the current CUDA device, not {anchor.device}")
    for t in others:
        if t is not None and t.get_device() != i:
            _bad(f"tensors lie on {anchor.device} and on {t.device}")


def _rows(anc: torch.Tensor) -> tuple[int, int]:
    if anc.dim() != 2 or anc.dtype != torch.int64 or not anc.is_contiguous():
        _bad("anc: a contiguous int64 [sequences, nodes]")
    R, C = anc.shape
    if not 1 <= C <= MAX_NODES:
        _bad(f"a tree has 1 to {MAX_NODES} nodes, not {C}")
    return R, C


def _vec(t: torch.Tensor, n: int, dtype: torch.dtype, name: str) -> None:
    if t.dtype != dtype or t.numel() != n or not t.is_contiguous():
        _bad(f"{name}: {n} contiguous {dtype}")


def _tables(t: torch.Tensor, R: int) -> None:
    if t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] != R or t.shape[1] < 1 or t.stride(1) != 1:
        _bad("block_tables: int32 [R, pages]")


# ------------------------------------------------------------------ attention
CTAS = 148          # pieces that the pages of all sequences are cut into: one CTA an SM


def attn_tree(q, proj, kpool, vpool, block_tables, positions, anc, out, *, nh: int, nkv: int, hd: int, kscale=None, vscale=None) -> torch.Tensor:
    """Attention of tree nodes over their sequences' pages and their own paths: ``q [R * C, nh, hd]`` normed and rotated, the nodes'
    keys and values in the pools already; ``proj`` supplies the output gate as for ``kernels.attn_prefill`` (``None``: no gate).
    ``block_tables [R, pages]`` and ``positions [R]`` (cached tokens, < 0: unused row) int32; rows without a node stay as they were.
    ``kscale`` / ``vscale``: the pools are int8."""
    R, C = _rows(anc)
    if hd not in (64, 128, 256) or nkv < 1 or nh < 1 or nh % nkv:
        _bad(f"{nh} query heads of {hd} over {nkv} kv heads")
    bf = torch.bfloat16
    if q.dtype != bf or not q.is_contiguous() or q.numel() != R * C * nh * hd or q.data_ptr() % 16:
        _bad("q: contiguous bf16 [R * C, nh, hd]")
    if (out.dtype != bf or out.dim() != 2 or out.shape[0] < R * C or out.shape[1] < nh * hd or out.stride(1) != 1 or out.stride(0) % 8
            or out.stride(0) < nh * hd or out.data_ptr() % 16):
        _bad("out: bf16 [R * C, nh * hd] in 16-byte rows")
    if proj is not None and (proj.dtype != bf or proj.dim() != 2 or proj.shape[0] < R * C or proj.shape[1] < 2 * nh * hd or proj.stride(1) != 1
                             or proj.stride(0) % 8 or proj.data_ptr() % 16):
        _bad("proj: bf16 rows that begin with (q | gate) of every head")
    kv, slots = torch.int8 if kscale is not None else bf, kpool.shape[0]
    for t, name in ((kpool, "kpool"), (vpool, "vpool")):
        if t.dtype != kv or t.shape != (slots, nkv, hd) or not t.is_contiguous() or t.data_ptr() % 16 or slots % K.BLOCK:
            _bad(f"{name}: contiguous {kv} [pages * {K.BLOCK}, {nkv}, {hd}]")
    if (kscale is None) != (vscale is None):
        _bad("kscale and vscale go together")
    if kscale is not None:
        for t in (kscale, vscale):
            if t.dtype != torch.float32 or not t.is_contiguous() or t.numel() != slots * nkv:
                _bad("scales: contiguous fp32 [slots, nkv]")
    _tables(block_tables, R)
    _vec(positions, R, torch.int32, "positions")
    _place(q, proj, kpool, vpool, block_tables, positions, anc, out, kscale, vscale)
    if R == 0:
        return out
    rows, status = C * (nh // nkv), K._status.get(q.get_device())
    part = torch.empty((CTAS + R * nkv * -(-rows // 128)) * min(rows, 128) * (hd + 2), dtype=torch.float32, device=q.device)
    call("attn_tree", q, proj, proj.stride(0) if proj is not None else 0, kpool, vpool, slots, kscale, vscale, block_tables, block_tables.stride(0),
         block_tables.shape[1], positions, anc, out, out.stride(0), part, CTAS, R, C, nh, nkv, hd, status if status is not None else K.status_word(q.device))
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
    if (dk, dv) not in ((128, 128), (64, 64)) or nk < 1 or nv < 1 or nv % nk:
        _bad(f"delta-net heads {nk} / {nv} of {dk} x {dv}")
    if (proj.dtype != bf or proj.dim() != 2 or proj.shape[0] < R * C or proj.shape[1] < conv + nv * dv + 2 * nv or proj.stride(1) != 1
            or proj.stride(0) % 8 or proj.data_ptr() % 16):
        _bad("proj: bf16 rows q | k | v | z | b | a of a multiple of 16 bytes")
    if (out.dtype != bf or out.dim() != 2 or out.shape[0] < R * C or out.shape[1] < nv * dv or out.stride(1) != 1 or out.stride(0) % 4
            or out.stride(0) < nv * dv or out.data_ptr() % 8):
        _bad("out: bf16 [R * C, nv * dv] in 8-byte rows")
    n = state.shape[0]
    if state.dtype != f32 or state.shape != (n, nv, dk, dv) or not state.is_contiguous() or state.data_ptr() % 16:
        _bad("state: contiguous fp32 [slots, nv, dk, dv]")
    if ring.dtype != bf or ring.shape != (n, K.RING, conv) or not ring.is_contiguous() or ring.data_ptr() % 16:
        _bad("ring: contiguous bf16 [slots, 16, conv]")
    _vec(conv_w, conv * 4, f32, "conv_w"), _vec(A_log, nv, f32, "A_log"), _vec(dt_bias, nv, f32, "dt_bias"), _vec(norm_w, dv, f32, "norm_w")
    if (conv_w.data_ptr() | norm_w.data_ptr()) % 16:
        _bad("conv_w, norm_w: 16-byte addresses")
    _vec(slots, R, torch.int32, "slots"), _vec(positions, R, torch.int32, "positions")
    _vec(record, R * C * nv * (dk + dv + 1), f32, "record"), _vec(raw, R * C * conv, bf, "raw")
    if raw.data_ptr() % 16:
        _bad("raw: a 16-byte address")
    _place(proj, conv_w, A_log, dt_bias, norm_w, ring, state, slots, positions, anc, out, record, raw)
    if R:
        rows = torch.empty(R * C * conv, dtype=f32, device=proj.device)
        call("gdn_tree", proj, proj.stride(0), conv_w, A_log, dt_bias, norm_w, ring, state, slots, positions, anc, out, out.stride(0), record, raw, rows,
             n, R, C, nk, nv, dk, dv, float(eps), int(gate_sigmoid))
        K._count(2)
    return out


# ------------------------------------------------------------------ verification
@functools.lru_cache(maxsize=256)
def _scratch_bytes(R: int, C: int, V: int) -> int:
    fn = _lib.lib().cb_verify_scratch
    fn.restype = ctypes.c_int64
    return int(fn(ctypes.c_int64(R), ctypes.c_int64(C), ctypes.c_int64(V)))


def _logits(logits: torch.Tensor, R: int, C: int) -> int:
    if logits.dtype != torch.float32 or logits.dim() != 3 or logits.shape[0] != R or logits.shape[1] != C or logits.shape[2] < 1 or (
            logits.stride(2) != 1 and logits.shape[2] != 1):
        _bad("logits: fp32 [R, C, vocabulary]")
    if R * C > 65535:
        _bad(f"{R} x {C} rows of logits")
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
    _place(logits, tokens, anc, temperature, u)
    path = torch.empty(R, C, dtype=torch.int32, device=dev)
    steps, nxt = torch.empty(R, dtype=torch.int32, device=dev), torch.empty(R, dtype=torch.int64, device=dev)
    if R:
        call("verify_tree", logits, logits.stride(0), logits.stride(1), tokens, anc, temperature, u, path, steps, nxt, torch.empty(_scratch_bytes(R, C, V), dtype=torch.uint8, device=dev), R, C, V)
        K._count(2)
    return path, steps, nxt


def verify_drafts(logits, tokens, lengths, draft_probs, temperature, u, u_draw) -> tuple[torch.Tensor, torch.Tensor]:
    """How much of a chain of drafts that were drawn from ``draft_probs`` is kept, and the token after it.

    Row ``r`` is a chain of ``lengths[r]`` (int32; 0: unused row) of the ``C`` tokens ``tokens[r]``: the token that was sampled last,
    then drafts, draft ``i`` drawn from ``draft_probs[r, i - 1]`` (fp32 ``[R, C - 1, vocabulary]``, each summing to one).  With
    ``p = softmax(logits / temperature)`` draft ``i`` is kept while ``u[r, i] q(x) < p(x)``; the next token is drawn with ``u_draw[r]`` from
    ``max(p - q, 0)`` of the first draft that is not, or from ``p`` behind the last one, so that the tokens are distributed as the target's.
    A temperature that is not positive stands for the arg-max.  Returns ``steps`` (int32 ``[R]``, tokens of the chain kept, the first
    one included) and ``next`` (int64 ``[R]``).  Comparisons and draws are 64-bit."""
    if tokens.dim() != 2 or not 1 <= tokens.shape[1] <= MAX_NODES:
        _bad(f"tokens: [sequences, 1 to {MAX_NODES}]")
    R, C = tokens.shape
    V = _logits(logits, R, C)
    _vec(tokens, R * C, torch.int64, "tokens"), _vec(lengths, R, torch.int32, "lengths"), _vec(temperature, R, torch.float32, "temperature")
    _vec(u, R * C, torch.float32, "u"), _vec(u_draw, R, torch.float32, "u_draw")
    if C > 1:
        if draft_probs.dtype != torch.float32 or draft_probs.shape != (R, C - 1, V) or (draft_probs.stride(2) != 1 and V != 1):
            _bad("draft_probs: fp32 [R, C - 1, vocabulary]")
    else:
        draft_probs = None
    dev = logits.device
    _place(logits, tokens, lengths, draft_probs, temperature, u, u_draw)
    steps, nxt = torch.empty(R, dtype=torch.int32, device=dev), torch.empty(R, dtype=torch.int64, device=dev)
    if R:
        call("verify_drafts", logits, logits.stride(0), logits.stride(1), tokens, lengths, draft_probs, draft_probs.stride(0) if C > 1 else 0,
             draft_probs.stride(1) if C > 1 else 0, temperature, u, u_draw, steps, nxt, torch.empty(_scratch_bytes(R, C, V), dtype=torch.uint8, device=dev), R, C, V)
        K._count(2)
    return steps, nxt


# ------------------------------------------------------------------ commit
def _path(path: torch.Tensor, steps: torch.Tensor, positions: torch.Tensor) -> tuple[int, int]:
    if path.dim() != 2 or path.dtype != torch.int32 or not path.is_contiguous():
        _bad("path: a contiguous int32 [sequences, nodes]")
    R, C = path.shape
    if not 1 <= C <= MAX_NODES:
        _bad(f"a tree has 1 to {MAX_NODES} nodes, not {C}")
    _vec(steps, R, torch.int32, "steps"), _vec(positions, R, torch.int32, "positions")
    return R, C


def kv_tree_commit(kpool, vpool, block_tables, positions, path, steps, kscale=None, vscale=None) -> None:
    """Keys and values of the accepted paths move to consecutive positions, in all layers at once: the row at ``positions[r] + path[r, i]``
    to ``positions[r] + i`` for ``i < steps[r]``.  ``kpool`` / ``vpool [layers, slots, nkv, hd]`` (with ``kscale`` / ``vscale [layers, slots, nkv]``
    int8), ``path`` and ``steps`` as :func:`verify_tree` returns them; a path's nodes are in increasing order."""
    R, C = _path(path, steps, positions)
    if kpool.dim() != 4 or kpool.shape != vpool.shape or kpool.dtype != vpool.dtype or not kpool.is_contiguous() or not vpool.is_contiguous():
        _bad("pools: two contiguous [layers, slots, nkv, hd]")
    L, slots, nkv, hd = kpool.shape
    row = nkv * hd * kpool.element_size()
    if row % 16 or row == 0 or kpool.data_ptr() % 16 or vpool.data_ptr() % 16:
        _bad("pools: rows of a multiple of 16 bytes")
    if (kscale is None) != (vscale is None) or (kscale is not None) != (kpool.dtype == torch.int8):
        _bad("kscale and vscale go with int8 pools")
    if kscale is not None:
        for t in (kscale, vscale):
            if t.dtype != torch.float32 or not t.is_contiguous() or t.numel() != L * slots * nkv:
                _bad("scales: contiguous fp32 [layers, slots, nkv]")
    _tables(block_tables, R)
    _place(kpool, vpool, block_tables, positions, path, steps, kscale, vscale)
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
    if state.dim() != 5 or state.dtype != torch.float32 or not state.is_contiguous() or state.data_ptr() % 16:
        _bad("state: contiguous fp32 [layers, slots, nv, dk, dv]")
    L, n, nv, dk, dv = state.shape
    if (dk, dv) not in ((128, 128), (64, 64)):
        _bad(f"delta-net states of {dk} x {dv}")
    conv = ring.shape[-1]
    if ring.dtype != torch.bfloat16 or ring.shape != (L, n, K.RING, conv) or not ring.is_contiguous() or conv % 8 or ring.data_ptr() % 16:
        _bad("ring: contiguous bf16 [layers, slots, 16, conv]")
    if record.dtype != torch.float32 or record.shape != (L, R, C, nv, dk + dv + 1) or not record.is_contiguous():
        _bad("record: contiguous fp32 [layers, R, C, nv, dk + dv + 1]")
    if raw.dtype != torch.bfloat16 or raw.shape != (L, R, C, conv) or not raw.is_contiguous() or raw.data_ptr() % 16:
        _bad("raw: contiguous bf16 [layers, R, C, conv]")
    to = slots if to_slots is None else to_slots
    _vec(slots, R, torch.int32, "slots"), _vec(to, R, torch.int32, "to_slots")
    _place(state, ring, record, raw, slots, to, positions, path, steps)
    if R and L:
        call("gdn_tree_commit", state, ring, record, raw, slots, to, positions, path, steps, L, n, R, C, nv, dk, dv, conv)
        K._count()
