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


_BF, _F32, _I32, _I64, _I8 = torch.bfloat16, torch.float32, torch.int32, torch.int64, torch.int8
_fns: dict[str, object] = {}
# the current device, and its current stream's handle without a Stream object around it (3 us less a call)
_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def call(name: str, device: int, *args) -> None:
    """``_lib.call`` for addresses (0: none) and numbers, with the argument types declared once per entry point: these calls are a few
    microseconds on the device, and so is what surrounds them here.  Attributes of tensors cost 0.05 to 0.2 us each, so every one is
    fetched once, shapes and strides whole."""
    fn = _fns.get(name)
    if fn is None:
        fn = _lib.lib()["cb_" + name]
        fn.restype = ctypes.c_int
        fn.argtypes = [ctypes.c_float if isinstance(a, float) else ctypes.c_int64 for a in args] + [ctypes.c_int64]
        _fns[name] = fn
    rc = fn(*args, _raw_stream(device))
    if rc:
        raise _lib.KernelError(f"cb_{name} failed: {_lib.ERRORS.get(rc, 'CUDA error')} ({rc})")


def _place(anchor: torch.Tensor, *others: torch.Tensor) -> int:
    """The current device, on which all tensors have to lie (launches go to its current stream)."""
    i = anchor.get_device()
    if i < 0 or i != _device():
        _bad(f"tensors have to lie on the current CUDA device, not {anchor.device}")
    for t in others:
        if t.get_device() != i:
            _bad(f"tensors lie on {anchor.device} and on {t.device}")
    return i


def _rows(anc: torch.Tensor) -> torch.Size:
    size = anc.shape
    if len(size) != 2 or anc.dtype is not _I64 or not anc.is_contiguous():
        _bad("anc: a contiguous int64 [sequences, nodes]")
    if not 1 <= size[1] <= MAX_NODES:
        _bad(f"a tree has 1 to {MAX_NODES} nodes, not {size[1]}")
    return size


def _vec(t: torch.Tensor, n: int, dtype: torch.dtype, name: str, align: int = 1) -> int:
    """Address of a contiguous tensor of n numbers."""
    p = t.data_ptr()
    if t.dtype is not dtype or t.numel() != n or not t.is_contiguous() or p % align:
        _bad(f"{name}: {n} contiguous {dtype}" + (f" at an address of {align} bytes" if align > 1 else ""))
    return p


def _matrix(t: torch.Tensor, dtype: torch.dtype, rows: int, cols: int, step: int, align: int, what: str) -> tuple[int, int]:
    """Address and row stride of a tensor of at least rows x cols numbers; rows begin at multiples of ``step`` numbers and of ``align`` bytes."""
    size, p = t.shape, t.data_ptr()
    if t.dtype is not dtype or len(size) != 2 or p % align:
        _bad(what)
    (n, w), (ld, one) = size, t.stride()
    if n < rows or w < cols or one != 1 or ld % step or ld < cols:
        _bad(what)
    return p, ld


def _tables(t: torch.Tensor, R: int) -> tuple[int, int, int]:
    """Address, row stride and width of block tables."""
    size = t.shape
    if t.dtype is not _I32 or len(size) != 2 or size[0] != R or size[1] < 1:
        _bad("block_tables: int32 [R, pages]")
    ld, one = t.stride()
    if one != 1 and size[1] > 1:
        _bad("block_tables: int32 [R, pages]")
    return t.data_ptr(), ld, size[1]


# ------------------------------------------------------------------ attention
CTAS = 148          # pieces that the pages of all sequences are cut into: one CTA an SM


def attn_tree(q, proj, kpool, vpool, block_tables, positions, anc, out, *, nh: int, nkv: int, hd: int, kscale=None, vscale=None) -> torch.Tensor:
    """Attention of tree nodes over their sequences' pages and their own paths: ``q [R * C, nh, hd]`` normed and rotated, the nodes'
    keys and values in the pools already; ``proj`` supplies the output gate as for ``kernels.attn_prefill`` (``None``: no gate).
    ``block_tables [R, pages]`` and ``positions [R]`` (cached tokens, < 0: unused row) int32; rows without a node stay as they were.
    ``kscale`` / ``vscale``: the pools are int8.  Scores that are NaN or +inf make a row NaN; a row whose scores are all -inf, or that sees
    no page, is 0."""
    R, C = _rows(anc)
    nh, nkv, hd = int(nh), int(nkv), int(hd)
    if hd not in (64, 128, 256) or nkv < 1 or nh < 1 or nh % nkv:
        _bad(f"{nh} query heads of {hd} over {nkv} kv heads")
    nodes, width = R * C, nh * hd
    qp = _vec(q, nodes * width, _BF, "q", 16)
    op, ldo = _matrix(out, _BF, nodes, width, 8, 16, "out: bf16 [R * C, nh * hd] in 16-byte rows")
    pp, ldp = (0, 0) if proj is None else _matrix(proj, _BF, nodes, 2 * width, 8, 16, "proj: bf16 rows that begin with (q | gate) of every head, 16 bytes each")
    slots = kpool.shape[0]
    kv, size = _BF if kscale is None else _I8, slots * nkv * hd
    if slots % K.BLOCK or kpool.shape != (slots, nkv, hd):
        _bad(f"kpool: [pages * {K.BLOCK}, {nkv}, {hd}]")
    if vpool.shape != kpool.shape:
        _bad(f"vpool: {list(kpool.shape)} as kpool")
    kp, vp = _vec(kpool, size, kv, "kpool", 16), _vec(vpool, size, kv, "vpool", 16)
    if (kscale is None) != (vscale is None):
        _bad("kscale and vscale go together")
    tp, ldt, pages = _tables(block_tables, R)
    posp = _vec(positions, R, _I32, "positions")
    ksp = vsp = 0
    if kscale is not None:
        ksp, vsp = _vec(kscale, slots * nkv, _F32, "scales of keys"), _vec(vscale, slots * nkv, _F32, "scales of values")
        _place(kscale, vscale)
    i = _place(q, kpool, vpool, block_tables, positions, anc, out)
    if proj is not None:
        _place(proj)
    if R == 0:
        return out
    rows, status = C * (nh // nkv), K._status.get(i)
    if status is None:
        status = K.status_word(q.device)
    part = torch.empty((CTAS * min(rows, 128) + R * nkv * (rows if rows <= 128 else -(-rows // 256) * 256)) * (hd + 2) + 1, dtype=_F32, device=q.device)
    call("attn_tree", i, qp, pp, ldp, kp, vp, slots, ksp, vsp, tp, ldt, pages, posp, anc.data_ptr(), op, ldo, part.data_ptr(), CTAS, R, C, nh, nkv, hd,
         status.data_ptr())
    K._count(2)
    return out


# ------------------------------------------------------------------ gated delta net
def gdn_tree(proj, conv_w, A_log, dt_bias, norm_w, ring, state, slots, positions, anc, out, record, raw, *, nk: int, nv: int, dk: int, dv: int,
             eps: float, gate_sigmoid: bool = False) -> torch.Tensor:
    """The layer of ``kernels.gdn_decode`` over the nodes of trees: ``proj [R * C, ...]`` raw projection rows, ``state [slots, nv, dk, dv]``
    and ``ring [slots, 16, conv]`` of the sequences (read, not written), ``slots [R]`` (< 0: unused row) and ``positions [R]`` int32.
    ``record [R, C, nv, dk + dv + 1]`` (fp32: key, update, decay) and ``raw [R, C, conv]`` are what ``gdn_tree_commit`` replays."""
    R, C = _rows(anc)
    nk, nv, dk, dv = int(nk), int(nv), int(dk), int(dv)
    if (dk, dv) not in ((128, 128), (64, 64)) or nk < 1 or nv < 1 or nv % nk:
        _bad(f"delta-net heads {nk} / {nv} of {dk} x {dv}")
    nodes, conv, width = R * C, 2 * nk * dk + nv * dv, nv * dv
    pp, ldp = _matrix(proj, _BF, nodes, conv + width + 2 * nv, 8, 16, "proj: bf16 rows q | k | v | z | b | a of a multiple of 16 bytes")
    op, ldo = _matrix(out, _BF, nodes, width, 4, 8, "out: bf16 [R * C, nv * dv] in 8-byte rows")
    n = state.shape[0]
    sp, rp = _vec(state, n * width * dk, _F32, "state", 16), _vec(ring, n * K.RING * conv, _BF, "ring", 16)
    if state.shape != (n, nv, dk, dv) or ring.shape != (n, K.RING, conv):
        _bad(f"state: [slots, {nv}, {dk}, {dv}]; ring: [slots, {K.RING}, {conv}]")
    wp, Ap, bp, np_ = _vec(conv_w, conv * 4, _F32, "conv_w", 16), _vec(A_log, nv, _F32, "A_log"), _vec(dt_bias, nv, _F32, "dt_bias"), _vec(norm_w, dv, _F32, "norm_w", 16)
    slp, posp = _vec(slots, R, _I32, "slots"), _vec(positions, R, _I32, "positions")
    recp, rawp = _vec(record, nodes * nv * (dk + dv + 1), _F32, "record"), _vec(raw, nodes * conv, _BF, "raw", 16)
    i = _place(proj, conv_w, A_log, dt_bias, norm_w, ring, state, slots, positions, anc, out, record, raw)
    if R:
        rows = torch.empty(nodes * conv, dtype=_F32, device=proj.device) if C > 8 else None      # few nodes: one kernel
        call("gdn_tree", i, pp, ldp, wp, Ap, bp, np_, rp, sp, slp, posp, anc.data_ptr(), op, ldo, recp, rawp, 0 if rows is None else rows.data_ptr(), n, R, C, nk, nv, dk, dv,
             float(eps), int(gate_sigmoid))
        K._count(1 if rows is None else 2)
    return out


# ------------------------------------------------------------------ verification
@functools.lru_cache(maxsize=256)
def _scratch_words(R: int, C: int, V: int) -> int:
    fn = _lib.lib().cb_verify_scratch
    fn.restype = ctypes.c_int64
    return int(fn(ctypes.c_int64(R), ctypes.c_int64(C), ctypes.c_int64(V))) // 8 + 1


def _logits(t: torch.Tensor, R: int, C: int) -> tuple[int, int, int, int]:
    """Address, sequence and node stride, vocabulary."""
    size = t.shape
    if t.dtype is not _F32 or len(size) != 3 or size[0] != R or size[1] != C or size[2] < 1:
        _bad("logits: fp32 [R, C, vocabulary]")
    lds, ldr, one = t.stride()
    if one != 1 and size[2] != 1:
        _bad("logits: fp32 [R, C, vocabulary] with neighbouring entries")
    if R * C > 65535:
        _bad(f"{R} x {C} rows of logits")
    return t.data_ptr(), lds, ldr, size[2]


def verify_tree(logits, tokens, anc, temperature, u) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The path that the request's own tokens take through its tree of drafts.

    The token of a node is drawn from ``softmax(logits[r, j] / temperature[r])`` by inverse CDF with ``u[r, depth of j]``, or is the arg-max
    (lowest index) where the temperature is not positive; from node 0 on the first child that carries the token (``tokens [R, C]``
    int64) is next.  Returns ``path`` (int32 ``[R, C]``, -1 behind its end), ``steps`` (int32 ``[R]``, nodes on the path) and ``next``
    (int64 ``[R]``, the token drawn at its end): the new tokens are those of the path behind node 0, then ``next``, the ones that
    one-node trees draw one by one with the same uniforms.  Draws are 64-bit (``kernels.sample`` sums in 32 bits and draws another token in
    0.3 to 2.6 % of 151936-token draws).  A sequence whose node 0 is none gets 0 steps and token -1."""
    R, C = _rows(anc)
    lp, lds, ldr, V = _logits(logits, R, C)
    tp, Tp, up = _vec(tokens, R * C, _I64, "tokens"), _vec(temperature, R, _F32, "temperature"), _vec(u, R * C, _F32, "u")
    i, dev = _place(logits, tokens, anc, temperature, u), logits.device
    path, steps, nxt = torch.empty(R, C, dtype=_I32, device=dev), torch.empty(R, dtype=_I32, device=dev), anc.new_empty(R)
    if R:
        scratch = anc.new_empty(_scratch_words(R, C, V))
        call("verify_tree", i, lp, lds, ldr, tp, anc.data_ptr(), Tp, up, path.data_ptr(), steps.data_ptr(), nxt.data_ptr(), scratch.data_ptr(), R, C, V)
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
    size = tokens.shape
    if len(size) != 2 or not 1 <= size[1] <= MAX_NODES:
        _bad(f"tokens: [sequences, 1 to {MAX_NODES}]")
    R, C = size
    lp, lds, ldr, V = _logits(logits, R, C)
    tp, np_, Tp = _vec(tokens, R * C, _I64, "tokens"), _vec(lengths, R, _I32, "lengths"), _vec(temperature, R, _F32, "temperature")
    up, dp = _vec(u, R * C, _F32, "u"), _vec(u_draw, R, _F32, "u_draw")
    qp = qs = qr = 0
    if C > 1:
        if draft_probs is None or draft_probs.dtype is not _F32 or draft_probs.shape != (R, C - 1, V):
            _bad("draft_probs: fp32 [R, C - 1, vocabulary]")
        qs, qr, one = draft_probs.stride()
        if one != 1 and V != 1:
            _bad("draft_probs: fp32 [R, C - 1, vocabulary] with neighbouring entries")
        qp = draft_probs.data_ptr()
        _place(draft_probs)
    i = _place(logits, tokens, lengths, temperature, u, u_draw)
    steps, nxt = torch.empty(R, dtype=_I32, device=logits.device), tokens.new_empty(R)
    if R:
        scratch = tokens.new_empty(_scratch_words(R, C, V))
        call("verify_drafts", i, lp, lds, ldr, tp, np_, qp, qs, qr, Tp, up, dp, steps.data_ptr(), nxt.data_ptr(), scratch.data_ptr(), R, C, V)
        K._count(2)
    return steps, nxt


# ------------------------------------------------------------------ commit
def _path(path: torch.Tensor) -> torch.Size:
    size = path.shape
    if len(size) != 2 or path.dtype is not _I32 or not path.is_contiguous():
        _bad("path: a contiguous int32 [sequences, nodes]")
    if not 1 <= size[1] <= MAX_NODES:
        _bad(f"a tree has 1 to {MAX_NODES} nodes, not {size[1]}")
    return size


def kv_tree_commit(kpool, vpool, block_tables, positions, path, steps, kscale=None, vscale=None) -> None:
    """Keys and values of the accepted paths move to consecutive positions, in all layers at once: the row at ``positions[r] + path[r, i]``
    to ``positions[r] + i`` for ``i < steps[r]``.  ``kpool`` / ``vpool [layers, slots, nkv, hd]`` (with ``kscale`` / ``vscale [layers, slots, nkv]``
    int8), ``path`` and ``steps`` as :func:`verify_tree` returns them (node 0 first, in increasing order).  Pages that are
    written belong to one sequence alone."""
    R, C = _path(path)
    size, kv = kpool.shape, kpool.dtype
    if len(size) != 4 or vpool.shape != size or kv is not vpool.dtype or not kpool.is_contiguous() or not vpool.is_contiguous():
        _bad("pools: two contiguous [layers, slots, nkv, hd]")
    L, slots, nkv, hd = size
    row, kp, vp = nkv * hd * kpool.element_size(), kpool.data_ptr(), vpool.data_ptr()
    if row % 16 or row == 0 or (kp | vp) % 16:
        _bad("pools: rows of a multiple of 16 bytes")
    if (kscale is None) != (vscale is None) or (kscale is None) == (kv is _I8):
        _bad("kscale and vscale go with int8 pools")
    stp, posp, (tp, ldt, pages) = _vec(steps, R, _I32, "steps"), _vec(positions, R, _I32, "positions"), _tables(block_tables, R)
    i = _place(kpool, vpool, block_tables, positions, path, steps)
    ksp = vsp = 0
    if kscale is not None:
        ksp, vsp = _vec(kscale, L * slots * nkv, _F32, "scales of keys"), _vec(vscale, L * slots * nkv, _F32, "scales of values")
        _place(kscale, vscale)
    if R and L and C > 1:
        call("kv_tree_commit", i, kp, vp, ksp, vsp, tp, ldt, pages, posp, path.data_ptr(), stp, L, slots, row, nkv, R, C)
        K._count()


def gdn_tree_commit(state, ring, record, raw, slots, positions, path, steps, *, to_slots=None) -> None:
    """Delta-net states and convolution rings advance along the accepted paths, in all layers at once: ``state [layers, slots, nv, dk, dv]``,
    ``ring [layers, slots, 16, conv]``, ``record [layers, R, C, nv, dk + dv + 1]`` and ``raw [layers, R, C, conv]`` as ``gdn_tree`` left
    them.  Sequence ``r`` is read in slot ``slots[r]`` (< 0: unused row) and written in ``to_slots[r]`` (the same ones by default; all
    slots that are written are distinct and none of them is read for another sequence)."""
    R, C = _path(path)
    size = state.shape
    if len(size) != 5 or state.dtype is not _F32 or not state.is_contiguous():
        _bad("state: contiguous fp32 [layers, slots, nv, dk, dv]")
    L, n, nv, dk, dv = size
    if (dk, dv) not in ((128, 128), (64, 64)):
        _bad(f"delta-net states of {dk} x {dv}")
    conv = ring.shape[-1]
    if conv % 8 or ring.shape != (L, n, K.RING, conv) or record.shape != (L, R, C, nv, dk + dv + 1) or raw.shape != (L, R, C, conv):
        _bad("ring: [layers, slots, 16, conv], record: [layers, R, C, nv, dk + dv + 1], raw: [layers, R, C, conv]")
    sp, rp = state.data_ptr(), _vec(ring, L * n * K.RING * conv, _BF, "ring", 16)
    if sp % 16:
        _bad("state: a 16-byte address")
    recp, rawp = _vec(record, L * R * C * nv * (dk + dv + 1), _F32, "record"), _vec(raw, L * R * C * conv, _BF, "raw", 16)
    slp, stp, posp = _vec(slots, R, _I32, "slots"), _vec(steps, R, _I32, "steps"), _vec(positions, R, _I32, "positions")
    top = slp if to_slots is None else _vec(to_slots, R, _I32, "to_slots")
    i = _place(state, ring, record, raw, slots, positions, path, steps)
    if to_slots is not None:
        _place(to_slots)
    if R and L:
        call("gdn_tree_commit", i, sp, rp, recp, rawp, slp, top, posp, path.data_ptr(), stp, L, n, R, C, nv, dk, dv, conv)
        K._count()
