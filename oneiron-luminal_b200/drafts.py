"""Operators of speculative decoding on torch tensors: thin calls of ``include/lum_tree.h``.

A step verifies, for every sequence of a batch, a tree of drafted tokens: node 0 is the token decoding stands at, the others are guesses of what
follows their parent.  Node ``i``'s key and value lie at cache row ``prefix + i``.

    tree = DraftTree(row_start, prefix, parent, max_rows=64, max_prefix=4096)
    cache = KvMap(rows=k.shape[0], page_table=table, page_rows=64, max_seq=4160)
    out = attn_tree(q, k, v, tree, cache, n_kv_heads=8, head_dim=128)           # per layer
    path, n_accepted, next_token = tree_accept(tree, tokens, logits=logits)     # the nodes that stand, and what follows them
    kv_compact(planes, cache, tree, path, n_accepted)                           # their rows close up, in every layer

All calls are asynchronous on the current stream of the tensors' device and can be captured into a CUDA graph.  A call that cannot be made
raises :class:`LumError`; what the kernels find wrong in the arrays (a parent that is no earlier node, a page outside the pool, ...) is left out
and raised by the next :func:`status`.
"""
from __future__ import annotations

import ctypes as C

from .runtime import DraftTreeDesc, KvMapDesc, LumError, TreeAttnDesc, load_library

MAX_NODES = 256
_F32, _BF16 = 0, 2
_INVALID = -1
_REFUSED = C.c_size_t(-1).value


torch = None               # the package itself does not need it: imported by the first tensor


def _use_torch():
    global torch
    if torch is None:
        import torch as t
        torch = t


_TYPES = {}


def _types():
    if not _TYPES:
        _TYPES.update({torch.float32: _F32, torch.bfloat16: _BF16})
    return _TYPES


def _bad(why: str):
    raise LumError(_INVALID, why)


def _ints(name, t, device, dims=1, optional=False):
    """Address of a contiguous int32 tensor on ``device``."""
    if t is None and optional:
        return None
    if torch is None:
        _use_torch()
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.dim() != dims or not t.is_contiguous() or t.device != device or t.get_device() < 0:
        _bad(f"{name}: a contiguous {dims}-d int32 tensor on {device} is wanted")
    return t.data_ptr()


def _check(rc: int) -> None:
    if rc:
        raise LumError(rc, load_library().lum_last_error(None).decode())


def _stream(index: int) -> int:
    return torch._C._cuda_getCurrentRawStream(index)       # what torch.cuda.current_stream(index).cuda_stream is, at a tenth of its time


class _Here:
    """Makes the tensors' device the current one for a call, where it is not."""

    __slots__ = ("index", "before")

    def __init__(self, index):
        self.index = index

    def __enter__(self):
        self.before = torch._C._cuda_getDevice()
        if self.before != self.index:
            torch.cuda.set_device(self.index)

    def __exit__(self, *exc):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


class DraftTree:
    """The trees of a batch.  ``row_start`` [n_seq + 1], ``prefix`` [n_seq] and ``parent`` [rows of the batch] are int32 tensors on the GPU; ``slot`` [n_seq] names
    the cache slots (None: sequence s is slot s); no tree has more than ``max_rows`` nodes, no sequence more than ``max_prefix`` cached rows before it."""

    def __init__(self, row_start, prefix, parent, *, max_rows: int, max_prefix: int, slot=None):
        device = getattr(parent, "device", None)
        n_seq = prefix.numel()
        self.device, self.n_seq, self.n_rows, self.max_rows, self.tensors = device, n_seq, parent.numel(), max_rows, (row_start, prefix, parent, slot)
        self.ref = C.byref(DraftTreeDesc(_ints("row_start", row_start, device), _ints("prefix", prefix, device), _ints("parent", parent, device),
                                         None if slot is None else _ints("slot", slot, device), n_seq, self.n_rows, max_rows, max_prefix))
        if row_start.numel() != n_seq + 1 or (slot is not None and slot.numel() != n_seq):
            _bad(f"row_start has {row_start.numel()} entries, slot {n_seq if slot is None else slot.numel()}, for {n_seq} sequences")


class KvMap:
    """Where the cached rows of a slot are: ``rows`` in all, contiguous slots of ``max_seq`` rows, or pages of ``page_rows`` rows named by ``page_table``
    [slots, pages per slot]."""

    def __init__(self, rows: int, *, max_seq: int, page_table=None, page_rows: int = 0, slots: int = 0):
        self.tensors, self.rows = (page_table,), rows
        if (page_table is None) != (page_rows == 0):
            _bad("pages come with a page table")
        if page_table is None:
            self.ref = C.byref(KvMapDesc(None, rows, slots or max(1, rows // max(1, max_seq)), max_seq, 0, 0))
        else:
            self.ref = C.byref(KvMapDesc(_ints("page_table", page_table, page_table.device, dims=2), rows, page_table.shape[0], max_seq, page_rows, page_table.shape[1]))


def _rows_of(name, t, device, width, rows):
    """(address, row stride) of a tensor whose rows are ``width`` elements, dense in a row, one behind the other (a row stride of 0, of a tensor expanded along
    its rows, would mean rows without gaps to the call, far more memory than the tensor has)."""
    shape = t.shape
    if t.device != device or len(shape) < 2 or shape[0] != rows:
        _bad(f"{name}: {rows} rows on {device} are wanted, got {tuple(shape)} on {t.device}")
    if t.is_contiguous() and t.numel() == rows * width:
        return t.data_ptr(), width
    inner = 1
    for size, stride in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
        if size != 1 and stride != inner:
            _bad(f"{name}: the elements of a row must follow each other")
        inner *= size
    if inner != width:
        _bad(f"{name}: rows of {width} elements are wanted, got {tuple(t.shape[1:])}")
    if rows > 1 and t.stride(0) < width:
        _bad(f"{name}: rows {t.stride(0)} elements apart overlap, rows of {width} are wanted in a place each (an expanded tensor needs .contiguous())")
    return t.data_ptr(), (t.stride(0) if rows > 1 else width)


def _no_gradient(q, k, v, sinks):
    """There is no backward pass: a result that looks like a constant where a gradient is being recorded is refused."""
    if torch is None:
        _use_torch()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (sinks is not None and sinks.requires_grad)):
        _bad("attn_tree has no gradient: call it under torch.no_grad(), or with tensors that require none")


def attn_tree(q, k, v, tree: DraftTree, cache: KvMap, *, n_kv_heads: int, head_dim: int, scale: float = 0.0, window: int = 0, sinks=None, out=None, workspace=None):
    """Attention of the drafted nodes over their sequences' cached rows and their own ancestors.

    ``q`` [rows, heads * head_dim] (or [rows, heads, head_dim]) in bf16 or f32; ``k`` and ``v`` [cache rows, n_kv_heads * head_dim] in bf16, or in f32 with f32
    queries; rows may be strided.  ``scale`` 0: 1 / sqrt(head_dim).  ``window``: a node sees only what is fewer than so many places before its own.  ``sinks``
    [heads] f32: a logit per head that joins the softmax's denominator.  Returns ``out`` (like q; rows of no sequence are left as they were; without ``out``
    given they are not set).  ``workspace``: scratch to use (None: taken from torch); calls that may overlap need one each.  There is no gradient: tensors that
    require one are refused while gradients are recorded."""
    device, q_type, k_type = q.device, _types().get(q.dtype), _types().get(k.dtype)
    _no_gradient(q, k, v, sinks)
    if device != tree.device or q_type is None or k_type is None or v.dtype != k.dtype:
        _bad(f"attn_tree: q {q.dtype} on {device}, tree on {tree.device}, k {k.dtype}, v {v.dtype}: bf16 or f32 on one device are wanted")
    rows = tree.n_rows
    width = 1
    for size in q.shape[1:]:
        width *= size
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.dtype != q.dtype:
        _bad(f"attn_tree: out is {out.dtype}, q {q.dtype}")
    q_at, q_stride = _rows_of("q", q, device, width, rows)
    o_at, o_stride = _rows_of("out", out, device, width, rows)
    k_at, k_stride = _rows_of("k", k, device, n_kv_heads * head_dim, cache.rows)
    v_at, v_stride = _rows_of("v", v, device, n_kv_heads * head_dim, cache.rows)
    if v_stride != k_stride or width % head_dim:
        _bad(f"attn_tree: k and v rows {k_stride} and {v_stride} elements apart, q rows of {width} for heads of {head_dim}")
    s_at = None
    if sinks is not None:
        if sinks.device != device or sinks.dtype != torch.float32 or not sinks.is_contiguous() or sinks.numel() != width // head_dim:
            _bad(f"attn_tree: sinks must be {width // head_dim} contiguous f32 values on {device}")
        s_at = sinks.data_ptr()
    desc = C.byref(TreeAttnDesc(q_type, k_type, width // head_dim, n_kv_heads, head_dim, window, scale, 0, q_stride, k_stride, o_stride))
    lib = load_library()
    with _Here(device.index):
        need = lib.lum_op_attn_tree_workspace(desc, tree.ref, cache.ref)
        if need == _REFUSED:
            _check(_INVALID)
        w_at, w_bytes = None, need
        if workspace is not None:
            if not workspace.is_contiguous():
                _bad("attn_tree: the workspace must be contiguous")
            w_at, w_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        elif need:
            workspace = tree.tensors[0].new_empty(need // 4 + 1)        # (a tensor's own kind: half the time of torch.empty)
            w_at = workspace.data_ptr()
        _check(lib.lum_op_attn_tree(desc, tree.ref, cache.ref, q_at, k_at, v_at, s_at, o_at, w_at, w_bytes, _stream(device.index)))
    return out


def tree_accept(tree: DraftTree, tokens, *, logits=None, picks=None, path_len: int = 0):
    """The nodes that stand: ``(path [n_seq, path_len], n_accepted [n_seq], next_token [n_seq])``, int32.

    Node 0 stands; at a node the model picks the arg-max of its row of ``logits`` [rows, vocab] f32 (the last maximum, as the greedy sample does) or
    ``picks`` [rows] (what a sampler drew); the first child whose token (``tokens`` [rows]) is the pick stands next.  ``path`` has -1 behind the nodes that stand;
    ``next_token`` is the pick at the last of them."""
    device, n, rows = tree.device, tree.n_seq, tree.n_rows
    path_len = path_len or tree.max_rows
    t_at, k_at = _ints("tokens", tokens, device), _ints("picks", picks, device, optional=True)
    if tokens.numel() != rows or (picks is not None and picks.numel() != rows):
        _bad(f"tree_accept: {tokens.numel()} tokens for {rows} rows")
    l_at, vocab, ld = None, 0, 0
    if logits is not None:
        if logits.dtype != torch.float32 or logits.dim() != 2:
            _bad(f"tree_accept: logits must be [{rows}, vocab] f32 on {device}, got {tuple(logits.shape)} {logits.dtype}")
        vocab = logits.shape[1]
        l_at, ld = _rows_of("logits", logits, device, vocab, rows)
    lib = load_library()
    with _Here(device.index):
        need = lib.lum_op_tree_accept_workspace(tree.ref, vocab) if logits is not None else 0
        if need == _REFUSED:
            _check(_INVALID)
        # one allocation (a tensor of torch's costs a third of a launch): the scratch first, for its alignment, then the results
        room, at = tokens.new_empty(need // 4 + n * (path_len + 2)), need // 4
        path, count, after = room.as_strided((n, path_len), (path_len, 1), at), room.as_strided((n,), (1,), at + n * path_len), room.as_strided((n,), (1,), at + n * (path_len + 1))
        base = room.data_ptr()
        p_at = base + need
        _check(lib.lum_op_tree_accept(tree.ref, t_at, l_at, vocab, ld, k_at, p_at, path_len, p_at + 4 * n * path_len, p_at + 4 * n * (path_len + 1), base if need else None, need,
                                      _stream(device.index)))
    return path, count, after


def _planes(planes):
    if torch is None:
        _use_torch()
    if planes.dtype != torch.int64 or planes.dim() != 2 or planes.shape[1] != 2 or not planes.is_contiguous() or not planes.is_cuda:
        _bad("planes: a contiguous [planes, 2] int64 tensor on the GPU is wanted (address and bytes of a row)")
    return planes.data_ptr(), planes.shape[0]


def kv_planes(tensors):
    """The table of planes that :func:`kv_compact` and :func:`kv_copy` take, of 2-d (or 3-d: one plane per first index) cache tensors whose rows follow each
    other.  Made once for a cache; the tensors have to outlive it."""
    _use_torch()
    entries, device = [], None
    for t in tensors:
        for p in (t.unbind(0) if t.dim() == 3 else [t]):
            bytes_ = p.shape[1] * p.element_size()
            if p.dim() != 2 or not p.is_contiguous() or bytes_ % 16 or p.data_ptr() % 16:
                _bad("kv_planes: contiguous rows of a multiple of 16 bytes, 16-byte aligned, are wanted")
            if device is not None and p.device != device:
                _bad("kv_planes: the planes are on different devices")
            device = p.device
            entries.append([p.data_ptr(), bytes_])
    if not entries:
        _bad("kv_planes: no planes")
    return torch.tensor(entries, dtype=torch.int64).to(device)


def kv_compact(planes, cache: KvMap, tree: DraftTree, path, n_accepted) -> None:
    """Row ``prefix + path[s, i]`` of every plane becomes row ``prefix + i``, for i < n_accepted[s]."""
    p_at, n = _planes(planes)
    device = planes.device
    path_at, n_at = _ints("path", path, device, dims=2), _ints("n_accepted", n_accepted, device)
    if device != tree.device or path.shape[0] != tree.n_seq or n_accepted.numel() != tree.n_seq:
        _bad(f"kv_compact: paths of {path.shape[0]} and counts of {n_accepted.numel()} sequences for {tree.n_seq}")
    with _Here(device.index):
        _check(load_library().lum_op_kv_compact(p_at, n, cache.ref, tree.ref, path_at, path.shape[1], n_at, _stream(device.index)))


def kv_copy(planes, rows: int, spans, *, max_rows: int) -> None:
    """Copies spans of rows in every plane of ``rows`` rows: ``spans`` [n, 3] int32 of {first source row, first destination row, rows <= max_rows}.
    Destinations overlap neither each other nor a source."""
    p_at, n = _planes(planes)
    s_at = _ints("spans", spans, planes.device, dims=2)
    if spans.shape[1] != 3:
        _bad("kv_copy: spans are [n, 3]")
    with _Here(planes.device.index):
        _check(load_library().lum_op_kv_copy(p_at, n, rows, s_at, spans.shape[0], max_rows, _stream(planes.device.index)))


def status(device=None) -> None:
    """Waits for the current stream of ``device`` and raises what a kernel of these operators found wrong since the last call."""
    _use_torch()
    index = torch.device("cuda" if device is None else device).index
    index = torch.cuda.current_device() if index is None else index
    with _Here(index):
        _check(load_library().lum_op_status(_stream(index)))
