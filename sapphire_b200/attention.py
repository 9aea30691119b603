"""Rotary positions, the paged key-value cache and the attention of one new
token, to all pages, to selected ones or behind a shared prefix (include/sapphire_attention.h) from Python.

Buffers are CUDA tensors of the context's GPU (torch tensors, or anything with
data_ptr(), shape, stride() and dtype); work is enqueued on the context's stream
and the calls return without waiting.  What only the device can see (a page or a
length outside the cache) is raised by the next Context.synchronize().
"""
from __future__ import annotations

import ctypes as C

from . import SapphireError, _lib, addr, lib
from ._lib import (DTYPE_BF16, DTYPE_F16, DTYPE_F32, DTYPE_NAMES, AttentionArgs, AttentionSharedArgs, KvArgs,
                   KvCacheStruct, KvSelectArgs, RopeArgs, RopeConfig)

_BY_NAME = {name.lower(): dt for dt, name in DTYPE_NAMES.items()}
_IO = {"float32": DTYPE_F32, "bfloat16": DTYPE_BF16, "float16": DTYPE_F16}
_io_seen: dict = {}          # dtype object -> tensor_dtype_t
_int_seen: dict = {}         # dtype object -> whether it is int32

LAYOUTS = {"half": 0, "interleaved": 1}
SCALINGS = {"none": 0, "linear": 1, "banded": 2, "yarn": 3}


def _dtype(dt) -> int:
    """tensor_dtype_t of a DTYPE_* number or its name."""
    if isinstance(dt, str):
        if dt.lower() not in _BY_NAME:
            raise SapphireError(f"unknown type {dt!r}")
        return _BY_NAME[dt.lower()]
    return dt


def _io(x, what: str) -> int:
    dt = _io_seen.get(x.dtype)
    if dt is None:
        dt = _IO.get(str(x.dtype).rsplit(".", 1)[-1])
        if dt is None:
            raise SapphireError(f"{what} must be float32, bfloat16 or float16, not {x.dtype}")
        _io_seen[x.dtype] = dt
    return dt


def _heads(x, what: str, rows: int | None, heads: int | None, dim: int, dt: int) -> tuple[int, int, int]:
    """(address, row stride, head stride) of x [rows, heads, dim] of type dt."""
    shape = x.shape
    if len(shape) != 3 or shape[2] != dim or (rows is not None and shape[0] != rows) or \
            (heads is not None and shape[1] != heads):
        want = ["any" if n is None else n for n in (rows, heads, dim)]
        raise SapphireError(f"{what} has shape {tuple(shape)}, not {want}")
    if _io_seen.get(x.dtype) != dt and _io(x, what) != dt:
        raise SapphireError(f"the tensors of a call must have one type: {what} is {x.dtype}")
    a, b, c = x.stride()
    if c != 1:
        raise SapphireError(f"{what}: the last dimension must be contiguous")
    # To the library a stride of 0 is a contiguous one.
    if (a == 0 and shape[0] > 1) or (b == 0 and shape[1] > 1):
        raise SapphireError(f"{what}: broadcast dimensions are not supported")
    return x.data_ptr(), a, b


def _int32(x, what: str) -> None:
    """Raises unless x is int32."""
    ok = _int_seen.get(x.dtype)
    if ok is None:
        ok = _int_seen[x.dtype] = str(x.dtype).rsplit(".", 1)[-1] == "int32"
    if not ok:
        raise SapphireError(f"{what} must be int32, not {x.dtype}")


def _ints(x, what: str, n: int | None):
    _int32(x, what)
    if n is not None and (len(x.shape) != 1 or x.shape[0] != n):
        raise SapphireError(f"{what} has shape {tuple(x.shape)}, not [{n}]")
    if not x.is_contiguous():
        raise SapphireError(f"{what} must be contiguous")
    return x.data_ptr()


def _table(x, sequences: int):
    """(address, pages a sequence, row stride) of an int32 page table [sequences, pages]."""
    _int32(x, "page_table")
    if len(x.shape) != 2 or x.shape[0] != sequences:
        raise SapphireError(f"page_table has shape {tuple(x.shape)}, not [{sequences}, pages]")
    if not x.is_contiguous():
        raise SapphireError("page_table must be contiguous")
    return x.data_ptr(), x.shape[1]


def _head_table(x, sequences: int, kv_heads: int, what: str = "page_table"):
    """(address, pages) of an int32 page table [sequences, kv_heads, pages]."""
    _int32(x, what)
    if len(x.shape) != 3 or x.shape[0] != sequences or x.shape[1] != kv_heads:
        raise SapphireError(f"{what} has shape {tuple(x.shape)}, not [{sequences}, {kv_heads}, pages]")
    if not x.is_contiguous():
        raise SapphireError(f"{what} must be contiguous")
    return x.data_ptr(), x.shape[2]


class Rope:
    """A rotation plan (sapphire_rope_create).

    layout 'half' pairs values i and i + rot_dim/2, 'interleaved' 2i and 2i + 1;
    scaling 'none', 'linear', 'banded' or 'yarn' as the header defines them."""

    def __init__(self, ctx, head_dim: int, rot_dim: int | None = None, layout: str = "half", theta: float = 1e4,
                 scaling: str = "none", factor: float = 1.0, original_context: int = 0, turns_slow: float = 0.0,
                 turns_fast: float = 0.0, attention_factor: float = 0.0):
        self.handle = None
        if layout not in LAYOUTS or scaling not in SCALINGS:
            raise SapphireError(f"unknown layout {layout!r} or scaling {scaling!r}")
        self.ctx, self.head_dim = ctx, head_dim
        cfg = RopeConfig(head_dim, head_dim if rot_dim is None else rot_dim, LAYOUTS[layout], SCALINGS[scaling], theta,
                         factor, original_context, turns_slow, turns_fast, attention_factor)
        if rot_dim == 0:
            raise SapphireError("rot_dim must be positive")
        self.handle = lib.sapphire_rope_create(ctx.handle, C.byref(cfg))
        if not self.handle:
            raise SapphireError(f"sapphire_rope_create failed: {ctx.last_error}")

    def apply(self, positions, q=None, k=None, q_out=None, k_out=None, inverse: bool = False) -> None:
        """Turn q and / or k [tokens, heads, head_dim] into q_out and k_out (in
        place where these are None)."""
        x = q if q is not None else k
        if x is None:
            return
        if not self.handle or not self.ctx.handle:
            raise SapphireError("the rotation plan or its context is closed")
        n, dim = x.shape[0], self.head_dim
        dt = _io_seen.get(x.dtype)
        if dt is None:
            dt = _io(x, "q" if q is not None else "k")
        qh = kh = qp = kp = qop = kop = qt = qs = kt = ks = qot = qos = kot = kos = 0
        if q is not None:
            qh = q.shape[1]
            qp, qt, qs = _heads(q, "q", n, None, dim, dt)
            qop, qot, qos = (qp, qt, qs) if q_out is None else _heads(q_out, "q_out", n, qh, dim, dt)
        if k is not None:
            kh = k.shape[1]
            kp, kt, ks = _heads(k, "k", n, None, dim, dt)
            kop, kot, kos = (kp, kt, ks) if k_out is None else _heads(k_out, "k_out", n, kh, dim, dt)
        args = RopeArgs(dt, n, _ints(positions, "positions", n), qp, qop, qh, qt, qs, qot, qos, kp, kop, kh, kt, ks, kot,
                        kos, inverse)
        if lib.sapphire_rope_device(self.handle, C.byref(args)) != 0:
            raise SapphireError(f"sapphire_rope_device failed: {self.ctx.last_error}")

    def close(self) -> None:
        if self.handle:
            if self.ctx.handle:
                lib.sapphire_rope_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def kv_page_bytes(dtype, page_size: int, kv_heads: int, head_dim: int) -> int:
    """Bytes of one page of a cache of this shape."""
    n = lib.sapphire_kv_page_bytes(C.byref(KvCacheStruct(_dtype(dtype), page_size, kv_heads, head_dim, 0, None)))
    if not n:
        raise SapphireError(f"no cache of {page_size}-token pages, {kv_heads} KV heads of {head_dim} in this type")
    return int(n)


class KVCache:
    """A paged cache over `pages`, a uint8 tensor [num_pages, kv_page_bytes(...)]."""

    def __init__(self, ctx, dtype, page_size: int, kv_heads: int, head_dim: int, pages):
        self.ctx, self.dtype, self.pages = ctx, _dtype(dtype), pages
        self.page_size, self.kv_heads, self.head_dim = page_size, kv_heads, head_dim
        per = kv_page_bytes(self.dtype, page_size, kv_heads, head_dim)
        if len(pages.shape) != 2 or pages.shape[1] != per or pages.element_size() != 1 or not pages.is_contiguous():
            raise SapphireError(f"pages must be a contiguous byte tensor [num_pages, {per}]")
        self._struct = KvCacheStruct(self.dtype, page_size, kv_heads, head_dim, pages.shape[0], pages.data_ptr())
        self._ref = C.byref(self._struct)

    def _rows(self, fn, what, k, v, page_table, start, cu_tokens) -> None:
        n, heads, dim = k.shape[0], self.kv_heads, self.head_dim
        dt = _io_seen.get(k.dtype)
        if dt is None:
            dt = _io(k, "k")
        kp, kt, kh = _heads(k, "k", n, heads, dim, dt)
        vp, vt, vh = _heads(v, "v", n, heads, dim, dt)
        seqs = page_table.shape[0]
        table, stride = _table(page_table, seqs)
        args = KvArgs(dt, n, seqs, None if cu_tokens is None else _ints(cu_tokens, "cu_tokens", seqs + 1),
                      None if start is None else _ints(start, "start", seqs), table, stride, kp, vp, kt, kh, vt, vh)
        if fn(self.ctx.handle, self._ref, C.byref(args)) != 0:
            raise SapphireError(f"{what} failed: {self.ctx.last_error}")

    def write(self, k, v, page_table, start=None, cu_tokens=None) -> None:
        """Store k and v [tokens, kv_heads, head_dim]: token j of sequence s is
        row cu_tokens[s] + j (without cu_tokens one token each) and gets
        position start[s] + j."""
        self._rows(lib.sapphire_kv_write_device, "sapphire_kv_write_device", k, v, page_table, start, cu_tokens)

    def read(self, k, v, page_table, start=None, cu_tokens=None) -> None:
        """Fill k and v with the positions that write would store them at."""
        self._rows(lib.sapphire_kv_read_device, "sapphire_kv_read_device", k, v, page_table, start, cu_tokens)

    def workspace_bytes(self, sequences: int, heads: int) -> int:
        n = lib.sapphire_attention_workspace_bytes(self.ctx.handle, self._ref, sequences, heads)
        if not n:
            raise SapphireError(f"no attention of {heads} query heads over {self.kv_heads} KV heads")
        return int(n)

    def attend(self, q, page_table, lengths, out, scale: float = 0.0, window: int = 0, length_offset: int = 0,
               lse=None, workspace=None) -> None:
        """out = attention of q [sequences, heads, head_dim] over the first
        lengths[s] + length_offset positions of each sequence (the last
        `window` of them, if set).  page_table: [sequences, pages], or
        [sequences, kv_heads, pages] where each KV head has pages of its own.
        lse: float32 [sequences, heads] or None.
        workspace: a byte tensor of workspace_bytes(...) (required when the
        call is captured into a graph)."""
        n, heads, dim = q.shape[0], q.shape[1], self.head_dim
        dt = _io_seen.get(q.dtype)
        if dt is None:
            dt = _io(q, "q")
        qp, qs, qh = _heads(q, "q", n, None, dim, dt)
        op, os, oh = _heads(out, "out", n, heads, dim, dt)
        if lse is not None and (tuple(lse.shape) != (n, heads) or _io(lse, "lse") != DTYPE_F32 or not lse.is_contiguous()):
            raise SapphireError(f"lse must be contiguous float32 [{n}, {heads}]")
        if workspace is not None and not workspace.is_contiguous():
            raise SapphireError("workspace must be contiguous")
        per_head = len(page_table.shape) == 3
        table, stride = _head_table(page_table, n, self.kv_heads) if per_head else _table(page_table, n)
        args = AttentionArgs(dt, n, heads, qp, op, qs, qh, os, oh,
                             0 if lse is None else lse.data_ptr(), table, stride, _ints(lengths, "lengths", n),
                             length_offset, window, scale, addr(workspace),
                             0 if workspace is None else workspace.numel() * workspace.element_size())
        fn = lib.sapphire_attention_per_head_device if per_head else lib.sapphire_attention_device
        if fn(self.ctx.handle, self._ref, C.byref(args)) != 0:
            raise SapphireError(f"{fn.__name__} failed: {self.ctx.last_error}")

    @property
    def summary_bytes(self) -> int:
        """Bytes of one page's summary."""
        return int(lib.sapphire_kv_summary_bytes(self._ref))

    def _summary(self, summary) -> int:
        """The address of a byte tensor [num_pages, summary_bytes]."""
        if tuple(summary.shape) != (self._struct.num_pages, self.summary_bytes) or summary.element_size() != 1 or \
                not summary.is_contiguous():
            raise SapphireError(f"summary must be a contiguous byte tensor [{self._struct.num_pages}, {self.summary_bytes}]")
        return summary.data_ptr()

    def summarise(self, summary, page_table, tokens: int | None = None, start=None, cu_tokens=None) -> None:
        """Bring the bounds in `summary`, a uint8 tensor [num_pages, summary_bytes],
        of the pages that a write of `tokens` rows went to up to date (its
        page_table, start and cu_tokens; without cu_tokens one token each)."""
        seqs = page_table.shape[0]
        if tokens is None:
            if cu_tokens is not None:
                raise SapphireError("with cu_tokens, tokens must say how many rows there are")
            tokens = seqs
        table, stride = _table(page_table, seqs)
        args = KvArgs(DTYPE_F32, tokens, seqs, None if cu_tokens is None else _ints(cu_tokens, "cu_tokens", seqs + 1),
                      None if start is None else _ints(start, "start", seqs), table, stride, None, None, 0, 0, 0, 0)
        if lib.sapphire_kv_summarise_device(self.ctx.handle, self._ref, self._summary(summary), C.byref(args)) != 0:
            raise SapphireError(f"sapphire_kv_summarise_device failed: {self.ctx.last_error}")

    def select(self, q, summary, page_table, lengths, selected, selected_lengths, first: int = 1, last: int = 1,
               length_offset: int = 0) -> None:
        """Select up to selected.shape[2] pages of each sequence for each KV head:
        the first `first`, the last `last`, and those whose bounds promise q
        [sequences, heads, head_dim] the largest scores.  selected (int32
        [sequences, kv_heads, budget]) and selected_lengths (int32 [sequences]) are
        the page_table and lengths of attend."""
        n, dim = q.shape[0], self.head_dim
        dt = _io_seen.get(q.dtype)
        if dt is None:
            dt = _io(q, "q")
        qp, qs, qh = _heads(q, "q", n, None, dim, dt)
        table, stride = _table(page_table, n)
        out, budget = _head_table(selected, n, self.kv_heads, "selected")
        args = KvSelectArgs(dt, n, q.shape[1], qp, qs, qh, self._summary(summary), table, stride,
                            _ints(lengths, "lengths", n), length_offset, budget, first, last, out,
                            _ints(selected_lengths, "selected_lengths", n))
        if lib.sapphire_kv_select_device(self.ctx.handle, self._ref, C.byref(args)) != 0:
            raise SapphireError(f"sapphire_kv_select_device failed: {self.ctx.last_error}")

    def shared_workspace_bytes(self, dtype, sequences: int, heads: int) -> int:
        """Workspace of attend_shared for queries of this type (a DTYPE_* number or its name)."""
        n = lib.sapphire_attention_shared_workspace_bytes(self.ctx.handle, self._ref, _dtype(dtype), sequences, heads)
        if not n:
            raise SapphireError(f"no attention of {heads} query heads over {self.kv_heads} KV heads, {sequences} sequences")
        return int(n)

    def attend_shared(self, q, prefix_table, prefix_length, page_table, lengths, out, scale: float = 0.0,
                      length_offset: int = 0, lse=None, workspace=None) -> None:
        """out = attention of q [sequences, heads, head_dim] over the positions
        0 .. prefix_length[0] - 1 that all sequences begin with, on the pages of
        prefix_table (int32 [pages]), and the first lengths[s] + length_offset
        positions of each sequence's own page_table [sequences, pages] behind
        them.  lse: float32 [sequences, heads] or None.  workspace: a byte tensor
        of shared_workspace_bytes(...) (required when the call is captured into a
        graph)."""
        n, heads, dim = q.shape[0], q.shape[1], self.head_dim
        dt = _io_seen.get(q.dtype)
        if dt is None:
            dt = _io(q, "q")
        qp, qs, qh = _heads(q, "q", n, None, dim, dt)
        op, os, oh = _heads(out, "out", n, heads, dim, dt)
        if lse is not None and (tuple(lse.shape) != (n, heads) or _io(lse, "lse") != DTYPE_F32 or not lse.is_contiguous()):
            raise SapphireError(f"lse must be contiguous float32 [{n}, {heads}]")
        if workspace is not None and not workspace.is_contiguous():
            raise SapphireError("workspace must be contiguous")
        if len(prefix_table.shape) != 1:
            raise SapphireError(f"prefix_table has shape {tuple(prefix_table.shape)}, not [pages]")
        table, stride = _table(page_table, n)
        args = AttentionSharedArgs(dt, n, heads, qp, op, qs, qh, os, oh, 0 if lse is None else lse.data_ptr(),
                                   _ints(prefix_table, "prefix_table", None), prefix_table.shape[0],
                                   _ints(prefix_length, "prefix_length", 1), table, stride, _ints(lengths, "lengths", n),
                                   length_offset, scale, addr(workspace),
                                   0 if workspace is None else workspace.numel() * workspace.element_size())
        if lib.sapphire_attention_shared_device(self.ctx.handle, self._ref, C.byref(args)) != 0:
            raise SapphireError(f"sapphire_attention_shared_device failed: {self.ctx.last_error}")
