"""Paged session cache: keys and values of many sequences of different lengths in
pages that forked sequences share.

`PagedCache` holds the pool, the page table and the counts as device tensors and
changes them through the C ABI (oasis_pages_*), in stream order and without reading
anything back: every call can be captured into a CUDA graph. What a call has to
refuse on the device (a full pool, a target in use) leaves bits in `status`;
`check()` reads them and raises.

Calls on one cache must be ordered: use one stream, or events between streams.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from .engine import _stream, workspace

DTYPES = {torch.bfloat16: _lib.OASIS_DTYPE_BF16, torch.float16: _lib.OASIS_DTYPE_F16}

BAD_SEQUENCE, IN_USE, NO_PAGES, TOO_LONG, BAD_PAGE = 1, 2, 4, 8, 16
STATUS = {
    BAD_SEQUENCE: "a sequence index outside the cache, or decreasing offsets",
    IN_USE: "a fork into a sequence that is not empty, or a sequence named twice",
    NO_PAGES: "the pool has no free page",
    TOO_LONG: "a sequence would pass its row of the page table",
    BAD_PAGE: "a page table entry outside the pool",
}


# The calls take a few microseconds: what is right is found with few questions, and only
# what is wrong is looked at closely.

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _on(stream, index: int) -> int:
    """The stream handle of a call: `stream`, or the device's current one."""
    if stream is None and _raw_stream is not None:
        return _raw_stream(index)
    return _stream(stream)


def _ints(t: torch.Tensor, name: str, index: int, numel: int) -> int:
    """Address of a contiguous int32 tensor of `numel` values on device `index`."""
    if t.dtype is torch.int32 and t.get_device() == index and t.numel() == numel and t.is_contiguous():
        return t.data_ptr()
    if t.get_device() != index:
        raise ValueError(f"{name} must be on CUDA device {index}, got {t.device}")
    if t.dtype is not torch.int32 or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32")
    raise ValueError(f"{name} must hold {numel} values, got {t.numel()}")


def _check_device(index: int):
    """The library launches on the current device."""
    if index < 0:
        raise ValueError("tensors must be on a CUDA device")
    if index != torch.cuda.current_device():
        raise ValueError(f"tensors are on cuda:{index}, but cuda:{torch.cuda.current_device()} is the current device")


def _rows(t: torch.Tensor, name: str, dtype, index: int, rows: int | None, heads: int | None, dim: int):
    """(rows, heads, address, row stride, head stride) of a [rows, heads, dim] tensor with
    contiguous, 16-byte aligned head vectors. Strides of dimensions of size one, which
    torch leaves open, are those of packed rows."""
    if t.dtype is dtype and t.get_device() == index and t.dim() == 3:
        n, h, d = t.shape
        if d == dim and (heads is None or h == heads) and (rows is None or n == rows):
            row, head, one = t.stride()
            if h == 1:
                head = dim
            if n <= 1:
                row = h * dim
            at = t.data_ptr()
            if one == 1 and not (at & 15 or (row | head) & 7):
                return n, h, at, row, head
    if t.get_device() != index:
        raise ValueError(f"{name} must be on CUDA device {index}, got {t.device}")
    if t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    want = f"[{'rows' if rows is None else rows}, {'heads' if heads is None else heads}, {dim}]"
    if t.dim() != 3 or t.shape[2] != dim or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be {want}, got {tuple(t.shape)}")
    if rows is not None and t.shape[0] != rows:
        raise ValueError(f"{name} has {t.shape[0]} rows, not {rows}")
    if t.stride(2) != 1:
        raise ValueError(f"{name}: the values of a head must be contiguous")
    raise ValueError(f"{name}: head vectors must be 16-byte aligned (strides multiples of 8 elements)")


def _new(t: torch.Tensor, shape, stream) -> torch.Tensor:
    """An output or a workspace of a call on `stream`: memory that this stream's earlier work
    has left (the current stream may still use what it gave back), kept from it until
    what the current stream does with the result is done."""
    if stream is None:
        return t.new_empty(shape)
    with torch.cuda.stream(stream):
        out = t.new_empty(shape)
    out.record_stream(torch.cuda.current_stream())
    return out


_MOST = (1 << 31) - 1
_void, _int, _long, _packed = C.c_void_p, C.c_int, C.c_longlong, C.c_char_p
_reserve = _lib.packed_call("oasis_pages_reserve", _packed, _void, _void, _int, _void, _void)
_write = _lib.packed_call("oasis_pages_write", _packed, _int, _void, _void, _long, _long, _long, _long, _void, _void,
                          _void, _int, _int, _void)
_fork = _lib.packed_call("oasis_pages_fork", _packed, _void, _void, _int, _int, _void)
_free = _lib.packed_call("oasis_pages_free", _packed, _void, _int, _void)
_compact = _lib.packed_call("oasis_pages_compact", _packed, _void)
_prompt = _lib.packed_call("oasis_attention_prompt", _packed, _void)
_shared = _lib.packed_call("oasis_attention_shared", _packed, _void)
_pack_prompt = _lib.packer(_lib.OasisPromptArgs).pack
_pack_shared = _lib.packer(_lib.OasisSharedArgs).pack


class PagedCache:
    """Pool [pages, layers, 2, kv_heads, page_size, head_dim], page table
    [sequences, max_pages], lengths [sequences] and page counts [pages].

    `from_tensors` builds the handle around existing tensors (a cache restored from
    a checkpoint, or shared with other code; `status` [1] too where its bits are to be
    kept)."""

    def __init__(self, pages: int, page_size: int, layers: int, kv_heads: int, head_dim: int, sequences: int,
                 max_pages: int, dtype=torch.bfloat16, device="cuda"):
        ints = dict(dtype=torch.int32, device=device)
        self._bind(torch.zeros(pages, layers, 2, kv_heads, page_size, head_dim, dtype=dtype, device=device),
                   torch.full((sequences, max_pages), -1, **ints), torch.zeros(sequences, **ints),
                   torch.zeros(pages, **ints))

    @classmethod
    def from_tensors(cls, pool: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
                     refs: torch.Tensor, status: torch.Tensor | None = None) -> "PagedCache":
        self = cls.__new__(cls)
        self._bind(pool, table, lengths, refs, status)
        return self

    def _bind(self, pool, table, lengths, refs, status=None):
        if pool.dim() != 6 or pool.shape[2] != 2 or not pool.is_contiguous():
            raise ValueError("pool must be contiguous [pages, layers, 2, kv_heads, page_size, head_dim]")
        if pool.dtype not in DTYPES:
            raise ValueError(f"pool must be bfloat16 or float16, got {pool.dtype}")
        if not pool.is_cuda:
            raise ValueError("pool must be a CUDA tensor")
        if table.dim() != 2:
            raise ValueError("table must be [sequences, max_pages]")
        self.device, index = pool.device, pool.get_device()
        _ints(table, "table", index, table.numel())
        _ints(lengths, "lengths", index, table.shape[0])
        _ints(refs, "refs", index, pool.shape[0])
        if status is None:
            status = torch.zeros(1, dtype=torch.int32, device=pool.device)
        _ints(status, "status", index, 1)
        self.pool, self.table, self.lengths, self.refs, self.status = pool, table, lengths, refs, status
        self.pages, self.layers, _, self.kv_heads, self.page_size, self.head_dim = pool.shape
        self.sequences, self.max_pages = table.shape
        self.dtype, self._index = pool.dtype, index
        self.ws = workspace(_lib.load().oasis_pages_workspace_size(self.pages, self.sequences), self.device)
        c = _lib.OasisPageCache(pool.data_ptr(), self.pages, self.layers, self.kv_heads, self.page_size, self.head_dim,
                                DTYPES[self.dtype], table.data_ptr(), self.sequences, self.max_pages, lengths.data_ptr(),
                                refs.data_ptr(), self.status.data_ptr(), self.ws.data_ptr(), self.ws.numel())
        self._c = bytes(c)  # the C struct, kept alive and passed as it is
        self._at = C.cast(self._c, C.c_void_p).value

    def __reduce__(self):
        """Copied and stored as its tensors: the struct holds their addresses. What has been
        refused since the last `check` is among them."""
        return PagedCache.from_tensors, (self.pool, self.table, self.lengths, self.refs, self.status)

    def reserve(self, seqs: torch.Tensor, cu: torch.Tensor, stream=None) -> torch.Tensor:
        """Room for cu[i + 1] - cu[i] more tokens behind sequence seqs[i]; returns
        each one's length before (-1: refused, see `status`), for `write`."""
        index, n = self._index, seqs.numel()
        _check_device(index)
        start = _new(seqs, n, stream)
        _reserve(self._c, _ints(seqs, "seqs", index, n), _ints(cu, "cu", index, n + 1), n, start.data_ptr(),
                 _on(stream, index))
        return start

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, seqs: torch.Tensor, cu: torch.Tensor,
              start: torch.Tensor, stream=None):
        """Keys and values [rows, kv_heads, head_dim] of the reserved tokens: packed rows
        [cu[i], cu[i + 1]) belong to sequence seqs[i], from position start[i] on."""
        index, n = self._index, seqs.numel()
        _check_device(index)
        rows, _, k_at, k_row, k_head = _rows(k, "k", self.dtype, index, None, self.kv_heads, self.head_dim)
        _, _, v_at, v_row, v_head = _rows(v, "v", self.dtype, index, rows, self.kv_heads, self.head_dim)
        _write(self._c, layer, k_at, v_at, k_row, k_head, v_row, v_head, _ints(seqs, "seqs", index, n),
               _ints(cu, "cu", index, n + 1), _ints(start, "start", index, n), n, rows, _on(stream, index))

    def fork(self, src: torch.Tensor, dst: torch.Tensor, deep: bool = False, stream=None):
        """The empty sequences dst[i] continue src[i]: whole pages are shared and a
        partial last page is copied; deep=True copies every page."""
        index, n = self._index, src.numel()
        _check_device(index)
        _fork(self._c, _ints(src, "src", index, n), _ints(dst, "dst", index, n), n, int(deep), _on(stream, index))

    def free(self, seqs: torch.Tensor, stream=None):
        """Empties sequences; their pages are free once nobody else holds them."""
        index, n = self._index, seqs.numel()
        _check_device(index)
        _free(self._c, _ints(seqs, "seqs", index, n), n, _on(stream, index))

    def compact(self, stream=None):
        """Moves the pages in use to the front of the pool."""
        _check_device(self._index)
        _compact(self._c, _on(stream, self._index))

    def check(self):
        """Raises if a call was refused on the device since the last check (synchronizes;
        a call on the current stream, ordered like the others)."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise _lib.OasisError("PagedCache", -1, "; ".join(t for b, t in STATUS.items() if bits & b))


def attention_prompt(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor, longest: int,
                     out: torch.Tensor | None = None, scale: float | None = None, stream=None) -> torch.Tensor:
    """Causal attention within packed sequences: rows [cu[i], cu[i + 1]) of q [rows, heads,
    dim] and k, v [rows, kv_heads, dim] (views of packed QKV rows are fine) are one
    sequence. dim is 64 or 128, heads a multiple of kv_heads. Rows of no sequence are
    left as they are in `out`, which must not overlap q, k or v. `longest` (the longest
    sequence, or a bound) chooses the kernel and nothing else."""
    index = q.get_device()
    _check_device(index)
    if q.dtype not in DTYPES:
        raise ValueError(f"q must be bfloat16 or float16, got {q.dtype}")
    dtype, dim = q.dtype, q.shape[-1]
    rows, heads, q_at, q_row, q_head = _rows(q, "q", dtype, index, None, None, dim)
    _, kv_heads, k_at, k_row, k_head = _rows(k, "k", dtype, index, rows, None, dim)
    _, _, v_at, v_row, v_head = _rows(v, "v", dtype, index, rows, kv_heads, dim)
    if out is None:
        out = _new(q, (rows, heads, dim), stream)
    _, _, out_at, out_row, out_head = _rows(out, "out", dtype, index, rows, heads, dim)
    n = max(cu.numel() - 1, 0)
    _prompt(_pack_prompt(q_at, k_at, v_at, out_at, q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head, rows,
                         _ints(cu, "cu", index, cu.numel()), n, min(longest, _MOST), heads, kv_heads, dim, DTYPES[dtype],
                         dim ** -0.5 if scale is None else scale), _on(stream, index))
    return out


class SharedPlan:
    """Which rows of a batch share a prefix: group g is the next group_rows[g] rows, and
    the first prefix_pages[g] pages of their sequences are the same (PagedCache.fork
    leaves them so; it is not checked). `longest`: the most tokens of a sequence in the
    calls to come (a hint that chooses splits). Made once for a batch and kept while it lasts:
    a row that is freed and filled again, or replaced by a full copy, no longer shares."""

    def __init__(self, group_rows: list[int], prefix_pages: list[int], longest: int, device="cuda"):
        if len(group_rows) != len(prefix_pages) or any(r < 0 for r in group_rows) or any(p < 0 for p in prefix_pages):
            raise ValueError("group_rows and prefix_pages must hold one count, not negative, for each group")
        starts = [0]
        for r in group_rows:
            starts.append(starts[-1] + r)
        self.groups, self.rows = len(group_rows), starts[-1]
        self.group_start = torch.tensor(starts, dtype=torch.int32, device=device)
        self.prefix_pages = torch.tensor(prefix_pages or [0], dtype=torch.int32, device=device)
        self.bytes = torch.empty(0, dtype=torch.uint8, device=device)  # for workspaces' type and device
        self.longest = longest
        self.most_rows = max(group_rows, default=0)
        self.most_pages = max(prefix_pages, default=0)
        self.least_pages = min(prefix_pages, default=0)


def attention_shared(q: torch.Tensor, cache: PagedCache, layer: int, seqs: torch.Tensor, plan: SharedPlan,
                     out: torch.Tensor | None = None, scale: float | None = None, stream=None) -> torch.Tensor:
    """One query per row: q [rows, heads, head_dim] over the tokens of sequences
    seqs [rows] of the cache, in one layer, after their newest token was written.
    Prefixes that `plan` names are read once for their group. `out` must not overlap q
    or the cache."""
    index, dim = cache._index, cache.head_dim
    _check_device(index)
    if plan.group_start.get_device() != index:
        raise ValueError(f"the cache is on cuda:{index}, the plan on {plan.group_start.device}")
    rows, heads, q_at, q_row, q_head = _rows(q, "q", cache.dtype, index, None, None, dim)
    seqs_at = _ints(seqs, "seqs", index, rows)
    if plan.rows > rows:
        raise ValueError(f"the plan is for {plan.rows} rows, q has {rows}")
    if out is None:
        out = _new(q, (rows, heads, dim), stream)
    _, _, out_at, out_row, out_head = _rows(out, "out", cache.dtype, index, rows, heads, dim)
    fields = (q_at, out_at, q_row, q_head, out_row, out_head, cache._at, layer, seqs_at, rows,
              heads, plan.group_start.data_ptr(), plan.prefix_pages.data_ptr(), plan.groups, plan.most_rows,
              plan.most_pages, min(max(0, plan.longest - plan.least_pages * cache.page_size), _MOST),
              dim ** -0.5 if scale is None else scale)
    size = _shared_workspace(_pack_shared(*fields, 0, 0))
    ws = _new(plan.bytes, size, stream) if size else None
    _shared(_pack_shared(*fields, ws.data_ptr() if size else 0, size), _on(stream, index))
    return out


def _shared_workspace(args: bytes) -> int:
    global _size_of
    if _size_of is None:
        _size_of = _lib.load()["oasis_attention_shared_workspace_size"]
        _size_of.restype, _size_of.argtypes = C.c_size_t, (C.c_char_p,)
    return _size_of(args)


_size_of = None
