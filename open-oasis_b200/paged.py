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


def _check_ints(t: torch.Tensor, name: str, device, numel: int | None = None):
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    if t.dtype != torch.int32 or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name} must hold {numel} values, got {t.numel()}")


def _check_device(device):
    """The library launches on the current device."""
    if device.type != "cuda":
        raise ValueError("tensors must be on a CUDA device")
    if device.index != torch.cuda.current_device():
        raise ValueError(f"tensors are on {device}, but cuda:{torch.cuda.current_device()} is the current device")


def _check_rows(t: torch.Tensor, name: str, dtype, device, heads: int | None, dim: int):
    """[rows, heads, dim] with contiguous, 16-byte aligned head vectors."""
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != 3 or t.shape[2] != dim or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be [rows, {'heads' if heads is None else heads}, {dim}], got {tuple(t.shape)}")
    if t.stride(2) != 1:
        raise ValueError(f"{name}: the values of a head must be contiguous")
    if t.data_ptr() % 16 or any(t.stride(d) % 8 for d in (0, 1) if t.shape[d] > 1):
        raise ValueError(f"{name}: head vectors must be 16-byte aligned (strides multiples of 8 elements)")


def _strides(t: torch.Tensor) -> tuple[int, int]:
    """Row and head strides; those of dimensions of size one are replaced by packed ones."""
    head = t.stride(1) if t.shape[1] > 1 else t.shape[2]
    return (t.stride(0) if t.shape[0] > 1 else t.shape[1] * t.shape[2]), head


class PagedCache:
    """Pool [pages, layers, 2, kv_heads, page_size, head_dim], page table
    [sequences, max_pages], lengths [sequences] and page counts [pages].

    `from_tensors` builds the handle around existing tensors (a cache restored from
    a checkpoint, or shared with other code)."""

    def __init__(self, pages: int, page_size: int, layers: int, kv_heads: int, head_dim: int, sequences: int,
                 max_pages: int, dtype=torch.bfloat16, device="cuda"):
        ints = dict(dtype=torch.int32, device=device)
        self._bind(torch.zeros(pages, layers, 2, kv_heads, page_size, head_dim, dtype=dtype, device=device),
                   torch.full((sequences, max_pages), -1, **ints), torch.zeros(sequences, **ints),
                   torch.zeros(pages, **ints))

    @classmethod
    def from_tensors(cls, pool: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
                     refs: torch.Tensor) -> "PagedCache":
        self = cls.__new__(cls)
        self._bind(pool, table, lengths, refs)
        return self

    def _bind(self, pool, table, lengths, refs):
        if pool.dim() != 6 or pool.shape[2] != 2 or not pool.is_contiguous():
            raise ValueError("pool must be contiguous [pages, layers, 2, kv_heads, page_size, head_dim]")
        if pool.dtype not in DTYPES:
            raise ValueError(f"pool must be bfloat16 or float16, got {pool.dtype}")
        if not pool.is_cuda:
            raise ValueError("pool must be a CUDA tensor")
        if table.dim() != 2:
            raise ValueError("table must be [sequences, max_pages]")
        self.device = pool.device
        _check_ints(table, "table", self.device)
        _check_ints(lengths, "lengths", self.device, table.shape[0])
        _check_ints(refs, "refs", self.device, pool.shape[0])
        self.pool, self.table, self.lengths, self.refs = pool, table, lengths, refs
        self.pages, self.layers, _, self.kv_heads, self.page_size, self.head_dim = pool.shape
        self.sequences, self.max_pages = table.shape
        self.dtype = pool.dtype
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.ws = workspace(_lib.load().oasis_pages_workspace_size(self.pages, self.sequences), self.device)
        self._c = _lib.OasisPageCache(pool.data_ptr(), self.pages, self.layers, self.kv_heads, self.page_size,
                                      self.head_dim, DTYPES[self.dtype], table.data_ptr(), self.sequences,
                                      self.max_pages, lengths.data_ptr(), refs.data_ptr(), self.status.data_ptr(),
                                      self.ws.data_ptr(), self.ws.numel())
        self._ref = C.byref(self._c)

    def reserve(self, seqs: torch.Tensor, cu: torch.Tensor, stream=None) -> torch.Tensor:
        """Room for cu[i + 1] - cu[i] more tokens behind sequence seqs[i]; returns
        each one's length before (-1: refused, see `status`), for `write`."""
        _check_device(self.device)
        _check_ints(seqs, "seqs", self.device)
        _check_ints(cu, "cu", self.device, seqs.numel() + 1)
        start = torch.empty(seqs.shape, dtype=torch.int32, device=self.device)
        if stream is not None:
            start.record_stream(stream)
        _lib.call("oasis_pages_reserve", self._ref, seqs.data_ptr(), cu.data_ptr(), seqs.numel(), start.data_ptr(),
                  _stream(stream))
        return start

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, seqs: torch.Tensor, cu: torch.Tensor,
              start: torch.Tensor, stream=None):
        """Keys and values [rows, kv_heads, head_dim] of the reserved tokens: packed rows
        [cu[i], cu[i + 1]) belong to sequence seqs[i], from position start[i] on."""
        _check_device(self.device)
        _check_rows(k, "k", self.dtype, self.device, self.kv_heads, self.head_dim)
        _check_rows(v, "v", self.dtype, self.device, self.kv_heads, self.head_dim)
        if k.shape[0] != v.shape[0]:
            raise ValueError(f"k has {k.shape[0]} rows and v {v.shape[0]}")
        n = seqs.numel()
        _check_ints(seqs, "seqs", self.device)
        _check_ints(cu, "cu", self.device, n + 1)
        _check_ints(start, "start", self.device, n)
        _lib.call("oasis_pages_write", self._ref, layer, k.data_ptr(), v.data_ptr(), *_strides(k), *_strides(v),
                  seqs.data_ptr(), cu.data_ptr(), start.data_ptr(), n, k.shape[0], _stream(stream))

    def fork(self, src: torch.Tensor, dst: torch.Tensor, deep: bool = False, stream=None):
        """The empty sequences dst[i] continue src[i]: whole pages are shared and a
        partial last page is copied; deep=True copies every page."""
        _check_device(self.device)
        _check_ints(src, "src", self.device)
        _check_ints(dst, "dst", self.device, src.numel())
        _lib.call("oasis_pages_fork", self._ref, src.data_ptr(), dst.data_ptr(), src.numel(), int(deep),
                  _stream(stream))

    def free(self, seqs: torch.Tensor, stream=None):
        """Empties sequences; their pages are free once nobody else holds them."""
        _check_device(self.device)
        _check_ints(seqs, "seqs", self.device)
        _lib.call("oasis_pages_free", self._ref, seqs.data_ptr(), seqs.numel(), _stream(stream))

    def compact(self, stream=None):
        """Moves the pages in use to the front of the pool."""
        _check_device(self.device)
        _lib.call("oasis_pages_compact", self._ref, _stream(stream))

    def check(self):
        """Raises if a call was refused on the device since the last check (synchronizes)."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise _lib.OasisError("PagedCache", -1, "; ".join(t for b, t in STATUS.items() if bits & b))


def attention_prompt(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor, longest: int,
                     out: torch.Tensor | None = None, scale: float | None = None, stream=None) -> torch.Tensor:
    """Causal attention within packed sequences: rows [cu[i], cu[i + 1]) of q [rows, heads,
    dim] and k, v [rows, kv_heads, dim] (views of packed QKV rows are fine) are one
    sequence. dim is 64 or 128, heads a multiple of kv_heads. Rows of no sequence are
    left as they are in `out`. `longest` (the longest sequence, or a bound) chooses the
    kernel and nothing else."""
    device = q.device
    _check_device(device)
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("q, k and v must be [rows, heads, dim]")
    rows, heads, dim = q.shape
    if q.dtype not in DTYPES:
        raise ValueError(f"q must be bfloat16 or float16, got {q.dtype}")
    _check_rows(q, "q", q.dtype, device, None, dim)
    _check_rows(k, "k", q.dtype, device, None, dim)
    _check_rows(v, "v", q.dtype, device, k.shape[1], dim)
    if k.shape[0] != rows or v.shape[0] != rows:
        raise ValueError(f"q, k and v have {rows}, {k.shape[0]} and {v.shape[0]} rows")
    _check_ints(cu, "cu", device)
    if out is None:
        out = torch.empty(rows, heads, dim, dtype=q.dtype, device=device)
        if stream is not None:
            out.record_stream(stream)
    else:
        _check_rows(out, "out", q.dtype, device, heads, dim)
        if out.shape[0] != rows:
            raise ValueError(f"out has {out.shape[0]} rows, q {rows}")
    a = _lib.OasisPromptArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), *_strides(q), *_strides(k),
                             *_strides(v), *_strides(out), rows, cu.data_ptr(), max(cu.numel() - 1, 0), longest, heads,
                             k.shape[1], dim, DTYPES[q.dtype], dim ** -0.5 if scale is None else scale)
    _lib.call("oasis_attention_prompt", C.byref(a), _stream(stream))
    return out


class SharedPlan:
    """Which rows of a batch share a prefix: group g is the next group_rows[g] rows, and
    the first prefix_pages[g] pages of their sequences are the same (PagedCache.fork
    leaves them so). `longest`: the most tokens of a sequence in the calls to come (a
    hint that chooses splits). Made once for a batch and kept while it lasts."""

    def __init__(self, group_rows: list[int], prefix_pages: list[int], longest: int, device="cuda"):
        if len(group_rows) != len(prefix_pages) or any(r < 0 for r in group_rows) or any(p < 0 for p in prefix_pages):
            raise ValueError("group_rows and prefix_pages must hold one count, not negative, for each group")
        starts = [0]
        for r in group_rows:
            starts.append(starts[-1] + r)
        self.groups, self.rows = len(group_rows), starts[-1]
        self.group_start = torch.tensor(starts, dtype=torch.int32, device=device)
        self.prefix_pages = torch.tensor(prefix_pages or [0], dtype=torch.int32, device=device)
        self.longest = longest
        self.most_rows = max(group_rows, default=0)
        self.most_pages = max(prefix_pages, default=0)
        self.least_pages = min(prefix_pages, default=0)


def attention_shared(q: torch.Tensor, cache: PagedCache, layer: int, seqs: torch.Tensor, plan: SharedPlan,
                     out: torch.Tensor | None = None, scale: float | None = None, stream=None) -> torch.Tensor:
    """One query per row: q [rows, heads, head_dim] over the tokens of sequences
    seqs [rows] of the cache, in one layer, after their newest token was written.
    Prefixes that `plan` names are read once for their group."""
    device = q.device
    _check_device(device)
    if cache.device != device or plan.group_start.device != device:
        raise ValueError(f"q is on {device}, the cache on {cache.device}, the plan on {plan.group_start.device}")
    _check_rows(q, "q", cache.dtype, device, None, cache.head_dim)
    rows, heads, dim = q.shape
    _check_ints(seqs, "seqs", device, rows)
    if plan.rows > rows:
        raise ValueError(f"the plan is for {plan.rows} rows, q has {rows}")
    if out is None:
        out = torch.empty(rows, heads, dim, dtype=q.dtype, device=device)
        if stream is not None:
            out.record_stream(stream)
    else:
        _check_rows(out, "out", q.dtype, device, heads, dim)
        if out.shape[0] != rows:
            raise ValueError(f"out has {out.shape[0]} rows, q {rows}")
    own = max(0, plan.longest - plan.least_pages * cache.page_size)
    a = _lib.OasisSharedArgs(q.data_ptr(), out.data_ptr(), *_strides(q), *_strides(out), C.pointer(cache._c), layer,
                             seqs.data_ptr(), rows, heads, plan.group_start.data_ptr(), plan.prefix_pages.data_ptr(),
                             plan.groups, plan.most_rows, plan.most_pages, own, dim ** -0.5 if scale is None else scale)
    ref = C.byref(a)
    size = _lib.load().oasis_attention_shared_workspace_size(ref)
    if size:
        ws = workspace(size, device)
        if stream is not None:
            ws.record_stream(stream)
        a.workspace, a.workspace_bytes = ws.data_ptr(), size
    _lib.call("oasis_attention_shared", ref, _stream(stream))
    return out
