"""A paged key/value cache held in 4 bits: keys and values of many sequences appended and
read back, attention over them, and their pages reserved, forked, freed, compacted and
copied (lsx_cache_append_device and the entries beside it, which state the formulas, the
storage and what happens to entries that name nothing).

The reference keeps one sequence's keys and values in f32 (src/model.rs:492,
src/gpu.rs:454-501).  These work on torch CUDA tensors:

  pages    uint8 [pages, kv_heads, page_size / 16, 18 * head_dim], one layer (`pages_shape`)
  tables   int32 [sequences, pages per sequence], -1 is no page
  lengths  int32 [sequences]
  refs     int32 [pages], table entries that name the page
  pool     the pages of all layers, [layers, pages, ...] of any type (those of a cache
           in another type as well), each page contiguous and a multiple of 16 bytes

A call's sequences are rows 0, 1, .. of the tables, or those that `sequences` (int32)
lists; `starts` (int32, one more than the sequences, ascending) says which of the call's
rows belong to each, its last positions; without it each sequence has one row.  The
lengths count the call's own rows: reserve positions, append, then attend.  Positions
are taken back by lowering `lengths` in place: their pages stay with the sequence for
the next reserve, or until it is freed (lsx.h says where that ends: at a forked page).

Calls enqueue on torch's current stream on the Gpu's device, copy nothing to the host
and may be captured into a CUDA graph.  `PagedCache` holds the tensors and passes them."""
from __future__ import annotations

import ctypes as C
import struct
from typing import NamedTuple

import torch

from ._lib import BF16, F16, F32, CachePool, CacheRows, CacheView, check, lib
from .distribution import _stream, _unrecorded, _written
from .gpu import Gpu

_KINDS = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
_I32 = torch.int32
_Tensor = torch.Tensor
# The descriptions of lsx.h as bytes, which take less time to form than ctypes' structures.
_VIEW, _ROWS, _POOL = (struct.Struct(f"{C.sizeof(s) // 8}Q").pack for s in (CacheView, CacheRows, CachePool))
_append, _read, _attention = lib.lsx_cache_append_device, lib.lsx_cache_read_device, lib.lsx_cache_attention_device
_reserve, _fork, _free = lib.lsx_cache_reserve_device, lib.lsx_cache_fork_device, lib.lsx_cache_free_device
_compact, _copy = lib.lsx_cache_compact_device, lib.lsx_cache_copy_device
_workspace_bytes, _compact_bytes = lib.lsx_cache_attention_workspace_bytes, lib.lsx_cache_compact_workspace_bytes
_PAGES = "pages must be a contiguous uint8 tensor [pages, kv_heads, page_size / 16, 18 * head_dim] on the Gpu's device"
GROUP = 64  # elements that share a step and a zero
MAX_LISTED = 1024  # sequences that one call reserves for or forks


def pages_shape(pages: int, kv_heads: int, page_size: int, head_dim: int) -> tuple[int, int, int, int]:
    """Shape of one layer's pages (uint8)."""
    if head_dim not in (64, 128, 192, 256):
        raise ValueError("the cache holds heads of 64, 128, 192 or 256 elements")
    if page_size < 16 or page_size % 16:
        raise ValueError("a page holds a multiple of 16 positions")
    return pages, kv_heads, page_size // 16, 18 * head_dim


def _ints(device: int, t: torch.Tensor, n: int | None, name: str) -> int:
    """Address of a contiguous int32 vector of n elements (None: any) on the device."""
    if isinstance(t, _Tensor) and t.dtype is _I32 and t.dim() == 1 and t.get_device() == device and t.is_contiguous() \
            and (n is None or t.size(0) == n):
        return t.data_ptr()
    raise ValueError(f"{name} must be a contiguous int32 tensor of shape [{'any' if n is None else n}] on the Gpu's device")


def _table(device: int, t: torch.Tensor, name: str = "tables"):
    """(address, rows, width) of a contiguous int32 matrix on the device."""
    if isinstance(t, _Tensor) and t.dtype is _I32 and t.dim() == 2 and t.get_device() == device and t.is_contiguous():
        return t.data_ptr(), t.size(0), t.size(1)
    raise ValueError(f"{name} must be a contiguous int32 matrix on the Gpu's device")


def _view(device: int, pages: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor):
    """(lsx_cache_view, kv_heads, head_dim, rows of the tables)."""
    if not (isinstance(pages, _Tensor) and pages.dtype is torch.uint8 and pages.dim() == 4 and pages.is_contiguous()
            and pages.get_device() == device):
        raise ValueError(_PAGES)
    count, heads, cells, width = pages.shape
    dim = width // 18
    if width % (18 * GROUP) or not (heads and cells and dim):
        raise ValueError(_PAGES)
    at, rows, entries = _table(device, tables)
    return _VIEW(pages.data_ptr(), count, cells * 16, heads, dim, at, rows, entries, _ints(device, lengths, rows, "lengths")), \
        heads, dim, rows


def _rows(device: int, rows: int, table_rows: int, starts: torch.Tensor | None, sequences: torch.Tensor | None):
    """(lsx_cache_rows, number of sequences)."""
    if sequences is not None:
        listed = _ints(device, sequences, None, "sequences")
        count = sequences.size(0)
        if starts is None:
            if count != rows:
                raise ValueError("without starts each sequence has one row")
            return _ROWS(rows, count, listed, 0), count
        return _ROWS(rows, count, listed, _ints(device, starts, count + 1, "starts")), count
    if starts is None:
        count, at = rows, 0
    else:
        at = _ints(device, starts, None, "starts")
        count = starts.size(0) - 1
        if count < 0:
            raise ValueError("starts holds one entry more than the sequences")
    if count > table_rows:
        raise ValueError("more sequences than the tables have rows")
    return _ROWS(rows, count, 0, at), count


def _heads(device: int, t: torch.Tensor, name: str, heads: int | None, dim: int):
    """(rows, heads, row stride, head stride, kind) of a [rows, heads, head_dim] tensor on the device."""
    kind = _KINDS.get(t.dtype) if isinstance(t, _Tensor) and t.dim() == 3 else None
    if kind is None:
        raise ValueError(f"{name} must be a [rows, heads, head_dim] tensor of float32, float16 or bfloat16")
    if t.get_device() != device:
        raise ValueError(f"{name} must be on the Gpu's device")
    n, h, width = t.shape
    if width != dim or (heads is not None and h != heads):
        raise ValueError(f"{name} must have the cache's heads and head_dim")
    row, head, unit = t.stride()
    if unit != 1:
        raise ValueError(f"{name} must have unit stride within a head")
    return n, h, row, head, kind


def _apart(rows: int, heads: int, dim: int, row: int, head: int, name: str):
    """Refuses a tensor to write whose rows or heads overlap."""
    if heads > 1 and head < dim or rows > 1 and row < dim or \
            (heads > 1 and rows > 1 and (row < head * (heads - 1) + dim if row >= head else head < row * (rows - 1) + dim)):
        raise ValueError(f"rows and heads of {name} must not overlap")


def append(gpu: Gpu, k: torch.Tensor, v: torch.Tensor, pages: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor,
           starts: torch.Tensor | None = None, *, sequences: torch.Tensor | None = None) -> None:
    """Writes keys and values [rows, kv_heads, head_dim] (any strides between rows and
    heads) at their positions (lsx_cache_append_device)."""
    device = gpu.device
    view, heads, dim, table_rows = _view(device, pages, tables, lengths)
    n, _, k_row, k_head, kind = _heads(device, k, "keys", heads, dim)
    m, _, v_row, v_head, other = _heads(device, v, "values", heads, dim)
    if n != m or kind != other:
        raise ValueError("keys and values must have the same rows and dtype")
    if k.requires_grad or v.requires_grad:
        _unrecorded("keys" if k.requires_grad else "values")
    rows, count = _rows(device, n, table_rows, starts, sequences)
    if n and count:
        check(_append(gpu.handle, view, rows, k.data_ptr(), v.data_ptr(), kind, k_row, k_head, v_row, v_head, _stream(device)))
        _written((pages,))


def read(gpu: Gpu, pages: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor | None = None,
         *, sequences: torch.Tensor | None = None, rows: int | None = None, dtype: torch.dtype = torch.float32, out=None):
    """Keys and values [rows, kv_heads, head_dim] that the cache holds at the rows'
    positions (lsx_cache_read_device), into `out` (16-byte aligned) or new tensors of
    `dtype`, 0 in rows of no sequence.  With starts and no `out`, `rows` says how many rows there are."""
    device = gpu.device
    view, heads, dim, table_rows = _view(device, pages, tables, lengths)
    if out is None:
        if rows is None:
            if starts is not None:
                raise ValueError("rows must be given with starts")
            rows = table_rows if sequences is None else len(sequences)
        shape = (int(rows), heads, dim)
        out = (torch.zeros(shape, dtype=dtype, device=pages.device), torch.zeros(shape, dtype=dtype, device=pages.device))
    k, v = out
    n, _, _, _, kind = _heads(device, k, "out[0]", heads, dim)
    m, _, _, _, other = _heads(device, v, "out[1]", heads, dim)
    if n != m or kind != other or not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError("out holds two contiguous tensors of the same shape and dtype")
    listed, count = _rows(device, n, table_rows, starts, sequences)
    if n and count:
        check(_read(gpu.handle, view, listed, kind, k.data_ptr(), v.data_ptr(), _stream(device)))
        _written((k, v))
    return k, v


def attention(gpu: Gpu, q: torch.Tensor, pages: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor,
              starts: torch.Tensor | None = None, *, sequences: torch.Tensor | None = None, scale: float | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of queries [rows, q_heads, head_dim] over their sequences'
    positions (lsx_cache_attention_device); scale defaults to head_dim ** -0.5.  A new
    result is contiguous, and 0 in rows of no sequence."""
    device = gpu.device
    view, kv_heads, dim, table_rows = _view(device, pages, tables, lengths)
    n, heads, q_row, q_head, kind = _heads(device, q, "queries", None, dim)
    if heads == 0 or heads % kv_heads:
        raise ValueError("query heads are a multiple of key heads")
    if q.requires_grad:
        _unrecorded("queries")
    rows, count = _rows(device, n, table_rows, starts, sequences)
    if out is None:
        new = torch.empty if starts is None else torch.zeros
        out = new(q.shape, dtype=q.dtype, device=q.device)
        out_row, out_head = heads * dim, dim
    else:
        m, out_heads, out_row, out_head, other = _heads(device, out, "out", heads, dim)
        if m != n or other != kind:
            raise ValueError("out must have the queries' shape and dtype")
        _apart(n, heads, dim, out_row, out_head, "out")
    if n and count:
        size = _workspace_bytes(gpu.handle, dim)
        workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
        check(_attention(gpu.handle, view, rows, q.data_ptr(), kind, heads, q_row, q_head, dim ** -0.5 if scale is None else scale,
                         out.data_ptr(), out_row, out_head, workspace.data_ptr(), size, _stream(device)))
        _written((out,))
    return out


# ---- pages ---------------------------------------------------------------------
def _pool(device: int, pool: torch.Tensor):
    """(lsx_cache_pool, pages)."""
    if not (isinstance(pool, _Tensor) and pool.dim() >= 3 and pool.get_device() == device and pool.numel()):
        raise ValueError("the pool must be a [layers, pages, ...] tensor on the Gpu's device")
    layers, pages, width = pool.size(0), pool.size(1), pool.element_size()
    elements = pool.numel() // layers
    stride = elements
    if not pool.is_contiguous():
        stride = pool.stride(0)
        if not pool[0].is_contiguous() or (layers > 1 and stride < elements):
            raise ValueError("a layer's pages must be contiguous, and layers must not overlap")
    return _POOL(pool.data_ptr(), layers, stride * width, elements // pages * width, pages), pages


def _state(device: int, tables, lengths, refs):
    at, rows, width = _table(device, tables)
    return at, rows, width, _ints(device, lengths, rows, "lengths"), _ints(device, refs, None, "refs")


def _missing(device: int, missing: torch.Tensor | None, like: torch.Tensor):
    """(address, tensor) of the pages that were short."""
    if missing is None:
        missing = torch.zeros(1, dtype=_I32, device=like.device)
        return missing.data_ptr(), missing
    return _ints(device, missing, 1, "missing"), missing


def reserve(gpu: Gpu, tables: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor, sequences: torch.Tensor,
            counts: torch.Tensor, page_size: int, *, missing: torch.Tensor | None = None) -> torch.Tensor:
    """Gives the sequences (int32, at most 1024) further positions and the pages for them
    (lsx_cache_reserve_device).  Returns `missing` (int32 [1]): how many pages were short;
    unless it is 0 nothing changed."""
    device = gpu.device
    state = _state(device, tables, lengths, refs)
    at, missing = _missing(device, missing, refs)
    listed = _ints(device, sequences, None, "sequences")
    n = sequences.size(0)
    more = _ints(device, counts, n, "counts")
    if n > MAX_LISTED:
        raise ValueError(f"at most {MAX_LISTED} sequences a call")
    if n == 0:
        return missing.zero_()
    check(_reserve(gpu.handle, *state, refs.size(0), page_size, listed, more, n, at, _stream(device)))
    _written((tables, lengths, refs, missing))
    return missing


def fork(gpu: Gpu, pool: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor,
         parents: torch.Tensor, children: torch.Tensor, page_size: int, *, missing: torch.Tensor | None = None) -> torch.Tensor:
    """Empty sequences `children` take the positions of `parents` (both int32, at most
    1024): whole pages are shared, a partly filled one is copied (lsx_cache_fork_device).
    Returns `missing` as reserve does."""
    device = gpu.device
    view, pages = _pool(device, pool)
    state = _state(device, tables, lengths, refs)
    if refs.size(0) != pages:
        raise ValueError("refs must have an entry for each page of the pool")
    at, missing = _missing(device, missing, refs)
    of = _ints(device, parents, None, "parents")
    n = parents.size(0)
    to = _ints(device, children, n, "children")
    if n > MAX_LISTED:
        raise ValueError(f"at most {MAX_LISTED} sequences a call")
    if n == 0:
        return missing.zero_()
    pairs = torch.empty((n, 2), dtype=_I32, device=refs.device)
    check(_fork(gpu.handle, view, *state, page_size, of, to, n, pairs.data_ptr(), at, _stream(device)))
    _written((pool, tables, lengths, refs, missing))
    return missing


def free(gpu: Gpu, tables: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor, sequences: torch.Tensor,
         page_size: int) -> None:
    """Empties the sequences (int32, at most 65536); pages that no other sequence shares
    become free (lsx_cache_free_device)."""
    device = gpu.device
    state = _state(device, tables, lengths, refs)
    listed = _ints(device, sequences, None, "sequences")
    n = sequences.size(0)
    if n:
        check(_free(gpu.handle, *state, refs.size(0), page_size, listed, n, _stream(device)))
        _written((tables, lengths, refs))


class Compaction(NamedTuple):
    tables: torch.Tensor
    refs: torch.Tensor


def compact(gpu: Gpu, pool: torch.Tensor, tables: torch.Tensor, refs: torch.Tensor, *, out=None) -> Compaction:
    """Moves pages so that those in use are the lowest (lsx_cache_compact_device), in
    the pool; the tables and counts afterwards go to `out`, which may be the ones passed,
    or to new tensors."""
    device = gpu.device
    view, pages = _pool(device, pool)
    table, rows, width = _table(device, tables)
    counts = _ints(device, refs, pages, "refs")
    if out is None:
        out = (torch.empty_like(tables), torch.empty_like(refs))
    elif len(out) != 2:
        raise ValueError("out holds the tables and the counts")
    table_out, rows_out, width_out = _table(device, out[0], "out[0]")
    if rows_out != rows or width_out != width:
        raise ValueError("out[0] must have the tables' shape")
    counts_out = _ints(device, out[1], pages, "out[1]")
    size = _compact_bytes(pages)
    workspace = torch.empty(size, dtype=torch.uint8, device=refs.device)
    check(_compact(gpu.handle, view, table, rows, width, counts, table_out, counts_out, workspace.data_ptr(), size,
                   _stream(device)))
    _written((pool, out[0], out[1]))
    return Compaction(*out)


def copy_pages(gpu: Gpu, pool: torch.Tensor, pairs: torch.Tensor) -> None:
    """Copies page pairs[i, 0] to page pairs[i, 1] (int32) in every layer
    (lsx_cache_copy_device); no page may be two pairs' target, nor source and target."""
    device = gpu.device
    view, _ = _pool(device, pool)
    at, n, two = _table(device, pairs, "pairs")
    if two != 2:
        raise ValueError("pairs is an [n, 2] matrix")
    if n:
        check(_copy(gpu.handle, view, at, n, _stream(device)))
        _written((pool,))


class PagedCache:
    """The tensors of a cache in 4 bits and its calls: `pool` [layers, pages, kv_heads,
    page_size / 16, 18 * head_dim], `tables`, `lengths`, `refs`.  Sequences are rows of
    the tables, named by int32 tensors on the device."""

    def __init__(self, gpu: Gpu, *, layers: int, pages: int, kv_heads: int, head_dim: int, sequences: int, longest: int,
                 page_size: int = 64):
        shape = pages_shape(pages, kv_heads, page_size, head_dim)
        if min(layers, pages, kv_heads, sequences, longest) < 1:
            raise ValueError("check the sizes of the cache")
        device = torch.device("cuda", gpu.device)
        self.gpu, self.page_size = gpu, page_size
        self.pool = torch.zeros((layers, *shape), dtype=torch.uint8, device=device)
        self.tables = torch.full((sequences, -(-longest // page_size)), -1, dtype=_I32, device=device)
        self.lengths = torch.zeros(sequences, dtype=_I32, device=device)
        self.refs = torch.zeros(pages, dtype=_I32, device=device)

    def reserve(self, sequences: torch.Tensor, counts: torch.Tensor, missing: torch.Tensor | None = None) -> torch.Tensor:
        return reserve(self.gpu, self.tables, self.lengths, self.refs, sequences, counts, self.page_size, missing=missing)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor | None = None,
               sequences: torch.Tensor | None = None) -> None:
        append(self.gpu, k, v, self.pool[layer], self.tables, self.lengths, starts, sequences=sequences)

    def read(self, layer: int, starts: torch.Tensor | None = None, sequences: torch.Tensor | None = None, **options):
        return read(self.gpu, self.pool[layer], self.tables, self.lengths, starts, sequences=sequences, **options)

    def attention(self, layer: int, q: torch.Tensor, starts: torch.Tensor | None = None,
                  sequences: torch.Tensor | None = None, **options) -> torch.Tensor:
        return attention(self.gpu, q, self.pool[layer], self.tables, self.lengths, starts, sequences=sequences, **options)

    def fork(self, parents: torch.Tensor, children: torch.Tensor, missing: torch.Tensor | None = None) -> torch.Tensor:
        return fork(self.gpu, self.pool, self.tables, self.lengths, self.refs, parents, children, self.page_size,
                    missing=missing)

    def free(self, sequences: torch.Tensor) -> None:
        free(self.gpu, self.tables, self.lengths, self.refs, sequences, self.page_size)

    def compact(self) -> None:
        """In place."""
        compact(self.gpu, self.pool, self.tables, self.refs, out=(self.tables, self.refs))


__all__ = ["PagedCache", "Compaction", "append", "read", "attention", "reserve", "fork", "free", "compact", "copy_pages",
           "pages_shape", "GROUP", "MAX_LISTED"]
