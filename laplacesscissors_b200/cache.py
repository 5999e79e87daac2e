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
lengths count the call's own rows: reserve positions, append, then attend.

Calls enqueue on torch's current stream on the Gpu's device, copy nothing to the host
and may be captured into a CUDA graph.  `PagedCache` holds the tensors and passes them."""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from ._lib import BF16, F16, F32, CachePool, CacheRows, CacheView, check, lib
from .distribution import _stream, _unrecorded, _written
from .gpu import Gpu

_KINDS = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
_I32 = torch.int32
_Tensor = torch.Tensor
GROUP = 64  # elements that share a step and a zero
MAX_LISTED = 1024  # sequences that one call reserves for or forks


def pages_shape(pages: int, kv_heads: int, page_size: int, head_dim: int) -> tuple[int, int, int, int]:
    """Shape of one layer's pages (uint8)."""
    if head_dim not in (64, 128, 192, 256):
        raise ValueError("the cache holds heads of 64, 128, 192 or 256 elements")
    if page_size < 16 or page_size % 16:
        raise ValueError("a page holds a multiple of 16 positions")
    return pages, kv_heads, page_size // 16, 18 * head_dim


def _ints(gpu: Gpu, t: torch.Tensor, shape: tuple, name: str) -> int:
    """Address of a contiguous int32 tensor of this shape (None: any extent) on the device."""
    if isinstance(t, _Tensor) and t.dtype is _I32 and t.get_device() == gpu.device and t.is_contiguous() \
            and len(t.shape) == len(shape) and all(n is None or n == m for n, m in zip(shape, t.shape)):
        return t.data_ptr()
    shape = ", ".join("any" if n is None else str(n) for n in shape)
    raise ValueError(f"{name} must be a contiguous int32 tensor of shape [{shape}] on the Gpu's device")


def _view(gpu: Gpu, pages: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor) -> CacheView:
    if not (isinstance(pages, _Tensor) and pages.dtype is torch.uint8 and pages.dim() == 4 and pages.is_contiguous()
            and pages.get_device() == gpu.device and pages.shape[3] % (18 * GROUP) == 0):
        raise ValueError("pages must be a contiguous uint8 tensor [pages, kv_heads, page_size / 16, 18 * head_dim] "
                         "on the Gpu's device")
    at = _ints(gpu, tables, (None, None), "tables")
    count, heads, cells, width = pages.shape
    return CacheView(pages.data_ptr(), count, cells * 16, heads, width // 18, at, tables.shape[0], tables.shape[1],
                     _ints(gpu, lengths, (tables.shape[0],), "lengths"))


def _rows(gpu: Gpu, rows: int, view: CacheView, starts: torch.Tensor | None, sequences: torch.Tensor | None) -> CacheRows:
    listed = None
    if sequences is not None:
        listed = _ints(gpu, sequences, (None,), "sequences")
        count = sequences.shape[0]
    elif starts is not None:
        count = starts.shape[0] - 1 if isinstance(starts, _Tensor) and starts.dim() == 1 else 0
    else:
        count = rows
    if sequences is None and count > view.table_rows:
        raise ValueError("more sequences than the tables have rows")
    if starts is None:
        if count != rows:
            raise ValueError("without starts each sequence has one row")
        return CacheRows(rows, count, listed, None)
    return CacheRows(rows, count, listed, _ints(gpu, starts, (count + 1,), "starts"))


def _heads(gpu: Gpu, t: torch.Tensor, name: str, heads: int | None, dim: int):
    """(rows, heads, row stride, head stride, kind) of a [rows, heads, head_dim] tensor on the device."""
    kind = _KINDS.get(t.dtype) if isinstance(t, _Tensor) and t.dim() == 3 else None
    if kind is None:
        raise ValueError(f"{name} must be a [rows, heads, head_dim] tensor of float32, float16 or bfloat16")
    if t.get_device() != gpu.device:
        raise ValueError(f"{name} must be on the Gpu's device")
    if t.shape[2] != dim or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must have the cache's heads and head_dim")
    row, head, unit = t.stride()
    if unit != 1:
        raise ValueError(f"{name} must have unit stride within a head")
    return t.shape[0], t.shape[1], row, head, kind


def _apart(t: torch.Tensor, name: str):
    """Refuses a tensor to write whose rows or heads overlap."""
    rows, heads, dim = t.shape
    row, head, _ = t.stride()
    small, large, n = (head, row, heads) if head <= row or rows <= 1 else (row, head, rows)
    if (n > 1 and small < dim) or (max(rows, heads) > 1 and rows > 1 and heads > 1 and large < small * (n - 1) + dim) \
            or (heads <= 1 and rows > 1 and row < dim):
        raise ValueError(f"rows and heads of {name} must not overlap")


def append(gpu: Gpu, k: torch.Tensor, v: torch.Tensor, pages: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor,
           starts: torch.Tensor | None = None, *, sequences: torch.Tensor | None = None) -> None:
    """Writes keys and values [rows, kv_heads, head_dim] (any strides between rows and
    heads) at their positions (lsx_cache_append_device)."""
    view = _view(gpu, pages, tables, lengths)
    n, _, k_row, k_head, kind = _heads(gpu, k, "keys", view.kv_heads, view.head_dim)
    m, _, v_row, v_head, other = _heads(gpu, v, "values", view.kv_heads, view.head_dim)
    if n != m or kind != other:
        raise ValueError("keys and values must have the same rows and dtype")
    if k.requires_grad or v.requires_grad:
        _unrecorded("keys" if k.requires_grad else "values")
    rows = _rows(gpu, n, view, starts, sequences)
    if n and rows.sequences:
        check(lib.lsx_cache_append_device(gpu.handle, C.byref(view), C.byref(rows), k.data_ptr(), v.data_ptr(), kind,
                                          k_row, k_head, v_row, v_head, _stream(gpu.device)))
        _written((pages,))


def read(gpu: Gpu, pages: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor | None = None,
         *, sequences: torch.Tensor | None = None, rows: int | None = None, dtype: torch.dtype = torch.float32, out=None):
    """Keys and values [rows, kv_heads, head_dim] that the cache holds at the rows'
    positions (lsx_cache_read_device), into `out` or new tensors of `dtype`.  With starts
    and no `out`, `rows` says how many rows there are."""
    view = _view(gpu, pages, tables, lengths)
    if out is None:
        if rows is None:
            if starts is not None:
                raise ValueError("rows must be given with starts")
            rows = view.table_rows if sequences is None else len(sequences)
        shape = (int(rows), view.kv_heads, view.head_dim)
        out = (torch.zeros(shape, dtype=dtype, device=pages.device), torch.zeros(shape, dtype=dtype, device=pages.device))
    k, v = out
    n, _, _, _, kind = _heads(gpu, k, "out[0]", view.kv_heads, view.head_dim)
    m, _, _, _, other = _heads(gpu, v, "out[1]", view.kv_heads, view.head_dim)
    if n != m or kind != other or not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError("out holds two contiguous tensors of the same shape and dtype")
    listed = _rows(gpu, n, view, starts, sequences)
    if n and listed.sequences:
        check(lib.lsx_cache_read_device(gpu.handle, C.byref(view), C.byref(listed), kind, k.data_ptr(), v.data_ptr(),
                                        _stream(gpu.device)))
        _written((k, v))
    return k, v


def attention(gpu: Gpu, q: torch.Tensor, pages: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor,
              starts: torch.Tensor | None = None, *, sequences: torch.Tensor | None = None, scale: float | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of queries [rows, q_heads, head_dim] over their sequences'
    positions (lsx_cache_attention_device); scale defaults to head_dim ** -0.5.  A new
    result is contiguous, and 0 in rows of no sequence."""
    view = _view(gpu, pages, tables, lengths)
    n, heads, q_row, q_head, kind = _heads(gpu, q, "queries", None, view.head_dim)
    if heads == 0 or heads % view.kv_heads:
        raise ValueError("query heads are a multiple of key heads")
    if q.requires_grad:
        _unrecorded("queries")
    rows = _rows(gpu, n, view, starts, sequences)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if starts is None else \
            torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError("out must have the queries' shape and dtype")
    else:
        _heads(gpu, out, "out", heads, view.head_dim)
        _apart(out, "out")
    if n and rows.sequences:
        size = lib.lsx_cache_attention_workspace_bytes(gpu.handle, view.head_dim)
        workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
        check(lib.lsx_cache_attention_device(
            gpu.handle, C.byref(view), C.byref(rows), q.data_ptr(), kind, heads, q_row, q_head,
            view.head_dim ** -0.5 if scale is None else scale, out.data_ptr(), out.stride(0), out.stride(1),
            workspace.data_ptr(), size, _stream(gpu.device)))
        _written((out,))
    return out


# ---- pages ---------------------------------------------------------------------
def _pool(gpu: Gpu, pool: torch.Tensor, pages: int | None = None) -> CachePool:
    if not (isinstance(pool, _Tensor) and pool.dim() >= 3 and pool.get_device() == gpu.device and pool.numel()):
        raise ValueError("the pool must be a [layers, pages, ...] tensor on the Gpu's device")
    if not pool[0].is_contiguous() or (pool.shape[0] > 1 and pool.stride(0) < pool[0].numel()):
        raise ValueError("a layer's pages must be contiguous, and layers must not overlap")
    if pages is not None and pool.shape[1] != pages:
        raise ValueError("refs must have an entry for each page of the pool")
    width = pool.element_size()
    return CachePool(pool.data_ptr(), pool.shape[0], pool.stride(0) * width, pool[0, 0].numel() * width, pool.shape[1])


def _state(gpu: Gpu, tables, lengths, refs):
    at = _ints(gpu, tables, (None, None), "tables")
    rows, width = tables.shape
    return (at, rows, width, _ints(gpu, lengths, (rows,), "lengths"), _ints(gpu, refs, (None,), "refs"))


def _missing(gpu: Gpu, missing: torch.Tensor | None, like: torch.Tensor) -> torch.Tensor:
    if missing is None:
        return torch.zeros(1, dtype=_I32, device=like.device)
    _ints(gpu, missing, (1,), "missing")
    return missing


def _listed(gpu: Gpu, t, n: int | None, name: str, most: int) -> int:
    at = _ints(gpu, t, (n,), name)
    if t.shape[0] > most:
        raise ValueError(f"{name}: at most {most} a call")
    return at


def reserve(gpu: Gpu, tables: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor, sequences: torch.Tensor,
            counts: torch.Tensor, page_size: int, *, missing: torch.Tensor | None = None) -> torch.Tensor:
    """Gives the sequences (int32) further positions and the pages for them
    (lsx_cache_reserve_device).  Returns `missing` (int32 [1]): how many pages were short;
    unless it is 0 nothing changed."""
    state = _state(gpu, tables, lengths, refs)
    missing = _missing(gpu, missing, refs)
    listed = _listed(gpu, sequences, None, "sequences", MAX_LISTED)
    more = _listed(gpu, counts, sequences.shape[0], "counts", MAX_LISTED)
    if sequences.shape[0] == 0:
        return missing.zero_()
    check(lib.lsx_cache_reserve_device(gpu.handle, *state, refs.shape[0], page_size, listed, more, sequences.shape[0],
                                       missing.data_ptr(), _stream(gpu.device)))
    _written((tables, lengths, refs, missing))
    return missing


def fork(gpu: Gpu, pool: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor,
         parents: torch.Tensor, children: torch.Tensor, page_size: int, *, missing: torch.Tensor | None = None) -> torch.Tensor:
    """Empty sequences `children` take the positions of `parents` (both int32): whole
    pages are shared, a partly filled one is copied (lsx_cache_fork_device).  Returns
    `missing` as reserve does."""
    at = _pool(gpu, pool, refs.shape[0] if isinstance(refs, _Tensor) and refs.dim() == 1 else 0)
    state = _state(gpu, tables, lengths, refs)
    missing = _missing(gpu, missing, refs)
    of = _listed(gpu, parents, None, "parents", MAX_LISTED)
    n = parents.shape[0]
    to = _listed(gpu, children, n, "children", MAX_LISTED)
    if n == 0:
        return missing.zero_()
    pairs = torch.empty((n, 2), dtype=_I32, device=refs.device)
    check(lib.lsx_cache_fork_device(gpu.handle, C.byref(at), *state, page_size, of, to, n, pairs.data_ptr(),
                                    missing.data_ptr(), _stream(gpu.device)))
    _written((pool, tables, lengths, refs, missing))
    return missing


def free(gpu: Gpu, tables: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor, sequences: torch.Tensor,
         page_size: int) -> None:
    """Empties the sequences (int32); pages that no other sequence shares become free
    (lsx_cache_free_device)."""
    state = _state(gpu, tables, lengths, refs)
    listed = _listed(gpu, sequences, None, "sequences", 1 << 20)
    if sequences.shape[0]:
        check(lib.lsx_cache_free_device(gpu.handle, *state, refs.shape[0], page_size, listed, sequences.shape[0],
                                        _stream(gpu.device)))
        _written((tables, lengths, refs))


class Compaction(NamedTuple):
    tables: torch.Tensor
    refs: torch.Tensor


def compact(gpu: Gpu, pool: torch.Tensor, tables: torch.Tensor, refs: torch.Tensor, *, out=None) -> Compaction:
    """Moves pages so that those in use are the lowest (lsx_cache_compact_device), in
    the pool; the tables and counts afterwards go to `out`, which may be the ones passed,
    or to new tensors."""
    at = _pool(gpu, pool, refs.shape[0] if isinstance(refs, _Tensor) and refs.dim() == 1 else 0)
    table = _ints(gpu, tables, (None, None), "tables")
    counts = _ints(gpu, refs, (None,), "refs")
    if out is None:
        out = (torch.empty_like(tables), torch.empty_like(refs))
    elif len(out) != 2:
        raise ValueError("out holds the tables and the counts")
    table_out = _ints(gpu, out[0], tuple(tables.shape), "out[0]")
    counts_out = _ints(gpu, out[1], tuple(refs.shape), "out[1]")
    size = lib.lsx_cache_compact_workspace_bytes(refs.shape[0])
    workspace = torch.empty(size, dtype=torch.uint8, device=refs.device)
    check(lib.lsx_cache_compact_device(gpu.handle, C.byref(at), table, tables.shape[0], tables.shape[1], counts, table_out,
                                       counts_out, workspace.data_ptr(), size, _stream(gpu.device)))
    _written((pool, out[0], out[1]))
    return Compaction(*out)


def copy_pages(gpu: Gpu, pool: torch.Tensor, pairs: torch.Tensor) -> None:
    """Copies page pairs[i, 0] to page pairs[i, 1] (int32) in every layer
    (lsx_cache_copy_device); no page may be two pairs' target, nor source and target."""
    at = _pool(gpu, pool)
    listed = _ints(gpu, pairs, (None, 2), "pairs")
    if pairs.shape[0]:
        check(lib.lsx_cache_copy_device(gpu.handle, C.byref(at), listed, pairs.shape[0], _stream(gpu.device)))
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
