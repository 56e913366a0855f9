"""Device operators of a cache that the backbone decodes from, on PyTorch-ROCm tensors.

The reference runs a sequence again for every call and has none of these.  They
follow :mod:`qdc_amd.ops`: each call enqueues kernels of ``libqdc_hip.so`` on the
tensor device's current PyTorch stream, torch supplies memory and stream only, and
argument errors raise ``ValueError`` before anything is enqueued.

A cache holds ``rows`` sequences (rows) in pages of ``page_size`` positions (16, 32,
64, 128 or 256).  Per attention layer the pages are two tensors ``[pages, kv_heads,
page_size, head_dim]``, planes of one pool ``[planes, pages, ...]``; which page is
whose is a :class:`PageTable`, on the device.  Per linear attention layer a row has a
state ``[value_heads, value_dim, key_dim]`` (float32) and a ring of its last ``taps``
convolution inputs.

A call's tokens are named by ``rows`` (the cache row) and ``positions``, contiguous
device int32 vectors; an entry with a negative row or position is no token.  What is
only known on the device -- a row, position or page outside its table, a row named
twice, too few free pages -- cannot raise: the kernels never follow it, do as each
function says, and set ``error_flag`` (a device int32 that the caller clears and
reads) where one is given.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from ._lib import check, lib
from .ops import (_DTYPES, _device, _dtype_code, _is_split, _rope_tables, _stream, _vector)

PAGE_SIZES = (16, 32, 64, 128, 256)


class PageTable(NamedTuple):
    """Which page holds which positions of which row (all device int32, contiguous):
    ``table [rows, width]`` (-1 behind a row's last page), ``lengths [rows]``, ``refs
    [pages]`` (rows that share a page) and ``free [1 + pages]`` (a count, then the
    free pages as a stack).  A page that is not full belongs to one row alone."""
    table: torch.Tensor
    lengths: torch.Tensor
    refs: torch.Tensor
    free: torch.Tensor
    page_size: int


def page_table(rows: int, width: int, pages: int, page_size: int, device) -> PageTable:
    """An empty :class:`PageTable` of ``rows`` rows of up to ``width`` pages each, the
    lowest of ``pages`` free pages on top of the stack."""
    if rows <= 0 or width <= 0 or pages <= 0 or page_size not in PAGE_SIZES:
        raise ValueError(f"rows, width and pages must be positive, page_size one of {PAGE_SIZES}")
    i32 = dict(dtype=torch.int32, device=device)
    free = torch.empty(1 + pages, **i32)
    free[0] = pages
    free[1:] = torch.arange(pages - 1, -1, -1, **i32)
    return PageTable(torch.full((rows, width), -1, **i32), torch.zeros(rows, **i32),
                     torch.zeros(pages, **i32), free, page_size)


def _ints(t: torch.Tensor, like: torch.Tensor, name: str, n: int | None = None) -> int:
    """Pointer of a contiguous device int32 vector (of ``n`` entries)."""
    if t.device != like.device:
        raise ValueError(f"tensors on different devices: {like.device} vs {t.device}")
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous() \
            or (n is not None and t.shape[0] != n):
        raise ValueError(f"{name} must be a contiguous int32 vector"
                         + ("" if n is None else f" of {n} entries"))
    return t.data_ptr()


def _flag(error_flag: torch.Tensor | None, like: torch.Tensor) -> int:
    if error_flag is None:
        return 0
    if error_flag.device != like.device or error_flag.dtype != torch.int32 \
            or error_flag.numel() < 1:
        raise ValueError("error_flag must be an int32 tensor on the call's device")
    return error_flag.data_ptr()


def _table(table: torch.Tensor, like: torch.Tensor) -> tuple:
    if table.device != like.device:
        raise ValueError(f"tensors on different devices: {like.device} vs {table.device}")
    if table.dtype != torch.int32 or table.dim() != 2 or not table.is_contiguous():
        raise ValueError("table must be a contiguous int32 [rows, width] tensor")
    return table.shape


def _pages(k_pages: torch.Tensor, v_pages: torch.Tensor, like: torch.Tensor, kv: int, hd: int):
    """(pages, page_size) of a layer's page tensors."""
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.shape[1] != kv \
            or k_pages.shape[3] != hd:
        raise ValueError("k_pages and v_pages must be [pages, kv_heads, page_size, head_dim]")
    for t in (k_pages, v_pages):
        if t.dtype != like.dtype or not t.is_contiguous() or t.device != like.device:
            raise ValueError("k_pages and v_pages must be contiguous, of q's dtype and device")
    return k_pages.shape[0], k_pages.shape[2]


def _heads(t: torch.Tensor, n: int) -> tuple:
    """(token stride, head stride) of a ``[n, heads, head_dim]`` view."""
    return (t.stride(0) if n > 1 else t.shape[1] * t.shape[2],
            t.stride(1) if t.shape[1] > 1 else t.shape[2])


# --------------------------------------------------------------- attention ---
def prepare_paged(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_norm: torch.Tensor,
                  k_norm: torch.Tensor, tables, rotary_dim: int, eps: float, rows: torch.Tensor,
                  positions: torch.Tensor, table: torch.Tensor, k_pages: torch.Tensor,
                  v_pages: torch.Tensor, q_out: torch.Tensor | None = None,
                  k_out: torch.Tensor | None = None,
                  error_flag: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`ops.prepare_heads` for tokens at positions of their own, with K and V
    stored into the cache in the same launch: ``q [T, H, hd]``, ``k`` and ``v [T, KV,
    hd]`` (views with contiguous rows), token ``t`` rotated to ``positions[t]`` and its
    k and v written to that position of cache row ``rows[t]``.  Returns the prepared q
    ``[T, H, hd]``; ``k_out`` (contiguous ``[T, KV, hd]``) takes the prepared k too, for
    attention within a prompt.  An entry that is no token is normalised, not rotated
    and not stored; the same, with ``error_flag`` set, for one whose position is beyond
    the rotation tables or the row's pages.  Of two tokens at one position of one row,
    either may be stored, or pieces of both.  head_dim 64, 128 or 256."""
    _device(q, k, v, q_norm, k_norm)
    code = _dtype_code(q, k, v, q_norm, k_norm)
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or q.shape[0] != k.shape[0] \
            or q.shape[2] != k.shape[2]:
        raise ValueError("q must be [T, H, hd] and k, v [T, KV, hd]")
    T, H, hd = q.shape
    KV = k.shape[1]
    for t in (q, k, v):
        if t.stride(2) != 1:
            raise ValueError("rows must be contiguous")
    _vector(q_norm, hd, "q_norm")
    _vector(k_norm, hd, "k_norm")
    pages, page = _pages(k_pages, v_pages, q, KV, hd)
    cos, sin = _rope_tables(tables, rotary_dim, q)
    n_rows, width = _table(table, q)
    index, at = _ints(rows, q, "rows", T), _ints(positions, q, "positions", T)
    if q_out is None:
        q_out = torch.empty((T, H, hd), dtype=q.dtype, device=q.device)
    for out, shape in ((q_out, (T, H, hd)), (k_out, (T, KV, hd))):
        if out is not None and (out.shape != shape or out.dtype != q.dtype
                                or not out.is_contiguous() or out.device != q.device):
            raise ValueError("q_out and k_out must be contiguous tensors of q's and k's shape, "
                             "of q's dtype and device")
    check(lib().qdc_prepare_paged(
        q_out.data_ptr(), 0 if k_out is None else k_out.data_ptr(), k_pages.data_ptr(),
        v_pages.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), q_norm.data_ptr(),
        k_norm.data_ptr(), 0 if cos is None else cos.data_ptr(),
        0 if sin is None else sin.data_ptr(), index, at, table.data_ptr(), T, H, KV, hd,
        rotary_dim, 0 if cos is None else cos.shape[0], n_rows, width, pages, page, *_heads(q, T),
        *_heads(k, T), *_heads(v, T), eps, code, _flag(error_flag, q), _stream(q)),
        "prepare_paged")
    return q_out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    table: torch.Tensor, rows: torch.Tensor, positions: torch.Tensor,
                    scale: float, gate: torch.Tensor | None = None, out_dtype=None,
                    error_flag: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one token's queries over its cache row, split over all keys of the
    batch and joined: entry ``i`` sees positions ``0 .. positions[i]`` of row
    ``rows[i]`` (several entries may name one row).  ``q`` and ``gate`` (optional: the
    output gate, as in :func:`ops.attention_fused`) ``[n, H, hd]`` views with
    contiguous rows -> ``[n, H*hd]`` in ``out_dtype`` (default: q's; ``BF16X2`` writes
    ``[n, 2*H*hd]``).  Entries that are no token give zeros; positions behind the
    table's width and pages that are none count as masked and set ``error_flag``.
    ``scale`` positive; head_dim 64, 128 or 256."""
    _device(q)
    code = _dtype_code(q)
    if q.dim() != 3 or q.stride(2) != 1:
        raise ValueError("q must be [n, H, hd] with contiguous rows")
    n, H, hd = q.shape
    if k_pages.dim() != 4 or k_pages.shape[1] == 0 or H % k_pages.shape[1]:
        raise ValueError("the query heads must be a multiple of the KV heads of k_pages")
    KV = k_pages.shape[1]
    pages, page = _pages(k_pages, v_pages, q, KV, hd)
    n_rows, width = _table(table, q)
    index, at = _ints(rows, q, "rows", n), _ints(positions, q, "positions", n)
    gate_at, gate_strides = 0, (0, hd)
    if gate is not None:
        if gate.shape != q.shape or gate.dtype != q.dtype or gate.stride(2) != 1 \
                or gate.device != q.device:
            raise ValueError("gate must be a view like q with contiguous rows")
        gate_at, gate_strides = gate.data_ptr(), _heads(gate, n)
    split = _is_split(out_dtype)
    odt = torch.bfloat16 if split else out_dtype or q.dtype
    if odt not in _DTYPES:
        raise ValueError("out_dtype must be float32, bfloat16 or BF16X2")
    out = torch.empty((n, 2 * H * hd if split else H * hd), dtype=odt, device=q.device)
    need = lib().qdc_paged_attention_workspace(n, H, KV, hd, width, page, code)
    work = torch.empty(need, dtype=torch.uint8, device=q.device)
    check(lib().qdc_paged_attention(
        out.data_ptr(), _lib.QDC_BF16X2 if split else _DTYPES[odt], q.data_ptr(),
        k_pages.data_ptr(), v_pages.data_ptr(), gate_at, table.data_ptr(), index, at, n, H, KV, hd,
        n_rows, width, pages, page, *_heads(q, n), *gate_strides, H * hd, scale, code,
        work.data_ptr(), need, _flag(error_flag, q), _stream(q)), "paged_attention")
    return out


# ------------------------------------------------------------------- pages ---
def _book(book: PageTable) -> tuple:
    """The C arguments of a page table: (four pointers), (rows, width, pages, size)."""
    table, lengths, refs, free, size = book
    _device(table, lengths, refs, free)
    if table.dtype != torch.int32 or table.dim() != 2 or not table.is_contiguous():
        raise ValueError("table must be a contiguous int32 [rows, width] tensor")
    rows, width = table.shape
    pages = refs.shape[0] if refs.dim() == 1 else -1
    _ints(lengths, table, "lengths", rows)
    _ints(refs, table, "refs")
    _ints(free, table, "free", 1 + pages)
    return ((table.data_ptr(), lengths.data_ptr(), refs.data_ptr(), free.data_ptr()),
            (rows, width, pages, size))


def _pool(pool: torch.Tensor | None, items: int, like: torch.Tensor, name: str):
    """``(pointer, planes, bytes of an item)`` of a contiguous ``[planes, items, ...]``."""
    if pool is None:
        return 0, 0, 0
    if pool.dim() < 3 or pool.shape[1] != items or not pool.is_contiguous() \
            or pool.device != like.device:
        raise ValueError(f"{name} must be a contiguous [planes, {items}, ...] tensor on the "
                         "call's device")
    return (pool.data_ptr(), pool.shape[0],
            pool.numel() // max(1, pool.shape[0] * items) * pool.element_size())


def extend_pages(book: PageTable, rows: torch.Tensor, counts: torch.Tensor | None = None,
                 positions: torch.Tensor | None = None,
                 error_flag: torch.Tensor | None = None) -> torch.Tensor:
    """``counts[i]`` more positions (default one each) for cache row ``rows[i]``: their
    pages are taken from the free ones and the lengths grow.  Returns ``positions``
    (int32), the first new position of each entry, -1 for a negative row.  A call that
    cannot be done whole -- a row out of range or named twice, a negative count, a row
    longer than its table, too few free pages -- does nothing but set every position
    to -1 and ``error_flag``."""
    at, sizes = _book(book)
    index = _ints(rows, book.table, "rows")
    n = rows.shape[0]
    many = 0 if counts is None else _ints(counts, book.table, "counts", n)
    if positions is None:
        positions = torch.empty(n, dtype=torch.int32, device=rows.device)
    out = _ints(positions, book.table, "positions", n)
    check(lib().qdc_pages_extend(out, *at, index, many, n, *sizes, _flag(error_flag, book.table),
                                 _stream(rows)), "extend_pages")
    return positions


def free_pages(book: PageTable, rows: torch.Tensor,
               error_flag: torch.Tensor | None = None) -> None:
    """Rows give up their pages and are empty; pages that no other row shares are free
    again (an empty row: nothing).  Negative rows are left out; a row out of range or
    named twice: nothing is done and ``error_flag`` is set."""
    at, sizes = _book(book)
    index = _ints(rows, book.table, "rows")
    check(lib().qdc_pages_free(*at, index, rows.shape[0], *sizes, _flag(error_flag, book.table),
                               _stream(rows)), "free_pages")


def fork_pages(book: PageTable, parents: torch.Tensor, children: torch.Tensor,
               pool: torch.Tensor | None = None,
               error_flag: torch.Tensor | None = None) -> None:
    """Row ``children[i]`` (empty) becomes a copy of row ``parents[i]``: full pages are
    shared, the one that is not full is copied within every plane of ``pool [planes,
    pages, kv_heads, page_size, head_dim]`` (the positions it holds).  Entries with a
    negative row are left out.  A child that is not empty, named twice or also a
    parent, a row out of range, too few free pages: nothing is done and ``error_flag``
    is set."""
    at, sizes = _book(book)
    src = _ints(parents, book.table, "parents")
    n = parents.shape[0]
    dst = _ints(children, book.table, "children", n)
    if pool is not None and (pool.dim() != 5 or pool.shape[3] != book.page_size):
        raise ValueError("pool must be [planes, pages, kv_heads, page_size, head_dim]")
    pool_at, planes, _ = _pool(pool, sizes[2], book.table, "pool")
    heads, token = (0, 0) if pool is None else (pool.shape[2], pool.shape[4] * pool.element_size())
    work = torch.empty(16 * n, dtype=torch.uint8, device=parents.device)
    check(lib().qdc_pages_fork(*at, src, dst, n, *sizes, pool_at, planes, heads, token,
                               work.data_ptr(), 16 * n, _flag(error_flag, book.table),
                               _stream(parents)), "fork_pages")


def compact_pages(book: PageTable, pool: torch.Tensor | None = None) -> None:
    """The pages in use move to the low end, in every plane of ``pool [planes, pages,
    ...]``: with ``m`` of them, the k-th free page below ``m`` takes the k-th page in
    use from ``m`` on.  Tables and refs follow; the stack holds the rest, lowest on top."""
    at, (rows, width, pages, _) = _book(book)
    pool_at, planes, nbytes = _pool(pool, pages, book.table, "pool")
    need = lib().qdc_pages_compact_workspace(pages)
    work = torch.empty(need, dtype=torch.uint8, device=book.table.device)
    check(lib().qdc_pages_compact(at[0], at[2], at[3], rows, width, pages, pool_at, planes, nbytes,
                                  work.data_ptr(), need, _stream(book.table)), "compact_pages")


def copy_pages(pool: torch.Tensor, src: torch.Tensor, dst: torch.Tensor,
               error_flag: torch.Tensor | None = None) -> None:
    """Items ``src[i]`` -> ``dst[i]`` in every plane of a contiguous ``pool [planes,
    items, ...]`` (items of a multiple of 16 bytes): pages, or the states and rings of
    rows.  Pairs with a negative index are left out; a pair out of range, or whose
    ``dst`` is an earlier pair's or any pair's ``src``, is not copied and sets
    ``error_flag``."""
    _device(pool)
    index = _ints(src, pool, "src")
    to = _ints(dst, pool, "dst", src.shape[0])
    items = pool.shape[1] if pool.dim() > 1 else -1
    at, planes, nbytes = _pool(pool, items, pool, "pool")
    check(lib().qdc_copy_pages(at, index, to, src.shape[0], planes, items, nbytes,
                               _flag(error_flag, pool), _stream(pool)), "copy_pages")


# -------------------------------------------------------- linear attention ---
def delta_step(proj: torch.Tensor, conv: torch.Tensor, a_decay: torch.Tensor,
               dt_bias: torch.Tensor, norm: torch.Tensor, eps: float, ring: torch.Tensor,
               state: torch.Tensor, rows: torch.Tensor, positions: torch.Tensor, key_heads: int,
               key_dim: int, value_heads: int, value_dim: int, out_dtype=None,
               error_flag: torch.Tensor | None = None) -> torch.Tensor:
    """One token of a linear attention layer for each entry, in one launch: what
    :func:`ops.delta_prologue`, :func:`ops.delta_scan` and :func:`ops.native_gated_rms`
    give for the newest token of a sequence.  ``proj [n, width]`` holds the packed
    projections ``q|k|v|z|a|b`` (rows contiguous); ``ring [cache rows, taps, q|k|v
    channels]`` (proj's dtype) the convolution's inputs, position ``p`` in slot ``p %
    taps``, and ``state [cache rows, value_heads, value_dim, key_dim]`` (float32) the
    recurrence's state: both are updated.  At position 0 a row starts empty, whatever
    they hold.  Returns the gated norm's result ``[n, value_heads*value_dim]`` in
    proj's dtype (``BF16X2``, of a bfloat16 proj: ``[n, 2*...]``).  Entries that are no
    token give zeros and leave the cache; so does a row out of range or that of an
    earlier token of the call, which sets ``error_flag``.  key_dim 32, 64 or 128,
    value_dim a multiple of 16 up to 256, up to 8 taps."""
    _device(proj, conv, a_decay, dt_bias, norm, ring, state)
    code = _dtype_code(proj, norm, ring)
    channels, vw = 2 * key_heads * key_dim + value_heads * value_dim, value_heads * value_dim
    if proj.dim() != 2 or proj.stride(1) != 1 or proj.shape[1] < channels + vw + 2 * value_heads:
        raise ValueError("proj must be [n, width] with contiguous rows of the q|k|v|z|a|b blocks")
    for t in (conv, a_decay, dt_bias, state):
        if t.dtype != torch.float32 or not t.is_contiguous():
            raise ValueError("conv, a_decay, dt_bias and state must be contiguous float32")
    if conv.dim() != 2 or conv.shape[0] != channels:
        raise ValueError(f"conv must be [{channels}, taps] (the q|k|v channels)")
    taps = conv.shape[1]
    _vector(a_decay, value_heads, "a_decay")
    _vector(dt_bias, value_heads, "dt_bias")
    _vector(norm, value_dim, "norm")
    if ring.dim() != 3 or ring.shape[1:] != (taps, channels) or not ring.is_contiguous():
        raise ValueError(f"ring must be a contiguous [cache rows, {taps}, {channels}] tensor")
    if state.shape != (ring.shape[0], value_heads, value_dim, key_dim):
        raise ValueError("state must be [cache rows, value_heads, value_dim, key_dim]")
    n = proj.shape[0]
    index, at = _ints(rows, proj, "rows", n), _ints(positions, proj, "positions", n)
    split = _is_split(out_dtype)
    if split and proj.dtype != torch.bfloat16:
        raise ValueError("the split output takes a bfloat16 proj")
    if not split and out_dtype not in (None, proj.dtype):
        raise ValueError("out_dtype must be proj's dtype or BF16X2")
    out = torch.empty((n, 2 * vw if split else vw), dtype=proj.dtype, device=proj.device)
    check(lib().qdc_delta_step(
        out.data_ptr(), _lib.QDC_BF16X2 if split else code, proj.data_ptr(), code,
        proj.stride(0) if n > 1 else proj.shape[1], conv.data_ptr(), taps, a_decay.data_ptr(),
        dt_bias.data_ptr(), norm.data_ptr(), ring.data_ptr(), state.data_ptr(), index, at, n,
        ring.shape[0], key_heads, key_dim, value_heads, value_dim, eps, _flag(error_flag, proj),
        _stream(proj)), "delta_step")
    return out
