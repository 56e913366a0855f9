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
from .ops import _DTYPES, _device, _is_split

PAGE_SIZES = (16, 32, 64, 128, 256)
_I32, _F32 = torch.int32, torch.float32
_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream


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


# The host's part of a call is the whole cost of a small one, so each check below is one
# expression of plain attributes (a device as its index, get_device, in 0.04 us where
# comparing device objects takes 0.12; new_empty of sizes in 1.0 where empty takes 1.7).
def _call(dev: int, name: str, fn, *args) -> None:
    """``fn(*args, stream)`` on device ``dev``, made the current one for the launch if it
    is not."""
    if _current_device() == dev:
        status = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, _raw_stream(dev))
    if status:
        check(status, name)


def _on(t: torch.Tensor) -> int:
    """The index of a call's device, that of its first tensor."""
    dev = t.get_device()
    if dev < 0:
        _device(t)
    return dev


def _ints(t: torch.Tensor, dev: int, name: str, n: int) -> int:
    """Pointer of a contiguous int32 vector of ``n`` entries (-1: any number)."""
    shape = t.shape
    if t.dtype is not _I32 or len(shape) != 1 or (n >= 0 and shape[0] != n) \
            or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 vector"
                         + (f" of {n} entries" if n >= 0 else "") + " on the call's device")
    return t.data_ptr()


def _flag(error_flag: torch.Tensor | None, dev: int) -> int:
    if error_flag is None:
        return 0
    if error_flag.get_device() != dev or error_flag.dtype is not _I32 or error_flag.numel() < 1:
        raise ValueError("error_flag must be an int32 tensor on the call's device")
    return error_flag.data_ptr()


def _table(table: torch.Tensor, dev: int) -> tuple:
    shape = table.shape
    if table.dtype is not _I32 or len(shape) != 2 or table.get_device() != dev \
            or not table.is_contiguous():
        raise ValueError("table must be a contiguous int32 [rows, width] tensor on the call's "
                         "device")
    return shape


def _pages(k_pages: torch.Tensor, v_pages: torch.Tensor, like: torch.Tensor, dev: int):
    """Shape of a layer's page tensors."""
    shape = k_pages.shape
    if len(shape) != 4 or v_pages.shape != shape or k_pages.dtype is not like.dtype \
            or v_pages.dtype is not like.dtype or k_pages.get_device() != dev \
            or v_pages.get_device() != dev or not k_pages.is_contiguous() \
            or not v_pages.is_contiguous():
        raise ValueError("k_pages and v_pages must be contiguous [pages, kv_heads, page_size, "
                         "head_dim] tensors of q's dtype and device")
    return shape


def _rows(t: torch.Tensor, like: torch.Tensor, dev: int, name: str):
    """Shape and (token, head) strides of a ``[n, heads, head_dim]`` view."""
    shape, strides = t.shape, t.stride()
    if len(shape) != 3 or strides[2] != 1 or t.dtype is not like.dtype or t.get_device() != dev:
        raise ValueError(f"{name} must be [tokens, heads, head_dim] with contiguous rows, of q's "
                         "dtype and device")
    return shape, (strides[0] if shape[0] > 1 else shape[1] * shape[2],
                   strides[1] if shape[1] > 1 else shape[2])


def _rope(tables, rotary_dim: int, dev: int) -> tuple:
    """(cos pointer, sin pointer, length) of the rotation tables."""
    if not rotary_dim:
        return 0, 0, 0
    if tables is None or len(tables) != 2:
        raise ValueError("rotation needs the (cos, sin) tables of rope_tables")
    cos, sin = tables
    shape = cos.shape
    if len(shape) != 2 or shape[1] != rotary_dim // 2 or sin.shape != shape \
            or cos.dtype is not _F32 or sin.dtype is not _F32 or cos.get_device() != dev \
            or sin.get_device() != dev or not cos.is_contiguous() or not sin.is_contiguous():
        raise ValueError("cos and sin must be contiguous float32 [n_pos, rotary_dim//2] tables of "
                         "one shape on the call's device")
    return cos.data_ptr(), sin.data_ptr(), shape[0]


def _code(t: torch.Tensor) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"unsupported dtype {t.dtype}; expected float32 or bfloat16")
    return code


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
    dev, code = _on(q), _code(q)
    (T, H, hd), q_strides = _rows(q, q, dev, "q")
    k_shape, k_strides = _rows(k, q, dev, "k")
    v_shape, v_strides = _rows(v, q, dev, "v")
    KV = k_shape[1]
    if v_shape != k_shape or k_shape[0] != T or k_shape[2] != hd:
        raise ValueError("q must be [T, H, hd] and k, v [T, KV, hd]")
    for w in (q_norm, k_norm):
        if w.dtype is not q.dtype or w.numel() != hd or w.get_device() != dev \
                or not w.is_contiguous():
            raise ValueError(f"q_norm and k_norm must be contiguous vectors of {hd} elements, of "
                             "q's dtype and device")
    page_shape = _pages(k_pages, v_pages, q, dev)
    if page_shape[1] != KV or page_shape[3] != hd:
        raise ValueError("k_pages and v_pages must hold k's heads")
    cos, sin, table_len = _rope(tables, rotary_dim, dev)
    n_rows, width = _table(table, dev)
    index, at = _ints(rows, dev, "rows", T), _ints(positions, dev, "positions", T)
    if q_out is None:
        q_out = q.new_empty(T, H, hd)
    elif q_out.shape != q.shape or q_out.dtype is not q.dtype or q_out.get_device() != dev \
            or not q_out.is_contiguous():
        raise ValueError("q_out must be a contiguous tensor of q's shape, dtype and device")
    if k_out is not None and (k_out.shape != k_shape or k_out.dtype is not q.dtype
                              or k_out.get_device() != dev or not k_out.is_contiguous()):
        raise ValueError("k_out must be a contiguous tensor of k's shape, dtype and device")
    _call(dev, "prepare_paged", lib().qdc_prepare_paged, q_out.data_ptr(),
          0 if k_out is None else k_out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
          q.data_ptr(), k.data_ptr(), v.data_ptr(), q_norm.data_ptr(), k_norm.data_ptr(),
          cos, sin, index, at, table.data_ptr(), T, H, KV, hd, rotary_dim, table_len, n_rows, width,
          page_shape[0], page_shape[2], *q_strides, *k_strides, *v_strides, eps, code,
          _flag(error_flag, dev))
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
    dev, code = _on(q), _code(q)
    (n, H, hd), q_strides = _rows(q, q, dev, "q")
    pages, KV, page, page_hd = _pages(k_pages, v_pages, q, dev)
    if page_hd != hd or KV == 0 or H % KV:
        raise ValueError("q's heads must be a multiple of those of k_pages, of one head_dim")
    n_rows, width = _table(table, dev)
    index, at = _ints(rows, dev, "rows", n), _ints(positions, dev, "positions", n)
    gate_at, gate_strides = 0, (0, hd)
    if gate is not None:
        gate_shape, gate_strides = _rows(gate, q, dev, "gate")
        if gate_shape != q.shape:
            raise ValueError("gate must be a view like q")
        gate_at = gate.data_ptr()
    if out_dtype is None:
        split, out_code, odt = False, code, q.dtype
    else:
        split = _is_split(out_dtype)
        odt = torch.bfloat16 if split else out_dtype
        out_code = _lib.QDC_BF16X2 if split else _DTYPES.get(odt)
        if out_code is None:
            raise ValueError("out_dtype must be float32, bfloat16 or BF16X2")
    out = q.new_empty(n, 2 * H * hd if split else H * hd, dtype=odt)
    need = lib().qdc_paged_attention_workspace(n, H, KV, hd, width, page, code)
    work = q.new_empty(need, dtype=torch.uint8) if need > 0 else None
    _call(dev, "paged_attention", lib().qdc_paged_attention, out.data_ptr(), out_code,
          q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), gate_at, table.data_ptr(), index,
          at, n, H, KV, hd, n_rows, width, pages, page, *q_strides, *gate_strides, H * hd, scale,
          code, 0 if work is None else work.data_ptr(), need, _flag(error_flag, dev))
    return out


# ------------------------------------------------------------------- pages ---
def _book(book: PageTable) -> tuple:
    """Of a page table: the device, (four pointers), (rows, width, pages, page size)."""
    table, lengths, refs, free, size = book
    dev = _on(table)
    rows, width = _table(table, dev)
    at = (table.data_ptr(), _ints(lengths, dev, "lengths", rows), _ints(refs, dev, "refs", -1),
          _ints(free, dev, "free", 1 + refs.shape[0]))
    return dev, at, (rows, width, refs.shape[0], size)


def _pool(pool: torch.Tensor | None, items: int, dev: int):
    """``(pointer, planes, bytes of an item)`` of a contiguous ``[planes, items, ...]``."""
    if pool is None:
        return 0, 0, 0
    shape = pool.shape
    if len(shape) < 3 or shape[1] != items or pool.get_device() != dev or not pool.is_contiguous():
        raise ValueError(f"pool must be a contiguous [planes, {items}, ...] tensor on the call's "
                         "device")
    # (strides of axes of one entry may be anything)
    return (pool.data_ptr(), shape[0],
            pool.numel() // max(1, shape[0] * items) * pool.element_size())


def extend_pages(book: PageTable, rows: torch.Tensor, counts: torch.Tensor | None = None,
                 positions: torch.Tensor | None = None,
                 error_flag: torch.Tensor | None = None) -> torch.Tensor:
    """``counts[i]`` more positions (default one each) for cache row ``rows[i]``: their
    pages are taken from the free ones and the lengths grow.  Returns ``positions``
    (int32), the first new position of each entry, -1 for a negative row.  A call that
    cannot be done whole -- a row out of range or named twice, a negative count, a row
    longer than its table, too few free pages -- does nothing but set every position
    to -1 and ``error_flag``."""
    dev, at, sizes = _book(book)
    index = _ints(rows, dev, "rows", -1)
    n = rows.shape[0]
    many = 0 if counts is None else _ints(counts, dev, "counts", n)
    if positions is None:
        positions = rows.new_empty(n)
    _call(dev, "extend_pages", lib().qdc_pages_extend, _ints(positions, dev, "positions", n), *at,
          index, many, n, *sizes, _flag(error_flag, dev))
    return positions


def free_pages(book: PageTable, rows: torch.Tensor,
               error_flag: torch.Tensor | None = None) -> None:
    """Rows give up their pages and are empty; pages that no other row shares are free
    again (an empty row: nothing).  Negative rows are left out; a row out of range or
    named twice: nothing is done and ``error_flag`` is set."""
    dev, at, sizes = _book(book)
    _call(dev, "free_pages", lib().qdc_pages_free, *at, _ints(rows, dev, "rows", -1),
          rows.shape[0], *sizes, _flag(error_flag, dev))


def fork_pages(book: PageTable, parents: torch.Tensor, children: torch.Tensor,
               pool: torch.Tensor | None = None,
               error_flag: torch.Tensor | None = None) -> None:
    """Row ``children[i]`` (empty) becomes a copy of row ``parents[i]``: full pages are
    shared, the one that is not full is copied within every plane of ``pool [planes,
    pages, kv_heads, page_size, head_dim]`` (the positions it holds).  Entries with a
    negative row are left out.  A child that is not empty, named twice or also a
    parent, a row out of range, too few free pages: nothing is done and ``error_flag``
    is set."""
    dev, at, sizes = _book(book)
    src = _ints(parents, dev, "parents", -1)
    n = parents.shape[0]
    dst = _ints(children, dev, "children", n)
    pool_at, planes, _ = _pool(pool, sizes[2], dev)
    heads = token = 0
    if pool is not None:
        shape = pool.shape
        if len(shape) != 5 or shape[3] != book.page_size:
            raise ValueError("pool must be [planes, pages, kv_heads, page_size, head_dim]")
        heads, token = shape[2], shape[4] * pool.element_size()
    need = lib().qdc_pages_fork_workspace(n, sizes[3], planes, heads, token)
    work = parents.new_empty(need, dtype=torch.uint8) if need else None
    _call(dev, "fork_pages", lib().qdc_pages_fork, *at, src, dst, n, *sizes, pool_at, planes,
          heads, token, work.data_ptr() if need else 0, need, _flag(error_flag, dev))


def compact_pages(book: PageTable, pool: torch.Tensor | None = None) -> None:
    """The pages in use move to the low end, in every plane of ``pool [planes, pages,
    ...]``: with ``m`` of them, the k-th free page below ``m`` takes the k-th page in
    use from ``m`` on.  Tables and refs follow; the stack holds the rest, lowest on top."""
    dev, at, (rows, width, pages, _) = _book(book)
    pool_at, planes, nbytes = _pool(pool, pages, dev)
    need = lib().qdc_pages_compact_workspace(pages)
    work = book.table.new_empty(need, dtype=torch.uint8)
    _call(dev, "compact_pages", lib().qdc_pages_compact, at[0], at[2], at[3], rows, width, pages,
          pool_at, planes, nbytes, work.data_ptr(), need)


def copy_pages(pool: torch.Tensor, src: torch.Tensor, dst: torch.Tensor,
               error_flag: torch.Tensor | None = None) -> None:
    """Items ``src[i]`` -> ``dst[i]`` in every plane of a contiguous ``pool [planes,
    items, ...]`` (items of a multiple of 16 bytes): pages, or the states and rings of
    rows.  Pairs with a negative index are left out; a pair out of range, or whose
    ``dst`` is an earlier pair's or any pair's ``src``, is not copied and sets
    ``error_flag``.  At most 4096 pairs a call."""
    dev = _on(pool)
    index = _ints(src, dev, "src", -1)
    n = src.shape[0]
    items = pool.shape[1] if pool.dim() > 1 else -1
    at, planes, nbytes = _pool(pool, items, dev)
    _call(dev, "copy_pages", lib().qdc_copy_pages, at, index, _ints(dst, dev, "dst", n), n, planes,
          items, nbytes, _flag(error_flag, dev))


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
    dev, code, dtype = _on(proj), _code(proj), proj.dtype
    vw = value_heads * value_dim
    channels = 2 * key_heads * key_dim + vw
    n, width = proj.shape if proj.dim() == 2 else (0, -1)
    if width < channels + vw + 2 * value_heads or proj.stride(1) != 1:
        raise ValueError("proj must be [n, width] with contiguous rows of the q|k|v|z|a|b blocks")
    taps = conv.shape[-1]
    if conv.shape != (channels, taps) or conv.dtype is not _F32 or conv.get_device() != dev \
            or not conv.is_contiguous():
        raise ValueError(f"conv must be a contiguous float32 [{channels}, taps] tensor (the q|k|v "
                         "channels) on proj's device")
    for t in (a_decay, dt_bias):
        if t.dtype is not _F32 or t.numel() != value_heads or t.get_device() != dev \
                or not t.is_contiguous():
            raise ValueError(f"a_decay and dt_bias must be contiguous float32 vectors of "
                             f"{value_heads} elements on proj's device")
    if norm.dtype is not dtype or norm.numel() != value_dim or norm.get_device() != dev \
            or not norm.is_contiguous():
        raise ValueError(f"norm must be a contiguous vector of {value_dim} elements of proj's "
                         "dtype and device")
    cache_rows = state.shape[0]
    if state.shape != (cache_rows, value_heads, value_dim, key_dim) or state.dtype is not _F32 \
            or state.get_device() != dev or not state.is_contiguous():
        raise ValueError("state must be a contiguous float32 [cache rows, value_heads, value_dim, "
                         "key_dim] tensor on proj's device")
    if ring.shape != (cache_rows, taps, channels) or ring.dtype is not dtype \
            or ring.get_device() != dev or not ring.is_contiguous():
        raise ValueError(f"ring must be a contiguous [cache rows, {taps}, {channels}] tensor of "
                         "proj's dtype and device")
    index, at = _ints(rows, dev, "rows", n), _ints(positions, dev, "positions", n)
    split = out_dtype is not None and _is_split(out_dtype)
    if split and dtype is not torch.bfloat16:
        raise ValueError("the split output takes a bfloat16 proj")
    if not split and out_dtype not in (None, dtype):
        raise ValueError("out_dtype must be proj's dtype or BF16X2")
    out = proj.new_empty(n, 2 * vw if split else vw)
    _call(dev, "delta_step", lib().qdc_delta_step, out.data_ptr(),
          _lib.QDC_BF16X2 if split else code, proj.data_ptr(), code,
          proj.stride(0) if n > 1 else width, conv.data_ptr(), taps, a_decay.data_ptr(),
          dt_bias.data_ptr(), norm.data_ptr(), ring.data_ptr(), state.data_ptr(), index, at, n,
          cache_rows, key_heads, key_dim, value_heads, value_dim, eps, _flag(error_flag, dev))
    return out
