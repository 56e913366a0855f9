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
from ._lib import calls
from .ops import _DTYPES, _is_split

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
    lowest of ``pages`` free pages on top of the stack.  ``rows`` below 2^18, ``width *
    page_size`` below 2^31, ``pages`` and ``rows * width`` at most 2^31 - 1024."""
    if rows <= 0 or width <= 0 or pages <= 0 or page_size not in PAGE_SIZES:
        raise ValueError(f"rows, width and pages must be positive, page_size one of {PAGE_SIZES}")
    most = 2 ** 31 - 1024
    if rows >= 2 ** 18 or width * page_size >= 2 ** 31 or pages > most or rows * width > most:
        raise ValueError("too many rows or pages, or too wide a table, for the operators")
    i32 = dict(dtype=torch.int32, device=device)
    free = torch.empty(1 + pages, **i32)
    free[0] = pages
    free[1:] = torch.arange(pages - 1, -1, -1, **i32)
    return PageTable(torch.full((rows, width), -1, **i32), torch.zeros(rows, **i32),
                     torch.zeros(pages, **i32), free, page_size)


# The host's part of a call is the whole cost of a small one, so the tensors are checked and
# the entry points called by a compiled module, csrc/qdc_calls.cpp (4.6 to 4.9 us of the
# host's time for a call of one launch, 5 to 7 less than the same in Python).


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
    cos, sin = (None, None) if tables is None or not rotary_dim else tables
    return calls().prepare_paged(q, k, v, q_norm, k_norm, cos, sin, rotary_dim, eps, rows, positions,
                                 table, k_pages, v_pages, q_out, k_out, error_flag)


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
    code = -1
    if out_dtype is not None:
        code = _lib.QDC_BF16X2 if _is_split(out_dtype) else _DTYPES.get(out_dtype)
        if code is None:
            raise ValueError("out_dtype must be float32, bfloat16 or BF16X2")
    return calls().paged_attention(q, k_pages, v_pages, table, rows, positions, scale, gate, code,
                                   error_flag)


# ------------------------------------------------------------------- pages ---
def extend_pages(book: PageTable, rows: torch.Tensor, counts: torch.Tensor | None = None,
                 positions: torch.Tensor | None = None,
                 error_flag: torch.Tensor | None = None) -> torch.Tensor:
    """``counts[i]`` more positions (default one each) for cache row ``rows[i]``: their
    pages are taken from the free ones and the lengths grow.  Returns ``positions``
    (int32), the first new position of each entry, -1 for a negative row.  A call that
    cannot be done whole -- a row out of range or named twice, a negative count, a row
    longer than its table, too few free pages -- does nothing but set every position
    to -1 and ``error_flag``."""
    return calls().extend_pages(*book, rows, counts, positions, error_flag)


def free_pages(book: PageTable, rows: torch.Tensor,
               error_flag: torch.Tensor | None = None) -> None:
    """Rows give up their pages and are empty; pages that no other row shares are free
    again (an empty row: nothing).  Negative rows are left out; a row out of range or
    named twice: nothing is done and ``error_flag`` is set."""
    calls().free_pages(*book, rows, error_flag)


def fork_pages(book: PageTable, parents: torch.Tensor, children: torch.Tensor,
               pool: torch.Tensor | None = None,
               error_flag: torch.Tensor | None = None) -> None:
    """Row ``children[i]`` (empty) becomes a copy of row ``parents[i]``: full pages are
    shared, the one that is not full is copied within every plane of ``pool [planes,
    pages, kv_heads, page_size, head_dim]`` (the positions it holds).  Entries with a
    negative row are left out.  A child that is not empty, named twice or also a
    parent, a row out of range, too few free pages: nothing is done and ``error_flag``
    is set."""
    calls().fork_pages(*book, parents, children, pool, error_flag)


def compact_pages(book: PageTable, pool: torch.Tensor | None = None) -> None:
    """The pages in use move to the low end, in every plane of ``pool [planes, pages,
    ...]``: with ``m`` of them, the k-th free page below ``m`` takes the k-th page in
    use from ``m`` on.  Tables and refs follow; the stack holds the rest, lowest on top."""
    calls().compact_pages(*book, pool)


def copy_pages(pool: torch.Tensor, src: torch.Tensor, dst: torch.Tensor,
               error_flag: torch.Tensor | None = None) -> None:
    """Items ``src[i]`` -> ``dst[i]`` in every plane of a contiguous ``pool [planes,
    items, ...]`` (items of a multiple of 16 bytes): pages, or the states and rings of
    rows.  Pairs with a negative index are left out; a pair out of range, or whose
    ``dst`` is an earlier pair's or any pair's ``src``, is not copied and sets
    ``error_flag``.  At most 4096 pairs a call."""
    calls().copy_pages(pool, src, dst, error_flag)


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
    split = out_dtype is not None and _is_split(out_dtype)
    if split and proj.dtype is not torch.bfloat16:
        raise ValueError("the split output takes a bfloat16 proj")
    if not split and out_dtype not in (None, proj.dtype):
        raise ValueError("out_dtype must be proj's dtype or BF16X2")
    return calls().delta_step(proj, conv, a_decay, dt_bias, norm, eps, ring, state, rows, positions,
                              key_heads, key_dim, value_heads, value_dim, split, error_flag)
