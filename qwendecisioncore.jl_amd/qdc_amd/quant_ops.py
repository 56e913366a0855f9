"""Device operators on weights held in 4 bits and rows held in 8, on PyTorch-ROCm tensors.

The reference keeps every weight in fp32 or bf16 and has none of these.  They follow
:mod:`qdc_amd.ops`: each call enqueues kernels of ``libqdc_hip.so`` on the tensor
device's current PyTorch stream, torch supplies memory and stream only, and argument
errors raise ``ValueError`` before anything is enqueued.  Nothing is kept between calls,
and every call can be captured into a HIP graph.  Tensors begin at 16-byte addresses (the
scales of 8-bit rows at 4-byte ones).

A :class:`W4` is a projection ``[out, inner]`` whose weights are whole numbers of -8..7
times a bfloat16 scale for each output and ``group`` inputs, laid out once by
:func:`pack_w4` as the products read it.  A :class:`Q8` is a matrix of rows whose values
are whole numbers of -127..127 times a float32 scale for each 128 columns.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from ._lib import calls
from .ops import _DTYPES

GROUPS = (32, 64, 128)


class W4(NamedTuple):
    """A weight in 4 bits.  ``packed`` int32 ``[blocks, ceil(inner / 128), 64, 4]`` and
    ``scales`` bfloat16 ``[blocks, ceil(inner / 128) * 128 / group, 16]``, blocks of 16
    outputs, as ``include/qdc_hip_quant.h`` lays them out.  ``gated``: two weights of
    ``out / 2`` outputs, gate and up, in alternating blocks, for :func:`gated_w4`."""
    packed: torch.Tensor
    scales: torch.Tensor
    out: int
    inner: int
    group: int
    gated: bool = False

    def outputs(self, first: int, last: int) -> "W4":
        """The weight of outputs ``first .. last - 1`` alone (a view; multiples of 16,
        ``last`` may be the end; not of a gated weight)."""
        if self.gated or not 0 <= first < last <= self.out or first % 16 \
                or (last % 16 and last != self.out):
            raise ValueError("outputs are taken in blocks of 16, and not of a gated weight")
        blocks = slice(first // 16, -(-last // 16))
        return W4(self.packed[blocks], self.scales[blocks], last - first, self.inner, self.group)


class Q8(NamedTuple):
    """Rows in 8 bits: ``values`` int8 ``[rows, width]`` and ``scales`` float32 ``[rows,
    ceil(width / 128)]``, both contiguous, width a multiple of 16.  A group of zeros has
    scale 0; one that held an infinity or NaN has it as its scale, and its values are NaN.
    As an ``out_dtype`` it asks for such rows."""
    values: torch.Tensor
    scales: torch.Tensor


def _code(dtype, what="out_dtype") -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"{what} must be float32 or bfloat16")
    return code


def pack_w4(w: torch.Tensor, group: int = 64, gated: bool = False) -> W4:
    """``w [out, inner]`` (float32 or bfloat16, contiguous rows, inner a multiple of 8) in
    4 bits: the scale of a group is ``max |w| / 7`` rounded to bfloat16, a weight the
    nearest whole number of it (ties to even) within -7..7.  A group that holds an infinity
    or NaN has a NaN scale.  ``gated``: ``w`` is ``[gate; up]``, for :func:`gated_w4`."""
    packed, scales = calls().pack_w4(w, group, gated)
    return W4(packed, scales, w.shape[0], w.shape[1], group, bool(gated))


def unpack_w4(w: W4, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The weights ``[out, inner]`` that ``w`` stands for, in float32 (exact) or bfloat16."""
    return calls().unpack_w4(*w, _code(dtype, "dtype"))


def quantize_q8(x: torch.Tensor) -> Q8:
    """Rows ``x [rows, width]`` (float32 or bfloat16, contiguous rows a multiple of 8
    elements apart) in 8 bits: the scale of 128 columns is ``max |x| / 127``, a value the
    nearest whole number of it (ties to even)."""
    return Q8(*calls().quantize_q8(x))


def dequantize_q8(q: Q8, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values ``[rows, width]`` that ``q`` stands for, in float32 or bfloat16."""
    return calls().dequantize_q8(*q, _code(dtype, "dtype"))


def residual_rms_q8(x: torch.Tensor, add: torch.Tensor | None, weight: torch.Tensor, eps: float,
                    token_mask: torch.Tensor | None = None):
    """:func:`ops.native_residual_rms` of a float32 stream with the normalised rows in 8
    bits: ``(x + add, Q8 of rms(x + add) * (1 + weight))``.  Without ``add`` (None) the
    first is ``x`` itself.  Rows whose ``token_mask`` (int32) is 0 are zeros.  ``x`` and
    ``add`` contiguous ``[rows, width]``, width a multiple of 16 up to 32768, ``weight``
    float32 or bfloat16."""
    residual, values, scales = calls().residual_rms_q8(x, add, weight, eps, token_mask)
    return residual, Q8(values, scales)


def linear_w4(x, w: W4, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x @ W.T [rows, out]`` for ``x [rows, inner]``: float32 or bfloat16 (contiguous rows
    a multiple of 8 elements and at most 2^26 bytes apart) or :class:`Q8`.  Sums are float32, of whole numbers
    times ``x`` within a group and scaled after, and rounded once to ``out_dtype`` (float32
    or bfloat16; default ``x``'s, bfloat16 for Q8 rows).  float32 rows keep all their bits.
    Up to 2^20 - 16 rows."""
    if w.gated:
        raise ValueError("a gated weight goes to gated_w4")
    return _product(x, w, -1 if out_dtype is None else _code(out_dtype))


def gated_w4(x, w: W4, out_dtype=None):
    """``silu(x @ gate.T) * (x @ up.T) [rows, out / 2]``, for ``w`` packed with ``gated=True`` and
    ``x`` as in :func:`linear_w4`: :func:`ops.native_mlp_gate` of both projections, kept in
    float32 in between.  ``out_dtype`` may also be :class:`Q8` (out / 2 a multiple of 16), for
    the next product.  One kernel; for 8-bit results of few rows two, with the float32 ones
    between them in a scratch tensor of the call's stream."""
    if not w.gated:
        raise ValueError("gated_w4 takes a weight packed with gated=True")
    if out_dtype is Q8:
        return Q8(*_product(x, w, _lib.QDC_Q8))
    return _product(x, w, -1 if out_dtype is None else _code(out_dtype))


def _product(x, w, code):
    if isinstance(x, Q8):
        return calls().linear_w4(x.values, x.scales, *w, code)
    return calls().linear_w4(x, None, *w, code)
