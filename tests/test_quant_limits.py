"""The operators on 4-bit weights and 8-bit rows at the ends of their documented ranges: rows
far apart, the largest and smallest scales, quotients next to a half, tensors at any address."""
import numpy as np
import pytest
import torch

from conftest import normwise
from qdc_amd import backbone, quant_ops as qo
from test_quant_backbone import BARS, inputs, weights_of
from test_quant_ops import DEV, GROUPS, near_on_device, near_q8, product, rows_of, silu_product


def device_weight(seed, out, inner, group, gated=False, scale=0.1):
    """A weight made on the device and the values that it stands for."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = qo.pack_w4(torch.randn(out, inner, generator=g, device=DEV) * scale, group, gated)
    return w, qo.unpack_w4(w).double()


# ------------------------------------------------------------ rows far apart --
@pytest.mark.gpu
@pytest.mark.parametrize("ld", [1 << 24, 17_000_000, 1 << 25])
def test_rows_far_apart(ld):
    """128 bf16 rows up to the documented 2^26 bytes apart, of as many outputs as take the
    tallest tile: at 17e6 elements its last rows are more than 2^32 bytes from its first."""
    rows, inner, out = 128, 64, 196608
    held = torch.empty((rows - 1) * ld + inner, dtype=torch.bfloat16, device=DEV)
    x = held.as_strided((rows, inner), (ld, 1))
    x.copy_(torch.randn(rows, inner, generator=torch.Generator().manual_seed(ld)))
    w, wv = device_weight(1, out, inner, 64)
    near_on_device(qo.linear_w4(x, w), *product(x.double(), wv, 64, False), torch.bfloat16)
    del w, wv
    w, wv = device_weight(2, out, inner, 64, gated=True)
    near_on_device(qo.gated_w4(x, w), *silu_product(x.double(), wv, 64, False), torch.bfloat16)
    got = qo.gated_w4(x, w, out_dtype=qo.Q8)
    want = qo.gated_w4(x.contiguous(), w, out_dtype=qo.Q8)
    # another tile may add the same products in another order: a step of the scale
    off = (qo.dequantize_q8(got) - qo.dequantize_q8(want)).abs()
    assert (off <= 1.01 * want.scales.repeat_interleave(128, 1)).all()


# ------------------------------------------------------------ extreme scales --
@pytest.mark.gpu
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("weights,scales", [(127, -116), (126, -115), (110, -100), (104, -100),
                                            (-95, 90)])
@pytest.mark.parametrize("rows,inner,out", [(3, 256, 64), (60, 1040, 512), (90, 272, 2080),
                                            (300, 400, 2000), (600, 144, 272), (2100, 272, 2048)])
def test_scales_of_8_bit_rows(rows, inner, out, weights, scales, group):
    """Weights up to the largest that fp32 holds, and far below 1, beside rows that make up
    for it: no kernel's way through the sums leaves the range of their result."""
    g = torch.Generator().manual_seed(rows + weights)
    q, _ = rows_of(g, rows, inner, torch.float32, "q8")
    x = q._replace(scales=q.scales * 2.0 ** scales)
    xv = qo.dequantize_q8(q).double() * 2.0 ** scales
    w, wv = device_weight(out, out, inner, group, scale=0.25 * 2.0 ** weights)
    assert wv.isfinite().all() and wv.abs().max() > 0.5 * 2.0 ** weights
    want, tol = product(xv, wv, group, True)
    near_on_device(qo.linear_w4(x, w, out_dtype=torch.float32), want, tol, torch.float32)
    w, wv = device_weight(out + 1, 2 * out, inner, group, gated=True, scale=0.25 * 2.0 ** weights)
    want, tol = silu_product(xv, wv, group, True)
    near_on_device(qo.gated_w4(x, w, out_dtype=torch.float32), want, tol, torch.float32)
    if out % 16 == 0:
        near_q8(qo.gated_w4(x, w, out_dtype=qo.Q8), want.cpu(), tol.cpu())


# ------------------------------------------------------------- any address --
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("fmt", [None, "w4", "w4a8"])
def test_checkpoint_tensors_at_any_address(fmt, dtype):
    """A model of device tensors that begin anywhere is the model of aligned ones."""
    cfg, weights = weights_of("synthetic")
    held = {k: torch.from_numpy(np.ascontiguousarray(w)).to(DEV, dtype) for k, w in weights.items()}

    def shifted(t):
        wide = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)
        wide[1:] = t.flatten()
        return wide[1:].view(t.shape)

    at_odd = {k: shifted(t) for k, t in held.items()}
    assert all(t.data_ptr() % 16 for t in at_odd.values())
    models = [backbone.QwenBackbone.from_weights(w, cfg, DEV, dtype, weight_format=fmt)
              for w in (held, at_odd)]
    for B, S in ((1, 1), (2, 40)):
        ids, mask = inputs(models[0], B, S, seed=S)
        want, got = (backbone.batch_backbone_states(m, ids, mask) for m in models)
        # where a table or norm is not aligned another kernel takes it, whose sums have
        # another order: as far apart as two paths of a model of the same values
        bar = BARS[fmt, dtype] if fmt else BARS["w4", dtype]
        assert normwise(got.cpu().numpy(), want.cpu().numpy()) <= bar
