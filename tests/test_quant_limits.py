"""The operators on 4-bit weights and 8-bit rows at the ends of their documented ranges: rows
far apart, the largest and smallest scales, quotients next to a half, tensors at any address."""
import importlib.machinery
import types

import numpy as np
import pytest
import torch

from conftest import normwise
from qdc_amd import _lib, backbone, quant_ops as qo
from test_quant_backbone import BARS, inputs, weights_of
from test_quant_ops import (DEV, GROUPS, blocks, feed_forward, near_on_device, near_q8,
                            plain_values, product, rows_of, silu_product)


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


# --------------------------------------------------- a program's own weights --
@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16", "q8"])
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("rows", [1, 40, 90, 300, 2100])
def test_weights_of_all_16_values(rows, group, kind):
    """A weight that a program has laid out itself, of -8 too, which packing never gives; its
    first outputs and rows are of the largest sums there are."""
    out, inner = 528, 272
    g = torch.Generator().manual_seed(rows + group)
    q = torch.randint(-8, 8, (out, inner), generator=g)
    q[:20] = -8
    s = (torch.rand(out, -(-inner // group), generator=g) * 0.02 + 0.01).bfloat16()
    packed, scales = (t.to(DEV) for t in blocks(q, s, group))
    w, wv = qo.W4(packed, scales, out, inner, group), plain_values(q, s, group).to(DEV)
    assert torch.equal(qo.unpack_w4(w).double(), wv)
    x, xv = rows_of(g, rows, inner, torch.bfloat16 if kind == "bf16" else torch.float32, kind)
    if kind == "q8":
        x.values[::3] = 127
        x.values[1::3, ::2] = -127
        xv = qo.dequantize_q8(x).double()
    want, tol = product(xv.to(DEV), wv, group, kind == "q8")
    for dtype in (torch.float32, torch.bfloat16):
        near_on_device(qo.linear_w4(x, w, out_dtype=dtype), want, tol, dtype)


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


# --------------------------------------------------- quotients next to a half --
def nearest_of(v, scale):
    """The nearest whole numbers of ``v / scale`` (fp32), ties to the even one, within -127..127:
    in 64 bits the product of a whole number and a half with a scale is exact, and so is what
    lies between it and v."""
    v, scale = v.double(), scale.double()
    q = (v / scale).round()
    for _ in range(2):
        left = 2 * (v - q * scale)
        over = (left.abs() > scale) | ((left.abs() == scale) & (q % 2 != 0))
        q = torch.where(over, q + left.sign(), q)
    return q.clamp(-127, 127)


def test_nearest_of():
    """The oracle itself, against fractions."""
    from fractions import Fraction
    g = torch.Generator().manual_seed(0)
    scale = torch.rand(40, generator=g) + 0.5
    half = torch.randint(-126, 126, (40,), generator=g) + 0.5
    exact = (half * scale).float()
    for v in (exact, torch.nextafter(exact, torch.tensor(9e9)),
              torch.nextafter(exact, torch.tensor(-9e9)), half * 0.5):
        s = torch.full((40,), 0.5) if v.equal(half * 0.5) else scale
        for a, b, q in zip(v.tolist(), s.tolist(), nearest_of(v, s).tolist()):
            assert q == round(Fraction(a) / Fraction(b))


@pytest.mark.gpu
@pytest.mark.parametrize("power", [0, -40, 110, -98, -110, -125, -135])
def test_8_bit_values_next_to_a_half(power):
    """Values on a half of their scale and as near to it as fp32 goes: the documented nearest
    whole number, of two the even one, for scales down to those that fp32 holds a few bits of."""
    rows = 600
    g = torch.Generator().manual_seed(power + 1000)
    most = (torch.rand(rows, generator=g) + 1) * 2.0 ** power
    most[:40] = 127 * 2.0 ** power           # scales of one bit: halves are exact
    scale = most / 127
    x = torch.zeros(rows, 256)
    half = torch.arange(126) + 0.5
    x[:, :126] = (half * scale[:, None].double()).float()
    x[:, 128:254] = torch.nextafter(x[:, :126], torch.tensor(float("inf")))
    x[rows // 2:, :126] = torch.nextafter(x[rows // 2:, :126], torch.tensor(0.0))
    x[:, 1:254:3] *= -1
    x[:, 126], x[:, 254] = most, -most
    x[:, :128] = torch.where(x[:, :128].abs() > most[:, None], 0.0, x[:, :128])
    x[:, 128:] = torch.where(x[:, 128:].abs() > most[:, None], 0.0, x[:, 128:])
    q = qo.quantize_q8(x.to(DEV))
    scales = q.scales.cpu()
    assert torch.equal(scales, scale[:, None].expand(rows, 2))
    wide = scales.repeat_interleave(128, 1)
    want = torch.where(wide > 0, nearest_of(x, wide), 0.0)
    assert torch.equal(q.values.cpu().double(), want)


# ----------------------------------------------------------- an earlier build --
def test_calls_of_an_earlier_build(monkeypatch):
    """A module built before the header existed has no version of it: refused with what to run."""
    class Earlier(importlib.machinery.ExtensionFileLoader):
        def create_module(self, spec):
            module = types.ModuleType("qdc_calls")
            module.version = _lib.lib().qdc_cache_version().decode()
            return module

        def exec_module(self, module):
            pass

    monkeypatch.setattr(importlib.machinery, "ExtensionFileLoader", Earlier)
    monkeypatch.setattr(_lib, "_calls", None)
    with pytest.raises(RuntimeError, match="csrc python"):
        _lib.calls()


# -------------------------------------------------------------------- refusals --
@pytest.mark.gpu
def test_a_flag_without_a_truth_value():
    """What is neither true nor false is refused with its own error, not with the call's end."""
    w = torch.zeros(32, 64, device=DEV)
    packed = qo.pack_w4(w)
    with pytest.raises(ValueError, match="truth value"):
        qo.pack_w4(w, gated=np.zeros(2))
    with pytest.raises(ValueError, match="truth value"):
        qo.unpack_w4(packed._replace(gated=np.zeros(2)))


# ------------------------------------------------------------ at the same time --
@pytest.mark.gpu
def test_graphs_side_by_side():
    """Two captured blocks and an eager one on three streams with nothing between them to wait
    for, all with 8-bit results that go through a workspace: every result is its own inputs'."""
    g = torch.Generator().manual_seed(11)
    up = qo.pack_w4((torch.randn(2 * 2048, 1024, generator=g) * 0.1).to(DEV), 64, gated=True)
    down = qo.pack_w4((torch.randn(1024, 2048, generator=g) * 0.1).to(DEV), 64)
    norm = torch.zeros(1024, device=DEV)
    sizes = (24, 40, 33)
    assert all(_lib.lib().qdc_linear_w4_workspace(n, 4096, 1024, 64, 1, _lib.QDC_Q8) > 0
               for n in sizes)
    streams = [torch.cuda.Stream() for _ in sizes]
    inputs_, outputs, replays = [], [], []
    for n, stream in zip(sizes, streams):
        x, a = (torch.randn(n, 1024, generator=g).to(DEV) for _ in range(2))
        inputs_.append((x, a))
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            feed_forward(x, a, norm, up, down)
        stream.synchronize()
        if len(replays) < 2:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outputs.append(feed_forward(x, a, norm, up, down))
            replays.append(graph)
    for turn in range(4):
        for x, _ in inputs_:
            x.copy_(torch.randn(x.shape, generator=g))
        want = [[t.clone() for t in feed_forward(x, a, norm, up, down)] for x, a in inputs_]
        torch.cuda.synchronize()
        eager = []
        for _ in range(10):
            for graph, stream in zip(replays, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
            with torch.cuda.stream(streams[2]):
                eager.append(feed_forward(*inputs_[2], norm, up, down))
        torch.cuda.synchronize()
        pairs = list(zip(outputs, want)) + [(e, want[2]) for e in eager]
        for got, right in pairs:
            assert torch.equal(got[0], right[0]) and torch.equal(got[1], right[1]), turn
