"""The operators on 4-bit weights and 8-bit rows (include/qdc_hip_quant.h,
qdc_amd.quant_ops): their argument checks, which need no GPU, and each against a plain
form in 64 bits, at the sizes and values where it can go wrong."""
import os
import re

import pytest
import torch

from conftest import ROOT
from qdc_amd import _lib, ops, quant_ops as qo

F32, BF16, X2, Q8 = _lib.QDC_F32, _lib.QDC_BF16, _lib.QDC_BF16X2, _lib.QDC_Q8
FAR = 1 << 56  # an aligned address never dereferenced by validation
DEV = "cuda:0"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}  # half a step, relative
GROUPS = [32, 64, 128]


# ---------------------------------------------------------- argument checks --
def test_exports_match_header():
    text = open(os.path.join(ROOT, "include", "qdc_hip_quant.h")).read()
    names = set(re.findall(r"^\s*(?:const\s+)?\w+\s*\*?\s*(qdc_\w+)\s*\(", text, re.M))
    assert names == set(_lib.QUANT_SIGNATURES)
    for name in names:
        assert hasattr(_lib.lib(), name), name
    version = re.search(r'#define\s+QDC_HIP_QUANT_VERSION\s+"([^"]+)"', text).group(1)
    assert _lib.lib().qdc_quant_version().decode() == version == _lib.calls().quant_version
    assert int(re.search(r"#define QDC_Q8 (\d)", text).group(1)) == Q8


def test_pack_validation():
    lib = _lib.lib()
    P, S, W = (FAR + (i << 40) for i in range(3))

    def pack(p=P, s=S, w=W, out=48, inner=256, ld=256, group=64, gated=0, dtype=BF16):
        return lib.qdc_pack_w4(p, s, w, out, inner, ld, group, gated, dtype, None)

    def unpack(p=P, s=S, w=W, out=48, inner=256, group=64, gated=0, dtype=BF16):
        return lib.qdc_unpack_w4(w, p, s, out, inner, group, gated, dtype, None)

    for f in (pack, unpack):
        assert f(dtype=X2) == -3 and f(dtype=Q8) == -3
        for bad in (dict(out=0), dict(out=1 << 24), dict(inner=0), dict(inner=252),
                    dict(inner=1 << 24), dict(group=16), dict(group=96), dict(group=256),
                    dict(out=47, gated=1), dict(out=1 << 20, inner=1 << 20)):
            assert f(**{**bad, **({"ld": 1 << 24} if f is pack else {})}) == -2, bad
        for n in "psw":
            assert f(**{n: None}) == -1 and f(**{n: FAR + (5 << 40) + 8}) == -2
    assert pack(ld=248) == -2 and pack(ld=260) == -2 and pack(ld=1 << 31) == -2
    # 3 x 2 blocks of 1024 bytes, 3 x 4 x 16 scales
    assert pack(w=P + 6 * 1024 - 16) == -5 and pack(s=P + 16) == -5 and pack(s=W + 32) == -5
    assert unpack(w=P + 16) == -5 and unpack(w=S + 16) == -5


def test_q8_validation():
    lib = _lib.lib()
    Q, S, X, R, A, N, M = (FAR + (i << 40) for i in range(7))

    def quant(q=Q, s=S, x=X, rows=3, width=256, ld=256, dtype=F32):
        return lib.qdc_quantize_q8(q, s, x, rows, width, ld, dtype, None)

    def back(q=Q, s=S, x=X, rows=3, width=256, dtype=F32):
        return lib.qdc_dequantize_q8(x, q, s, rows, width, dtype, None)

    def rms(q=Q, s=S, x=X, rows=3, width=256, dtype=F32, r=R, a=A, n=N, m=M):
        return lib.qdc_residual_rmsnorm_q8(r, q, s, x, a, n, m, rows, width, 1e-6, dtype, None)

    for f in (quant, back, rms):
        assert f(dtype=X2) == -3 and f(dtype=Q8) == -3
        for bad in (dict(rows=-1), dict(rows=1 << 26), dict(width=0), dict(width=264),
                    dict(width=1 << 24), dict(rows=1 << 20, width=1 << 16)):
            assert f(**{**bad, **({"ld": 1 << 24} if f is quant else {})}) == -2, bad
        for n in "qsx":
            assert f(**{n: None}) == -1, n
        assert f(q=FAR + (9 << 40) + 4) == -2 and f(s=FAR + (9 << 40) + 2) == -2
        assert f(rows=0, q=None, s=None, x=None) == 0
    assert quant(ld=248) == -2 and quant(ld=260) == -2
    assert quant(x=Q + 16) == -5 and quant(s=Q + 764) == -5 and back(x=S + 16) == -5
    assert rms(width=32784) == -2 and rms(n=None) == -1 and rms(r=None) == -1
    assert rms(m=M + 2) == -2 and rms(a=A + 8) == -2 and rms(r=X + 16) == -5
    assert rms(r=A) == -5 and rms(q=R + 16) == -5 and rms(s=N + 16) == -5 and rms(q=X) == -5


def test_linear_validation():
    lib = _lib.lib()
    Y, YS, X, XS, P, S = (FAR + (i << 40) for i in range(6))

    def f(y=Y, ys=YS, x=X, xs=XS, p=P, s=S, yt=BF16, xt=BF16, rows=3, out=96, inner=256, group=64,
          ld=256, gated=0, ws=FAR + (6 << 40), nbytes=3 * 48 * 4):
        return lib.qdc_linear_w4(y, ys, yt, x, xs, xt, p, s, rows, out, inner, group, ld, gated, ws,
                                 nbytes, None)

    size = lib.qdc_linear_w4_workspace
    assert size(3, 96, 256, 64, 1, Q8) == 3 * 48 * 4
    assert size(3, 96, 256, 64, 1, BF16) == 0 and size(3, 96, 256, 64, 0, F32) == 0
    assert size(9000, 7168, 1024, 64, 1, Q8) == 0 and size(0, 96, 256, 64, 1, Q8) == 0
    assert size(-1, 96, 256, 64, 1, Q8) == -1 and size(3, 80, 256, 64, 1, Q8) == -1
    assert size(3, 96, 256, 64, 0, Q8) == -1 and size(3, 96, 252, 64, 1, Q8) == -1
    for bad in (dict(nbytes=3 * 48 * 4 - 1), dict(ws=FAR + (6 << 40) + 8)):
        assert f(yt=Q8, gated=1, **bad) == -2
    assert f(yt=Q8, gated=1, ws=None) == -1 and f(yt=Q8, gated=1, ws=X) == -5
    assert f(yt=Q8, gated=1, ws=Y + 64) == -5

    assert f(xt=X2) == -3 and f(yt=X2) == -3 and f(yt=Q8) == -3 and f(xt=7) == -3
    for bad in (dict(rows=-1), dict(rows=(1 << 20) - 15), dict(out=0), dict(inner=252),
                dict(group=48), dict(ld=248), dict(ld=260), dict(out=95, gated=1),
                dict(out=2 * 40, gated=1, yt=Q8), dict(xt=Q8, inner=248, ld=248),
                dict(xt=Q8, ld=272), dict(ld=(1 << 25) + 8), dict(xt=F32, ld=(1 << 24) + 8)):
        assert f(**bad) == -2, bad
    for n in ("y", "x", "p", "s"):
        assert f(**{n: None}) == -1 and f(**{n: FAR + (9 << 40) + 8}) == -2, n
    assert f(xt=Q8, xs=None) == -1 and f(yt=Q8, gated=1, ys=None) == -1
    assert f(xt=Q8, xs=XS + 2) == -2
    assert f(y=X + 16) == -5 and f(y=P + 32) == -5 and f(y=S + 32) == -5
    assert f(xt=Q8, y=XS) == -5 and f(yt=Q8, gated=1, ys=Y + 16) == -5
    assert f(rows=0, y=None, x=None) == 0


def test_calls_refuse():
    cpu = torch.zeros(4, 64)
    with pytest.raises(ValueError):
        qo.pack_w4(cpu)
    with pytest.raises(ValueError):
        qo.quantize_q8(cpu)
    with pytest.raises(ValueError):
        qo.residual_rms_q8(cpu, None, torch.zeros(64), 1e-6)
    with pytest.raises(TypeError):
        qo.pack_w4(None)
    w = qo.W4(torch.zeros(1, 1, 64, 4, dtype=torch.int32),
              torch.zeros(1, 2, 16, dtype=torch.bfloat16), 16, 64, 64)
    with pytest.raises(ValueError):
        qo.linear_w4(cpu, w)
    with pytest.raises(ValueError):
        qo.gated_w4(cpu, w)                       # not a gated weight
    with pytest.raises(ValueError):
        qo.linear_w4(cpu, w._replace(gated=True))
    with pytest.raises(ValueError):
        qo.linear_w4(cpu, w, out_dtype=torch.float16)
    for first, last in ((0, 8), (8, 16), (16, 16), (0, 32)):
        with pytest.raises(ValueError):
            w.outputs(first, last)
    with pytest.raises(ValueError):
        w._replace(gated=True).outputs(0, 16)


# -------------------------------------------------------------- plain forms --
def plain_pack(w, group):
    """Whole numbers and scales of ``w [out, inner]`` (CPU), in 64 bits."""
    out, inner = w.shape
    v = torch.nn.functional.pad(w.double(), (0, -inner % group)).view(out, -1, group)
    s = (v.abs().amax(-1, keepdim=True).float() / 7).bfloat16().double()
    q = torch.where(s > 0, v / s, 0.0).round().clamp(-7, 7)
    bad = ~v.isfinite().all(-1, keepdim=True)
    return torch.where(bad, 0.0, q).flatten(1)[:, :inner], torch.where(bad, torch.nan, s)[..., 0]


def plain_values(q, s, group):
    return q.double() * s.double().repeat_interleave(group, 1)[:, :q.shape[1]]


def blocks(q, s, group):
    """The documented layout, place by place (CPU)."""
    out, inner = q.shape
    nb, kb = -(-out // 16), -(-inner // 128)
    packed = torch.zeros(nb, kb, 64, 4, dtype=torch.int64)
    full = torch.zeros(nb * 16, kb * 128, dtype=torch.int64)
    full[:out, :inner] = q.long() & 15
    lane, t = torch.arange(64), torch.arange(4)
    for b in range(nb):
        for c in range(kb):
            for i in range(8):
                k = 128 * c + 32 * t[None] + 8 * (lane[:, None] // 16) + i
                shift = 8 * i if i < 4 else 8 * (i - 4) + 4
                packed[b, c] |= full[16 * b + lane[:, None] % 16, k] << shift
    packed = torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).int()
    sc = torch.zeros(nb * 16, kb * 128 // group, dtype=torch.bfloat16)
    sc[:out, :s.shape[1]] = s.bfloat16()
    return packed, sc.view(nb, 16, -1).transpose(1, 2).contiguous()


def plain_q8(v):
    """Values and scales that 8 bits hold of ``v`` (64 bits)."""
    rows, width = v.shape
    p = torch.nn.functional.pad(v, (0, -width % 128)).view(rows, -1, 128)
    a = p.abs().amax(-1) / 127
    q = torch.where(a[..., None] > 0, p / a[..., None], 0.0).round()
    return (q * a[..., None]).flatten(1)[:, :width], a


def rows_of(g, rows, width, dtype, kind="f32"):
    """Rows on the device with NaN between them, and their 64-bit values; 8-bit ones whole."""
    if kind == "q8":
        q = torch.randint(-127, 128, (rows, width), generator=g).to(torch.int8)
        a = torch.rand(rows, -(-width // 128), generator=g) * 0.05
        return qo.Q8(q.to(DEV), a.to(DEV)), plain_values(q, a, 128)
    x = torch.randn(rows, width, generator=g).to(dtype)
    x[:, width // 3] *= 20
    held = torch.full((rows, width + 24), float("nan"), dtype=dtype)
    held[:, 16:16 + width] = x
    return held.to(DEV)[:, 16:16 + width], x.double()


def weight_of(g, out, inner, group, gated=False):
    """A weight on the device and its 64-bit values ``[out, inner]``."""
    w = torch.randn(out, inner, generator=g) * 0.1
    w[:, inner // 2] *= 5
    packed = qo.pack_w4(w.to(DEV), group, gated)
    return packed, plain_values(*plain_pack(w, group), group)


def product(x, w, group, whole):
    """``x w^T`` in 64 bits, and how far a product of fp32 sums may be from it: within a
    group (none for whole numbers) and over the groups and the wavefronts' parts every
    addition is off by a step at most, as is each scaling."""
    adds = x.shape[1] // group + 20 + (0 if whole else group)
    return x @ w.t(), adds * 2.0 ** -23 * (x.abs() @ w.abs().t())


def silu_product(x, w, group, whole):
    y, e = product(x, w, group, whole)
    (g, u), (eg, eu) = y.chunk(2, 1), e.chunk(2, 1)
    act = g * torch.sigmoid(g) * u
    # the slope of silu is at most 1.1; exp and its argument are off by |g| steps and a few
    return act, 1.1 * eg * (u.abs() + eu) + (g * torch.sigmoid(g)).abs() * eu + \
        (g.abs() + 10) * 2.0 ** -23 * act.abs() + 1e-37


def near(got, want, tol, dtype):
    got = got.double().cpu()
    over = (got - want).abs() - tol - HALF[dtype] * (want.abs() + tol)
    assert got.shape == want.shape and not got.isnan().any()
    assert over.max() <= 0, (float(over.max()), float((got - want).abs().max()))


def near_q8(q, want, tol):
    """8-bit rows of values that are themselves off by ``tol``."""
    got = qo.dequantize_q8(q).double().cpu()
    _, a = plain_q8(want)
    pad = torch.nn.functional.pad(tol, (0, -tol.shape[1] % 128)).view(*a.shape, 128).amax(-1)
    assert ((q.scales.double().cpu() - a).abs() <= pad / 127 + 2.0 ** -23 * a).all()
    step = q.scales.double().cpu().repeat_interleave(128, 1)[:, :want.shape[1]]
    # half a step, the product with the inverse off by two roundings of up to 127
    assert ((got - want).abs() <= 0.5 * step * (1 + 2.0 ** -14) + tol + 2.0 ** -24 * got.abs()).all()


# ------------------------------------------------------------------ packing --
@pytest.mark.gpu
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("out,inner", [(16, 128), (1, 8), (37, 200), (130, 1000)])
def test_pack(out, inner, dtype, group):
    g = torch.Generator().manual_seed(out + inner + group)
    w = (torch.randn(out, inner, generator=g) * 0.05).to(dtype)
    w[0, :7] = torch.tensor([7, 0.5, -0.5, 1.5, 2.5, -3.5, 6.5]) * 0.25   # ties
    w[0, 7:] = 0
    w[out // 2, : inner // 2] = 0                                         # groups of zeros
    held = torch.full((out, inner + 16), float("nan"), dtype=dtype)
    held[:, 8:8 + inner] = w
    q, s = plain_pack(w, group)
    got = qo.pack_w4(held.to(DEV)[:, 8:8 + inner], group)
    packed, scales = blocks(q, s, group)
    assert torch.equal(got.packed.cpu(), packed)
    assert torch.equal(got.scales.cpu(), scales)
    back = qo.unpack_w4(got)
    assert torch.equal(back.double().cpu(), plain_values(q, s, group))
    assert torch.equal(qo.unpack_w4(got, torch.bfloat16), back.bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("out,inner", [(16, 128), (2, 8), (74, 200)])
def test_pack_gated(out, inner):
    g = torch.Generator().manual_seed(out)
    w = torch.randn(out, inner, generator=g).to(DEV)
    got = qo.pack_w4(w, 64, gated=True)
    halves = [qo.pack_w4(h.contiguous(), 64) for h in w.chunk(2)]
    for name in ("packed", "scales"):
        both = torch.stack([getattr(h, name) for h in halves], 1).flatten(0, 1)
        assert torch.equal(getattr(got, name), both)
    assert torch.equal(qo.unpack_w4(got), torch.cat([qo.unpack_w4(h) for h in halves]))


@pytest.mark.gpu
def test_pack_values_at_the_edge():
    """Infinities and NaN in one group, values whose scale vanishes or is the largest, and
    quotients a hair beside a half."""
    w = torch.zeros(6, 128)
    w[0] = torch.linspace(-1, 1, 128)
    w[0, 5] = float("inf")
    w[1, 70] = float("nan")
    w[2] = 1e-45
    w[3, ::2] = 3.4e38
    w[4, :64] = torch.tensor([0.4999999, 0.5, 0.50000006, 1.4999999, 1.5, 1.5000001, -2.5, -2.5000002] * 8)
    w[4, 63] = 7
    w[5] = torch.randn(128, generator=torch.Generator().manual_seed(1)) * 1e-38
    q, s = plain_pack(w, 64)
    got = qo.pack_w4(w.to(DEV), 64)
    packed, scales = blocks(q, s, 64)
    assert torch.equal(got.packed.cpu(), packed)
    assert torch.equal(got.scales.isnan().cpu(), scales.isnan())
    assert torch.equal(got.scales.nan_to_num().cpu(), scales.nan_to_num())


# ---------------------------------------------------------------- 8-bit rows --
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,width", [(1, 16), (3, 128), (5, 1040), (300, 272), (0, 64)])
def test_quantize(rows, width, dtype):
    g = torch.Generator().manual_seed(rows + width)
    x, v = rows_of(g, rows, width, dtype) if rows else (torch.zeros(0, width, device=DEV),
                                                        torch.zeros(0, width).double())
    q = qo.quantize_q8(x)
    assert q.values.shape == (rows, width) and q.scales.shape == (rows, -(-width // 128))
    if rows:
        near_q8(q, v, torch.zeros_like(v))
    assert torch.equal(qo.dequantize_q8(q, torch.bfloat16), qo.dequantize_q8(q).bfloat16())


@pytest.mark.gpu
def test_quantize_values_at_the_edge():
    x = torch.zeros(6, 256)
    x[0, 3], x[0, 200] = float("inf"), 1.0
    x[1, 3], x[1, 200] = float("nan"), -2.0
    x[2] = 3.4e38
    x[3, :5] = torch.tensor([1e-45, -1e-45, 0, 0, 0])
    x[4] = torch.linspace(-1e-38, 1e-38, 256)
    x[5, 128:] = torch.linspace(-1e-33, 1e-33, 128)
    q = qo.quantize_q8(x.to(DEV))
    back = qo.dequantize_q8(q).cpu()
    assert back[:2, :128].isnan().all() and (back[0, 128:] == x[0, 128:]).all()
    assert back[1, 200] == -2.0
    assert q.values[2].eq(127).all() and (back[2] - x[2]).abs().max() <= 2.0 ** -22 * 3.4e38
    assert (back[3] == 0).all()        # a scale of 1e-45 / 127 is none
    # denormal scales hold what they can: half a step of theirs
    for r in (4, 5):
        step = q.scales[r].cpu().repeat_interleave(128).double()
        off = (back[r].double() - x[r].double()).abs()
        assert (off <= 0.5001 * step + 127 * 2.0 ** -149).all()
    assert (q.scales[5, 0] == 0) and (back[5, :128] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,width", [(1, 16), (1, 1024), (7, 256), (300, 1024), (5, 2064),
                                        (260, 768), (300, 2048), (3, 4096), (2, 8208), (3, 5120),
                                        (1, 32768)])
@pytest.mark.parametrize("add,masked", [(True, True), (False, False), (True, False)])
def test_residual_rms(rows, width, add, masked, dtype):
    g = torch.Generator().manual_seed(rows * width)
    x, a = torch.randn(rows, width, generator=g), torch.randn(rows, width, generator=g)
    w = (torch.randn(width, generator=g) * 0.2).to(dtype)
    mask = torch.randint(0, 2, (rows,), generator=g).int() if masked else None
    if masked:
        x[mask == 0, 0] = float("nan")     # what is masked is not looked at
    residual, q = qo.residual_rms_q8(x.to(DEV), a.to(DEV) if add else None, w.to(DEV), 1e-6,
                                     None if mask is None else mask.to(DEV))
    want = x + a if add else x
    assert torch.equal(residual.cpu().nan_to_num(7e7), want.nan_to_num(7e7))
    y = want.double()
    y = y * torch.rsqrt(y.square().mean(1, keepdim=True) + 1e-6) * (1 + w.double())
    if masked:
        y = torch.where(mask[:, None] != 0, y, 0.0)
        assert (q.values.cpu()[mask == 0] == 0).all() and (q.scales.cpu()[mask == 0] == 0).all()
    # the sum of squares: a lane's chain of at most 32 values, then a tree; then a root, a
    # reciprocal, three products and a sum
    near_q8(q, y, (32 + 10 + 10) * 2.0 ** -24 * y.abs())


@pytest.mark.gpu
def test_residual_rms_in_place_of_x():
    x = torch.randn(4, 256, device=DEV)
    residual, _ = qo.residual_rms_q8(x, None, torch.zeros(256, device=DEV), 1e-6)
    assert residual.data_ptr() == x.data_ptr()
    a, w = torch.randn(4, 256, device=DEV), torch.zeros(256, device=DEV)
    want, q = qo.residual_rms_q8(x, a, w, 1e-6)
    v, s = torch.empty_like(q.values), torch.empty_like(q.scales)
    status = _lib.lib().qdc_residual_rmsnorm_q8(
        x.data_ptr(), v.data_ptr(), s.data_ptr(), x.data_ptr(), a.data_ptr(), w.data_ptr(), None, 4,
        256, 1e-6, F32, torch.cuda.current_stream().cuda_stream)
    assert status == 0 and torch.equal(x, want) and torch.equal(v, q.values)


# ----------------------------------------------------------------- products --
SHAPES = [(1, 128, 16), (1, 256, 768), (3, 1040, 37), (16, 1024, 130), (17, 528, 64),
          (40, 2048, 50), (65, 336, 300), (300, 272, 513), (600, 400, 264)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16", "q8"])
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("rows,inner,out", SHAPES)
def test_linear(rows, inner, out, group, kind):
    g = torch.Generator().manual_seed(rows + inner + out + group)
    x, xv = rows_of(g, rows, inner, torch.bfloat16 if kind == "bf16" else torch.float32, kind)
    w, wv = weight_of(g, out, inner, group)
    want, tol = product(xv, wv, group, kind == "q8")
    for dtype in (torch.float32, torch.bfloat16):
        near(qo.linear_w4(x, w, out_dtype=dtype), want, tol, dtype)
    default = qo.linear_w4(x, w)
    assert default.dtype == {"f32": torch.float32}.get(kind, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16", "q8"])
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("rows,inner,inter", [(1, 128, 16), (1, 1024, 304), (5, 272, 37),
                                              (16, 256, 128), (33, 512, 144), (70, 208, 1),
                                              (150, 640, 272), (700, 144, 160), (40, 1200, 272),
                                              (17, 128, 1040)])
def test_gated(rows, inner, inter, group, kind):
    g = torch.Generator().manual_seed(rows + inner + inter + group)
    x, xv = rows_of(g, rows, inner, torch.bfloat16 if kind == "bf16" else torch.float32, kind)
    w, wv = weight_of(g, 2 * inter, inner, group, gated=True)
    want, tol = silu_product(xv, wv, group, kind == "q8")
    for dtype in (torch.float32, torch.bfloat16):
        near(qo.gated_w4(x, w, out_dtype=dtype), want, tol, dtype)
    if inter % 16 == 0:
        near_q8(qo.gated_w4(x, w, out_dtype=qo.Q8), want, tol)


# Row and output counts at which the next larger tile is taken, the last two with several
# tiles a workgroup; of 2 and 3 blocks of inputs, the last not whole.
MANY = [(300, 2000, 272), (520, 2056, 144), (1030, 2056, 272), (2050, 2051, 144),
        (4100, 2056, 272), (8200, 4104, 144)]


def on_device(*tensors):
    return [t.to(DEV) for t in tensors]


def near_on_device(got, want, tol, dtype):
    over = (got.double() - want).abs() - tol - HALF[dtype] * (want.abs() + tol)
    assert got.shape == want.shape and not got.isnan().any() and float(over.max()) <= 0


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16", "q8"])
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("rows,out,inner", MANY)
def test_linear_many(rows, out, inner, group, kind):
    g = torch.Generator().manual_seed(rows + out + group)
    x, xv = rows_of(g, rows, inner, torch.bfloat16 if kind == "bf16" else torch.float32, kind)
    w, wv = weight_of(g, out, inner, group)
    want, tol = product(*on_device(xv, wv), group, kind == "q8")
    for dtype in (torch.float32, torch.bfloat16):
        near_on_device(qo.linear_w4(x, w, out_dtype=dtype), want, tol, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16", "q8"])
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("rows,out,inner", MANY)
def test_gated_many(rows, out, inner, group, kind):
    inter = out // 2 if out % 2 else out // 2 // 16 * 16 - 16 * (rows % 3)
    g = torch.Generator().manual_seed(rows + out + group + 1)
    x, xv = rows_of(g, rows, inner, torch.bfloat16 if kind == "bf16" else torch.float32, kind)
    w, wv = weight_of(g, 2 * inter, inner, group, gated=True)
    want, tol = silu_product(*on_device(xv, wv), group, kind == "q8")
    for dtype in (torch.float32, torch.bfloat16):
        near_on_device(qo.gated_w4(x, w, out_dtype=dtype), want, tol, dtype)
    if inter % 16 == 0:
        near_q8(qo.gated_w4(x, w, out_dtype=qo.Q8), want.cpu(), tol.cpu())


# Between few rows and many, on both sides of where the next kernel is taken: of 2 to 18 blocks
# of inputs, with the last block of outputs and of inputs not whole.
BETWEEN = [(24, 5098, 400), (48, 4090, 272), (48, 7030, 272), (47, 7030, 1040), (41, 7030, 2192),
           (90, 2050, 2192), (128, 7190, 144), (200, 7190, 144), (33, 7190, 656)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16", "q8"])
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("rows,out,inner", BETWEEN)
def test_between_few_and_many(rows, out, inner, group, kind):
    g = torch.Generator().manual_seed(rows + out + inner + group)
    x, xv = rows_of(g, rows, inner, torch.bfloat16 if kind == "bf16" else torch.float32, kind)
    w, wv = weight_of(g, out, inner, group)
    want, tol = product(*on_device(xv, wv), group, kind == "q8")
    gated, gv = weight_of(g, out, inner, group, gated=True)
    both, both_tol = silu_product(*on_device(xv, gv), group, kind == "q8")
    for dtype in (torch.float32, torch.bfloat16):
        near_on_device(qo.linear_w4(x, w, out_dtype=dtype), want, tol, dtype)
        near_on_device(qo.gated_w4(x, gated, out_dtype=dtype), both, both_tol, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16", "q8"])
@pytest.mark.parametrize("rows,out,inner", [(9000, 1, 272), (9000, 30, 144), (4200, 60, 272),
                                            (9000, 100, 144)])
def test_few_outputs_of_many_rows(rows, out, inner, kind):
    g = torch.Generator().manual_seed(out)
    x, xv = rows_of(g, rows, inner, torch.bfloat16 if kind == "bf16" else torch.float32, kind)
    w, wv = weight_of(g, out, inner, 64)
    near_on_device(qo.linear_w4(x, w, out_dtype=torch.float32),
                   *product(*on_device(xv, wv), 64, kind == "q8"), torch.float32)
    if out > 1:
        up, upv = weight_of(g, out, inner, 32, gated=True)
        near_on_device(qo.gated_w4(x, up, out_dtype=torch.float32),
                       *silu_product(*on_device(xv, upv), 32, kind == "q8"), torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,out", [(1, 768), (40, 4096), (300, 2000), (1030, 2056), (4100, 2056)])
def test_nothing_behind_the_result(rows, out):
    """Rows behind the last, and the gap behind the last output, are left as they were."""
    g = torch.Generator().manual_seed(out)
    w, _ = weight_of(g, out, 136, 64)
    x = torch.randn(rows, 136, generator=g).bfloat16().to(DEV)
    want = qo.linear_w4(x, w)
    held = torch.full((rows + 70, out), 7.0, dtype=torch.bfloat16, device=DEV)
    status = _lib.lib().qdc_linear_w4(
        held.data_ptr(), None, BF16, x.data_ptr(), None, BF16, w.packed.data_ptr(),
        w.scales.data_ptr(), rows, out, 136, 64, 136, 0, None, 0,
        torch.cuda.current_stream().cuda_stream)
    assert status == 0 and torch.equal(held[:rows], want) and (held[rows:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("inner", [8, 24, 120, 136, 264])
@pytest.mark.parametrize("rows", [2, 80])
def test_linear_short_inner(inner, rows):
    """Inner sizes that end inside a block, for rows that are not whole groups either."""
    g = torch.Generator().manual_seed(inner)
    for dtype in (torch.float32, torch.bfloat16):
        x, xv = rows_of(g, rows, inner, dtype)
        w, wv = weight_of(g, 20, inner, 32)
        near(qo.linear_w4(x, w, out_dtype=torch.float32), *product(xv, wv, 32, False),
             torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("inner", [256, 200])
@pytest.mark.parametrize("rows,out", [(1, 48), (20, 48), (100, 48), (600, 48), (300, 2000),
                                      (2050, 2056)])
def test_linear_values_at_the_edge(rows, out, inner):
    """fp32 rows keep all 24 bits; an infinity or NaN reaches its own row alone, a NaN scale
    its own output alone; large values stay finite."""
    g = torch.Generator().manual_seed(3)
    w, wv = weight_of(g, out, inner, 64)
    x = torch.randn(rows, inner, generator=g) * torch.exp(torch.randn(rows, inner, generator=g) * 8)
    want, tol = product(x.double(), wv, 64, False)
    near(qo.linear_w4(x.to(DEV), w), want, tol, torch.float32)
    big = x.clone()
    big[0] = 2.0 ** 100
    assert qo.linear_w4(big.to(DEV), w).isfinite().all()
    for dtype in (torch.float32, torch.bfloat16):
        bad = x.clone()
        bad[0, 7] = float("nan")
        got = qo.linear_w4(bad.to(dtype).to(DEV), w)
        assert got[0].isnan().all() and got[1:].isfinite().all()
        bad[0, 7] = float("inf")
        got = qo.linear_w4(bad.to(dtype).to(DEV), w).cpu()
        q = wv[:, 7]
        assert (got[0][q > 0] == float("inf")).all() and (got[0][q < 0] == -float("inf")).all()
        assert got[0][q == 0].isnan().all() and got[1:].isfinite().all()
    # a NaN whose bits all lie in the half that a bf16 term drops
    bad[0, 7] = torch.tensor([0x7f800001], dtype=torch.int32).view(torch.float32)
    assert qo.linear_w4(bad.to(DEV), w)[0].isnan().all()
    w.scales[1, 0, 5] = float("nan")
    got = qo.linear_w4(x.to(DEV), w)
    assert got[:, 21].isnan().all() and got.isnan().sum() == rows


@pytest.mark.gpu
def test_rows_do_not_depend_on_their_neighbours():
    """Within a call of one kernel a row's result is its own, whatever lies beside it."""
    g = torch.Generator().manual_seed(5)
    w, _ = weight_of(g, 64, 512, 64)
    for n in (16, 64, 400, 1000, 9000):
        x = torch.randn(n, 512, generator=g).to(DEV)
        y = qo.linear_w4(x, w)
        order = torch.randperm(n, generator=g).to(DEV)
        assert torch.equal(qo.linear_w4(x[order], w), y[order])
        assert torch.equal(qo.linear_w4(x, w), y)


@pytest.mark.gpu
def test_outputs_of_a_weight():
    g = torch.Generator().manual_seed(6)
    w, _ = weight_of(g, 100, 256, 32)
    x = torch.randn(9, 256, generator=g).to(DEV)
    y = qo.linear_w4(x, w)
    assert torch.equal(qo.linear_w4(x, w.outputs(16, 64)), y[:, 16:64])
    assert torch.equal(qo.linear_w4(x, w.outputs(96, 100)), y[:, 96:])


@pytest.mark.gpu
def test_no_rows():
    w = qo.pack_w4(torch.randn(32, 64, device=DEV))
    assert qo.linear_w4(torch.zeros(0, 64, device=DEV), w).shape == (0, 32)
    assert qo.linear_w4(qo.quantize_q8(torch.zeros(0, 64, device=DEV)), w).shape == (0, 32)
    up = qo.pack_w4(torch.randn(32, 64, device=DEV), gated=True)
    assert qo.gated_w4(torch.zeros(0, 64, device=DEV), up, out_dtype=qo.Q8).values.shape == (0, 16)
    r, q = qo.residual_rms_q8(torch.zeros(0, 64, device=DEV), None, torch.zeros(64, device=DEV), 0.1)
    assert r.shape == (0, 64) and q.scales.shape == (0, 1)


@pytest.mark.gpu
def test_refusals_on_the_device():
    dev = dict(device=DEV)
    w = qo.pack_w4(torch.randn(32, 64, **dev))
    up = qo.pack_w4(torch.randn(80, 64, **dev), gated=True)
    x = torch.zeros(4, 64, **dev)
    bad = [lambda: qo.pack_w4(torch.zeros(32, 60, **dev)),
           lambda: qo.pack_w4(torch.zeros(32, 64, **dev), group=16),
           lambda: qo.pack_w4(torch.zeros(31, 64, **dev), gated=True),
           lambda: qo.pack_w4(torch.zeros(32, 64, **dev).half()),
           lambda: qo.pack_w4(torch.zeros(0, 64, **dev)),
           lambda: qo.unpack_w4(w, torch.float16),
           lambda: qo.unpack_w4(w._replace(out=64)),
           lambda: qo.unpack_w4(w._replace(group=32)),
           lambda: qo.unpack_w4(w._replace(scales=w.scales.float())),
           lambda: qo.linear_w4(x[:, :56], w),
           lambda: qo.linear_w4(x.t(), w),
           lambda: qo.linear_w4(x.half(), w),
           lambda: qo.linear_w4(x.cpu(), w),
           lambda: qo.linear_w4(torch.zeros(4 * 68, **dev).view(4, 68)[:, 4:], w),  # stride, start
           lambda: qo.linear_w4(x[:1].expand(4, 64), w),
           lambda: qo.linear_w4(x, w, out_dtype=qo.Q8),
           lambda: qo.linear_w4(qo.Q8(x.to(torch.int8), torch.zeros(4, 2, **dev)), w),
           lambda: qo.gated_w4(x, w),
           lambda: qo.gated_w4(x, up, out_dtype=qo.Q8),                    # 40 columns
           lambda: qo.quantize_q8(torch.zeros(4, 40, **dev)),
           lambda: qo.dequantize_q8(qo.quantize_q8(x), torch.int8),
           lambda: qo.residual_rms_q8(x.bfloat16(), None, x[0], 1e-6),
           lambda: qo.residual_rms_q8(x, x[:2], x[0], 1e-6),
           lambda: qo.residual_rms_q8(x, None, x[0, :32], 1e-6),
           lambda: qo.residual_rms_q8(x, None, x[0], 1e-6, torch.ones(3, **dev).int()),
           lambda: qo.residual_rms_q8(x, None, x[0], 1e-6, torch.ones(4, **dev))]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


# --------------------------------------------------------- used as they are --
def feed_forward(x, add, norm, up, down, mask=None):
    residual, rows = qo.residual_rms_q8(x, add, norm, 1e-6, mask)
    act = qo.gated_w4(rows, up, out_dtype=qo.Q8)
    return residual, qo.linear_w4(act, down, out_dtype=torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 30, 200, 1100])
def test_feed_forward_block(rows):
    """Norm, gated product and down projection together: each against 64 bits on what the
    one before it gave."""
    g = torch.Generator().manual_seed(rows)
    x, a = torch.randn(rows, 256, generator=g), torch.randn(rows, 256, generator=g)
    norm = torch.randn(256, generator=g) * 0.1
    up, upv = weight_of(g, 2 * 512, 256, 64, gated=True)
    down, downv = weight_of(g, 256, 512, 64)
    residual, y = feed_forward(x.to(DEV), a.to(DEV), norm.to(DEV), up, down)
    _, q = qo.residual_rms_q8(x.to(DEV), a.to(DEV), norm.to(DEV), 1e-6)
    act = qo.gated_w4(q, up, out_dtype=qo.Q8)
    want, tol = silu_product(qo.dequantize_q8(q).double().cpu(), upv, 64, True)
    near_q8(act, want, tol)
    near(y, *product(qo.dequantize_q8(act).double().cpu(), downv, 64, True), torch.float32)


@pytest.mark.gpu
def test_captured_on_another_stream():
    """Two captured graphs of one weight, replayed in turn on streams of their own with eager
    calls in between: every replay is the eager result of its own inputs."""
    g = torch.Generator().manual_seed(9)
    up, _ = weight_of(g, 2 * 256, 256, 64, gated=True)
    down, _ = weight_of(g, 256, 256, 64)
    norm = torch.zeros(256, device=DEV)
    sets = []
    for n in (1, 90):
        x, a = (torch.randn(n, 256, generator=g).to(DEV) for _ in range(2))
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            feed_forward(x, a, norm, up, down)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = feed_forward(x, a, norm, up, down)
        sets.append((x, a, stream, graph, out))
    for turn in range(3):
        for x, a, stream, graph, out in sets:
            x.copy_(torch.randn(x.shape, generator=g))
            want = feed_forward(x, a, norm, up, down)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                graph.replay()
            stream.synchronize()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
