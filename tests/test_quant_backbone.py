"""Backbones whose projections are held in 4 bits, with rows in 8 bits or not: the forward
against a model that holds the same values in fp32, and a cache's steps, recorded graphs and
last-token calls against that forward."""
import numpy as np
import pytest
import torch

from conftest import normwise

FORMATS = ["w4", "w4a8"]
DTYPES = [torch.float32, torch.bfloat16]
# Both fp32 paths hold 1e-5 of the exact forward, and bf16 storage 1e-2, so twice that
# between two.  8-bit rows: fp32 sums in another order move a value over a rounding border
# once in some 10^4 values, by a step, 1/50 of the rows' size, so by 2e-4 of a row at each of
# up to 3 roundings a layer, and a layer passes on no more than a few times what it is given.
BARS = {("w4", torch.float32): 2e-5, ("w4", torch.bfloat16): 2e-2,
        ("w4a8", torch.float32): 1e-2, ("w4a8", torch.bfloat16): 2e-2}


def weights_of(config, seed=5):
    from oracle import qdc_oracle as O
    from qdc_amd import config as C
    from qdc_amd.weights import random_weights
    cfg = {"synthetic": C.synthetic_inference_config, "plumbing": C.plumbing_config}[config]()
    return cfg, {k: O.round_bf16(v) for k, v in random_weights(cfg, seed=seed).items()}


def model_of(fmt, dtype, config="synthetic", group=64):
    from qdc_amd import backbone
    cfg, weights = weights_of(config)
    return backbone.QwenBackbone.from_weights(weights, cfg, "cuda:0", dtype, weight_format=fmt,
                                              weight_group=group)


def plain_model(fmt, config="synthetic", group=64):
    """The same values in fp32, multiplied by the library, 8-bit rows as what they stand for."""
    from qdc_amd import backbone, quant_ops as qo
    cfg, weights = weights_of(config)
    for name, w in weights.items():
        if name.endswith("_proj.weight") or "in_proj" in name:
            t = torch.from_numpy(np.ascontiguousarray(w)).cuda()
            weights[name] = qo.unpack_w4(qo.pack_w4(t, group)).cpu().numpy()

    class Plain(backbone.QwenBackbone):
        def _held(self, x):
            return qo.dequantize_q8(qo.quantize_q8(x.contiguous())) if fmt == "w4a8" else x

        def _first_rows(self, h, normed, token_mask):
            return self._held(normed)

        def _add_norm(self, h, mixed, norm, token_mask=None, out_dtype=None):
            h, normed = super()._add_norm(h, mixed, norm, token_mask, out_dtype)
            return h, normed if norm is self.final_norm else self._held(normed)

        def _activate(self, normed, w):
            return self._held(super()._activate(normed, w))

    model = Plain.from_weights(weights, cfg, "cuda:0", torch.float32)
    model.fused_f32 = False
    return model


def inputs(model, B, S, seed=0, padded=False):
    rng = np.random.default_rng(seed)
    ids = rng.integers(0, model.vocab, (B, S))
    mask = np.ones((B, S), np.int64)
    if padded:
        for i in range(B):
            mask[i, :rng.integers(0, S // 2)] = 0
    return ids, mask


def test_refused_without_a_gpu():
    """What a model with 4-bit weights refuses before it looks at a weight."""
    from dataclasses import replace

    from qdc_amd import backbone
    cfg, _ = weights_of("synthetic")
    make = lambda cfg=cfg, dtype=torch.float32, **kw: backbone.QwenBackbone(  # noqa: E731
        cfg, {}, "cpu", dtype, **kw)
    for kw in (dict(weight_format="int4"), dict(weight_format="w4", weight_group=16),
               dict(weight_format="w4", split_gemm_inputs="all", dtype=torch.bfloat16),
               dict(weight_format="w4", cfg=replace(cfg, hidden=12)),
               dict(weight_format="w4a8", cfg=replace(cfg, intermediate=520))):
        with pytest.raises(ValueError):
            make(**kw)


@pytest.mark.gpu
@pytest.mark.parametrize("config", ["synthetic", "plumbing"])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS)
def test_forward(fmt, dtype, group, config):
    from qdc_amd import backbone
    model, plain = model_of(fmt, dtype, config, group), plain_model(fmt, config, group)
    for B, S, padded in ((1, 1, False), (1, 37, False), (3, 200, True)):
        ids, mask = inputs(model, B, S, seed=S, padded=padded)
        got = backbone.batch_backbone_states(model, ids, mask).cpu().numpy()
        want = backbone.batch_backbone_states(plain, ids, mask).cpu().numpy()
        kept = mask.astype(bool)
        assert normwise(got[kept], want[kept]) <= BARS[fmt, dtype], (B, S)
        last = backbone.batch_backbone_hidden(model, ids, mask)
        assert normwise(last, want[:, -1]) <= BARS[fmt, dtype], (B, S)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", FORMATS)
def test_cache_and_graphs(fmt, dtype):
    """Prompts, forks and steps of a cache, eagerly and from recorded graphs, and the
    recorded last-token forward, against the forward of the whole sequence."""
    from qdc_amd import backbone, graphs
    from qdc_amd.cache import BackboneCache
    model = model_of(fmt, dtype)
    whole = lambda ids: backbone.backbone_last_hidden(  # noqa: E731
        model, np.asarray(ids), np.ones(len(ids), np.int64))
    bar = BARS[fmt, dtype]
    cache = BackboneCache(model, rows=10, pages=40, page_size=16, max_tokens=120)
    ids, mask = inputs(model, 3, 50, seed=1, padded=True)
    rows, got = cache.prefill(ids, mask)
    held = {r: i[m == 1].tolist() for r, i, m in zip(rows, ids, mask)}
    for kid in cache.fork([rows[0]] * 2):
        held[kid] = list(held[rows[0]])
    for r, g in zip(rows, got):
        assert normwise(g, whole(held[r])) <= bar
    steps = graphs.StepGraphs(cache)
    rng = np.random.default_rng(2)
    for turn in range(6):
        which = list(held)[: 1 + turn % len(held)]
        token = rng.integers(0, model.vocab, len(which))
        got = (cache.step if turn % 2 else steps)(which, token)
        for r, t, g in zip(which, token, got):
            held[r].append(int(t))
            assert normwise(g, whole(held[r])) <= bar, (turn, r)
    last = graphs.LastHiddenGraphs(model)
    for n in (20, 33, 20):
        ids = rng.integers(0, model.vocab, n)
        assert normwise(last(ids, np.ones(n, np.int64)), whole(ids)) <= bar


@pytest.mark.gpu
def test_memory():
    """Projections take 4 bits a weight and the scales' 16 a group."""
    model = model_of("w4", torch.bfloat16)
    cfg = model.cfg
    for layer in model.layers:
        w = layer["gate_up"]
        assert w.gated and (w.out, w.inner) == (2 * cfg.intermediate, cfg.hidden)
        assert w.packed.numel() * 8 == w.out * w.inner
        assert w.scales.numel() * w.group == w.out * w.inner
        assert "down_rows" not in layer and "out_rows" not in layer
