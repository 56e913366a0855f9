"""Sequences continued token by token (qdc_amd.cache.BackboneCache): prompts, steps,
forks, ends and moves together, as a server uses them, against the forward of the
whole sequence."""
import numpy as np
import pytest
import torch

from conftest import normwise

MODES = {"f32": (torch.float32, False), "bf16": (torch.bfloat16, False),
         "mlp": (torch.bfloat16, "mlp"), "all": (torch.bfloat16, "all")}
# fp32: both paths hold 1e-5 of the exact forward.  bf16 with split GEMM inputs: 1e-2,
# the bar that both paths hold; stored in bf16 throughout: each within it, so twice that
# between the two.
BARS = {"f32": 2e-5, "bf16": 2e-2, "mlp": 1e-2, "all": 1e-2}


def model_of(mode, config="synthetic", seed=21):
    from qdc_amd import backbone
    from qdc_amd import config as C
    from qdc_amd.weights import random_weights
    cfg = {"synthetic": C.synthetic_inference_config, "plumbing": C.plumbing_config}[config]()
    weights = random_weights(cfg, seed=seed)
    dtype, split = MODES[mode]
    if dtype == torch.bfloat16:
        from oracle import qdc_oracle as O
        weights = {k: O.round_bf16(v) for k, v in weights.items()}
    return backbone.QwenBackbone.from_weights(weights, cfg, "cuda:0", dtype, split_gemm_inputs=split)


def whole(model, ids):
    from qdc_amd import backbone
    return backbone.backbone_last_hidden(model, np.asarray(ids), np.ones(len(ids), np.int64))


@pytest.mark.gpu
@pytest.mark.parametrize("config", ["synthetic", "plumbing"])
@pytest.mark.parametrize("mode", list(MODES))
def test_sequences(mode, config):
    """Padded prompts of several lengths, steps, forks that part, a parent that ends
    before its children, a move of all pages and steps after it."""
    from qdc_amd.cache import BackboneCache
    model = model_of(mode, config)
    cache = BackboneCache(model, rows=10, pages=40, page_size=16, max_tokens=120)
    rng = np.random.default_rng(1)
    vocab = model.vocab
    held = {}

    def check(rows, got):
        for r, g in zip(rows, got):
            exp = whole(model, held[r])
            assert normwise(g, exp) <= BARS[mode], (r, len(held[r]), normwise(g, exp))

    lengths = [50, 33, 3, 64]
    ids = rng.integers(0, vocab, (4, 70))
    mask = np.zeros((4, 70), np.int64)
    for i, n in enumerate(lengths):
        mask[i, 70 - n:] = 1
    rows, got = cache.prefill(ids, mask)
    held.update({r: ids[i, 70 - n:].tolist() for i, (r, n) in enumerate(zip(rows, lengths))})
    check(rows, got)
    one, got = cache.prefill(rng.integers(0, vocab, 1))   # a prompt of one token
    free_before = cache.free_page_count()
    cache.free(one)
    assert cache.free_page_count() == free_before + 1

    def step(which):
        new = rng.integers(0, vocab, len(which))
        got = cache.step(which, new)
        for r, t in zip(which, new):
            held[r].append(int(t))
        check(which, got)

    for _ in range(3):
        step(rows)
    step([rows[2], rows[0]])
    kids = cache.fork([rows[0], rows[3], rows[0], rows[2]])
    for k, p in zip(kids, (rows[0], rows[3], rows[0], rows[2])):
        held[k] = list(held[p])
    for _ in range(2):
        step(kids + rows)
    cache.free([rows[0], kids[1]])
    del held[rows[0]], held[kids[1]]
    left = [kids[2], rows[1], kids[0], rows[3], rows[2], kids[3]]
    step(left)
    cache.compact()
    used = 40 - cache.free_page_count()
    assert cache.book.table.max().item() == used - 1
    for _ in range(18):                                   # over page borders
        step(left)
    assert cache.lengths() == {r: len(t) for r, t in held.items()}
    cache.free(left)
    assert cache.free_page_count() == 40 and not cache.lengths()


@pytest.mark.gpu
@pytest.mark.parametrize("mode", list(MODES))
def test_long_sequences(mode):
    """Rows that may hold some thousands of tokens, so that attention is dealt out by what
    they hold: a long and a short one, forks and a move, eager and recorded steps."""
    from qdc_amd import _lib
    from qdc_amd.cache import BackboneCache
    from qdc_amd.graphs import StepGraphs
    model = model_of(mode)
    cfg, dtype = model.cfg, _lib.QDC_F32 if mode == "f32" else _lib.QDC_BF16
    cache = BackboneCache(model, rows=6, pages=150, page_size=16)
    assert _lib.lib().qdc_paged_attention_workspace(1, cfg.heads, cfg.kv_heads, cfg.head_dim, 150,
                                                    16, dtype) > 0
    graphs = StepGraphs(cache, gemm_libraries=None)
    rng = np.random.default_rng(6)
    ids = rng.integers(0, model.vocab, (2, 1205))
    mask = np.ones_like(ids)
    mask[1, :-3] = 0
    (a, b), got = cache.prefill(ids, mask)
    held = {a: ids[0].tolist(), b: ids[1, -3:].tolist()}

    def check(rows, got):
        for r, g in zip(rows, got):
            exp = whole(model, held[r])
            assert normwise(g, exp) <= BARS[mode], (r, len(held[r]), normwise(g, exp))

    check((a, b), got)
    kids = cache.fork([a, b, a])
    held.update({k: list(held[p]) for k, p in zip(kids, (a, b, a))})
    for i in range(4):
        if i == 2:
            cache.free([kids[0]])
            del held[kids[0]]
            cache.compact()
        rows = list(held)[::-1]
        tokens = rng.integers(0, model.vocab, len(rows))
        got = (graphs if i % 2 else cache.step)(rows, tokens)
        for r, t in zip(rows, tokens):
            held[r].append(int(t))
        check(rows, got)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["mlp", "all"])
@pytest.mark.parametrize("intermediate,parts", [(1536, 8), (2560, 16), (3584, 16)])
def test_few_rows_of_split_inputs(mode, intermediate, parts):
    """The wide inner product of a step's MLP through the product cut in parts, from 1 to 63
    rows, beside the whole product, which takes the others; then steps of such a model."""
    import dataclasses

    from oracle import qdc_oracle as O
    from qdc_amd import backbone, ops
    from qdc_amd.cache import BackboneCache
    from qdc_amd.config import synthetic_inference_config
    from qdc_amd.weights import random_weights
    cfg = dataclasses.replace(synthetic_inference_config(), intermediate=intermediate)
    weights = {k: O.round_bf16(v) for k, v in random_weights(cfg, seed=4).items()}
    model = backbone.QwenBackbone.from_weights(weights, cfg, "cuda:0", torch.bfloat16,
                                               split_gemm_inputs=mode)
    cache = BackboneCache(model, rows=8, pages=60, page_size=16)
    layer, norm = model.layers[1], model.layers[2]["input_norm"]
    w = layer["down_rows"]
    assert w.shape == (cfg.hidden, intermediate)
    used = []
    cut = ops.linear_residual_rms

    def record(*args, **kwargs):
        used.append(args[5])
        return cut(*args, **kwargs)

    g = torch.Generator(device="cuda:0").manual_seed(intermediate)
    with pytest.MonkeyPatch.context() as m:
        m.setattr(ops, "linear_residual_rms", record)
        for n in (1, 2, 33, 63, 64):
            t = lambda *s: torch.randn(s, generator=g, device="cuda:0")  # noqa: E731
            h = t(n, cfg.hidden)
            act = ops.native_mlp_gate(t(n, intermediate), t(n, intermediate), out_dtype=ops.BF16X2)
            keep = torch.ones(n, dtype=torch.int32, device="cuda:0")
            keep[n // 2] = int(n == 1)
            used.clear()
            got = cache._project_add_norm(h, act, layer, "down", norm, token_mask=keep,
                                          out_dtype=ops.BF16X2)
            assert used == ([parts] if n < 64 else used)
            # fp32 sums of exact products of bf16, two a value of the input
            x = ops.join_split(act).double()
            exp = h.double() + x @ w.double().t()
            tol = (2 * intermediate + 20) * 2.0 ** -24 * (h.double().abs() + x.abs() @ w.double().abs().t())
            assert ((got[0].double() - exp).abs() <= tol).all()
            scale = 1 / torch.sqrt(exp.square().mean(-1, keepdim=True) + cfg.eps)
            out = exp * scale * (1 + norm.double()) * keep[:, None]
            # the norm's sum and root add 300 half steps at most; the split form 2^-17
            tol = (tol + exp.abs() * tol.amax(-1, keepdim=True) * scale) * scale * 2 \
                + (300 * 2.0 ** -24 + 2.0 ** -17) * out.abs()
            assert ((ops.join_split(got[1]).double() - out).abs() <= tol).all()
            assert (got[1][keep == 0] == 0).all()
        used.clear()
        ids = np.arange(8 * 5).reshape(8, 5)
        rows, _ = cache.prefill(ids)
        used.clear()
        got = cache.step(rows, np.arange(8))
        assert used.count(parts) == len(model.layers)
    for i, out in enumerate(got):
        assert normwise(out, whole(model, ids[i].tolist() + [i])) <= BARS[mode]


@pytest.mark.gpu
def test_too_few_pages_leaves_everything():
    """A prompt, a step or a fork that does not fit raises, and what was there goes on."""
    from qdc_amd.cache import BackboneCache
    model = model_of("f32")
    cache = BackboneCache(model, rows=5, pages=6, page_size=16, max_tokens=64)
    rng = np.random.default_rng(2)
    tokens = rng.integers(0, model.vocab, (2, 47)).tolist()
    (a, b), _ = cache.prefill(tokens)
    held = {a: list(tokens[0]), b: list(tokens[1])}
    for call in (lambda: cache.prefill(rng.integers(0, model.vocab, 5)), lambda: cache.fork([a]),
                 lambda: cache.fork([a, b, a, b])):
        with pytest.raises(RuntimeError):
            call()
        assert cache.lengths() == {a: 47, b: 47}

    def step(rows):
        new = rng.integers(0, model.vocab, len(rows))
        for r, t, g in zip(rows, new, cache.step(rows, new)):
            held[r].append(int(t))
            assert normwise(g, whole(model, held[r])) <= BARS["f32"]

    step([a, b])                                          # 48: the pages are full
    with pytest.raises(RuntimeError):
        cache.step([b, a], [1, 2])
    assert cache.lengths() == {a: 48, b: 48}
    kid, = cache.fork([a])                                # full pages are shared
    held[kid] = list(held[a])
    cache.free([b])
    for _ in range(3):
        step([a, kid])


@pytest.mark.gpu
def test_a_call_that_raises_ends_its_rows(monkeypatch):
    from qdc_amd import ops
    from qdc_amd.cache import BackboneCache
    model = model_of("f32")
    cache = BackboneCache(model, rows=4, pages=20, page_size=16)
    (a, b), _ = cache.prefill(np.arange(60).reshape(2, 30))

    def fail(*args, **kwargs):
        raise MemoryError("none left")

    for call in (lambda: cache.prefill([1, 2, 3]), lambda: cache.step([b], [5])):
        with monkeypatch.context() as m:
            m.setattr(ops, "native_residual_rms", fail)
            with pytest.raises(MemoryError):
                call()
    assert cache.lengths() == {a: 30} and cache.free_page_count() == 18
    got = cache.step([a], [7])
    assert normwise(got[0], whole(model, list(range(30)) + [7])) <= BARS["f32"]
    rows, _ = cache.prefill(np.arange(6).reshape(3, 2))
    assert len(rows) == 3 and sorted(cache.lengths()) == [0, 1, 2, 3]


@pytest.mark.gpu
def test_a_call_that_raises_leaves_no_flag_and_no_rows(monkeypatch):
    """A fork whose copies raise gives its rows back, and a call that raises after its
    kernels found too few pages does not fail the next one."""
    from qdc_amd import cache as module
    from qdc_amd.cache import BackboneCache
    model = model_of("f32")
    cache = BackboneCache(model, rows=4, pages=5, page_size=16)
    (a,), _ = cache.prefill(np.arange(30))

    def fail(*args, **kwargs):
        raise MemoryError("none left")

    for name, call in (("copy_pages", lambda: cache.fork([a, a])),
                       ("prepare_paged", lambda: cache.prefill(np.arange(70)))):
        with monkeypatch.context() as m:
            m.setattr(module.cache_ops, name, fail)
            with pytest.raises(MemoryError):
                call()
        assert cache.lengths() == {a: 30} and cache.free_page_count() == 3
    kids = cache.fork([a, a, a])
    assert len(kids) == 3 and cache.free_page_count() == 0
    for got in cache.step([a] + kids, [7] * 4):
        assert normwise(got, whole(model, list(range(30)) + [7])) <= BARS["f32"]


@pytest.mark.gpu
def test_an_upload_that_raises_changes_nothing(monkeypatch):
    """No memory for a call's own numbers: every row, free or not, is what it was."""
    from qdc_amd import backbone
    from qdc_amd.cache import BackboneCache
    model = model_of("f32")
    cache = BackboneCache(model, rows=4, pages=20, page_size=16)
    (a,), _ = cache.prefill(np.arange(30))

    def fail(*args, **kwargs):
        raise MemoryError("none left")

    prompt = lambda: cache.prefill([1, 2, 3])  # noqa: E731
    for where, name, call in ((backbone, "_upload", prompt), (BackboneCache, "_ints", prompt),
                              (BackboneCache, "_ints", lambda: cache.fork([a, a])),
                              (BackboneCache, "_ints", lambda: cache.step([a], [1])),
                              (BackboneCache, "_ints", lambda: cache.free([a]))):
        with monkeypatch.context() as m:
            m.setattr(where, name, fail)
            with pytest.raises(MemoryError):
                call()
        assert cache.lengths() == {a: 30} and cache.free_page_count() == 18
    assert sorted([a] + cache.fork([a, a, a])) == [0, 1, 2, 3]
    got = cache.step([a], [7])
    assert normwise(got[0], whole(model, list(range(30)) + [7])) <= BARS["f32"]


def interrupted(wait):
    """``wait`` with an interrupt that arrives while it waits, once."""
    left = [1]

    def call(*args, **kwargs):
        out = wait(*args, **kwargs)
        if left:
            left.pop()
            raise KeyboardInterrupt
        return out
    return call


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["prefill", "step", "fork", "graphs"])
@pytest.mark.parametrize("wait", ["cpu", "item", "synchronize"])
def test_an_interrupted_call_ends_its_rows(monkeypatch, what, wait):
    """An interrupt while a call waits for the device: the rows that it was at are ended
    or, where it did not wait so, as the call leaves them; no row has tokens that
    ``lengths`` does not say, and every row and page can be taken again."""
    from qdc_amd.cache import BackboneCache
    from qdc_amd.graphs import StepGraphs
    model = model_of("f32")
    cache = BackboneCache(model, rows=4, pages=12, page_size=16)
    graphs = StepGraphs(cache, gemm_libraries=None)
    rng = np.random.default_rng(3)
    prompts = rng.integers(0, model.vocab, (2, 31))
    (a, b), _ = cache.prefill(prompts)
    held = {a: prompts[0].tolist(), b: prompts[1].tolist()}
    graphs([a], [1]), held[a].append(1)
    where = torch.cuda.Stream if wait == "synchronize" else torch.Tensor
    with monkeypatch.context() as m:
        m.setattr(where, wait, interrupted(getattr(where, wait)))
        try:
            if what == "prefill":
                rows, _ = cache.prefill(prompts[0, :20])
                held[rows[0]] = prompts[0, :20].tolist()
            elif what == "fork":
                kid, = cache.fork([b])
                held[kid] = list(held[b])
            else:
                (cache.step if what == "step" else graphs)([b], [5])
                held[b].append(5)
            stopped = False
        except KeyboardInterrupt:
            stopped = True
    if stopped and what in ("step", "graphs"):
        del held[b]
    assert stopped == ((wait, what) in (("cpu", "prefill"), ("cpu", "step"), ("item", "prefill"),
                                        ("item", "step"), ("item", "fork"),
                                        ("synchronize", "graphs")))
    assert cache.lengths() == {r: len(t) for r, t in held.items()}
    lengths = cache.book.lengths.tolist()
    assert lengths == [len(held.get(r, [])) for r in range(4)]
    for r in held:
        got = cache.step([r], [9])
        held[r].append(9)
        assert normwise(got[0], whole(model, held[r])) <= BARS["f32"]
    rest = 4 - len(held)
    rows, got = cache.prefill(np.tile(prompts[1], (rest, 1)))
    assert sorted(rows + list(held)) == [0, 1, 2, 3]
    for g in got:
        assert normwise(g, whole(model, prompts[1])) <= BARS["f32"]
    cache.free(list(cache.lengths()))
    assert cache.free_page_count() == 12


@pytest.mark.gpu
def test_an_interrupted_replay_without_memory(monkeypatch):
    """Where the rows of an interrupted call cannot be ended either, they are out of use."""
    from qdc_amd.cache import BackboneCache
    from qdc_amd.graphs import StepGraphs
    model = model_of("f32")
    cache = BackboneCache(model, rows=3, pages=12, page_size=16)
    graphs = StepGraphs(cache, gemm_libraries=None)
    (a, b), _ = cache.prefill([[1, 2, 3], [4, 5, 6]])
    graphs([a], [1])

    def fail(*args, **kwargs):
        raise MemoryError("none left")

    with monkeypatch.context() as m:
        m.setattr(torch.cuda.Stream, "synchronize", interrupted(torch.cuda.Stream.synchronize))
        m.setattr(BackboneCache, "_ints", fail)
        with pytest.raises((MemoryError, KeyboardInterrupt)):
            graphs([b], [1])
    assert cache.lengths() == {a: 4}
    for call in (graphs, cache.step):
        with pytest.raises(ValueError):
            call([b], [2])
    got = cache.step([a], [7])
    assert normwise(got[0], whole(model, [1, 2, 3, 1, 7])) <= BARS["f32"]


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["f32", "mlp"])
def test_step_graphs(mode):
    """Recorded steps beside eager ones of a second cache: the same bits with the same
    GEMM library, over page borders, forks, a move, other row counts and eager steps
    between, and too few pages raise and leave everything."""
    from qdc_amd.cache import BackboneCache
    from qdc_amd.graphs import StepGraphs
    model = model_of(mode)
    new = lambda: BackboneCache(model, rows=6, pages=13, page_size=16)  # noqa: E731
    cache, twin = new(), new()
    graphs = StepGraphs(cache, max_graphs=2, gemm_libraries=None)
    rng = np.random.default_rng(8)
    ids = rng.integers(0, model.vocab, (2, 30))
    (a, b), _ = cache.prefill(ids)
    assert twin.prefill(ids)[0] == [a, b]
    held = {a: ids[0].tolist(), b: ids[1].tolist()}

    def step(rows, eager=False):
        tokens = rng.integers(0, model.vocab, len(rows))
        got = (cache.step if eager else graphs)(rows, tokens)
        assert np.array_equal(got, twin.step(rows, tokens))
        for r, t in zip(rows, tokens):
            held[r].append(int(t))
        assert cache.lengths() == twin.lengths() == {r: len(t) for r, t in held.items()}
        return got

    for i in range(4):
        got = step([b, a], eager=i == 2)                  # 32 and on: another page each
    for r, g in zip((b, a), got):
        assert normwise(g, whole(model, held[r])) <= BARS[mode]
    kids = cache.fork([a, b])
    assert twin.fork([a, b]) == kids
    held.update({k: list(held[p]) for k, p in zip(kids, (a, b))})
    for _ in range(3):
        step(kids + [a, b])
    step([a])                                             # a third key: the first is dropped
    assert list(graphs._entries) == [(4,), (1,)] and not graphs.eager_keys
    cache.free([b]), twin.free([b])
    del held[b]
    cache.compact()
    for _ in range(2):
        got = step([kids[1], a])
    assert normwise(got[0], whole(model, held[kids[1]])) <= BARS[mode]
    for c in (cache, twin):                               # the pages that are left
        c.prefill(np.ones(16 * c.free_page_count()))
    full, = set(cache.lengths()) - set(held)
    held[full] = [1] * cache.lengths()[full]
    before = cache.lengths()
    for call in (graphs, cache.step):
        with pytest.raises(RuntimeError):
            call([full, a], [1, 2])
        assert cache.lengths() == before
    step([a])
    for bad in (lambda: graphs([a], [model.vocab]), lambda: graphs([a, a], [1, 2]),
                lambda: graphs([5], [1]), lambda: graphs([], [])):
        with pytest.raises(ValueError):
            bad()
    both = StepGraphs(cache, trials=2)                    # the faster of the two libraries
    got = both([a], [3])
    held[a].append(3)
    assert normwise(got[0], whole(model, held[a])) <= BARS[mode]
    with pytest.raises(ValueError):
        StepGraphs(cache, max_graphs=0)


@pytest.mark.gpu
def test_refusals():
    import dataclasses

    from qdc_amd import backbone
    from qdc_amd.cache import BackboneCache
    from qdc_amd.config import synthetic_inference_config
    from qdc_amd.weights import random_weights
    model = model_of("f32")
    for bad in (dict(rows=0, pages=4), dict(rows=2, pages=0), dict(rows=2, pages=4, page_size=20),
                dict(rows=2, pages=4, max_tokens=0)):
        with pytest.raises(ValueError):
            BackboneCache(model, **bad)
    for change in (dict(head_dim=32), dict(key_dim=48), dict(value_dim=40), dict(conv_kernel=9)):
        cfg = dataclasses.replace(synthetic_inference_config(), **change)
        other = backbone.QwenBackbone.from_weights(random_weights(cfg, seed=1), cfg)
        with pytest.raises(ValueError):
            BackboneCache(other, rows=2, pages=4)
    cache = BackboneCache(model, rows=3, pages=8, page_size=16, max_tokens=40)
    (row,), _ = cache.prefill([1, 2, 3])
    mask = lambda *m: np.array([m])  # noqa: E731
    for bad in (lambda: cache.prefill([]), lambda: cache.prefill([model.vocab]),
                lambda: cache.prefill([[1, 2]], mask(1, 0)), lambda: cache.prefill([[1, 2]], mask(0, 0)),
                lambda: cache.prefill([[1, 2, 3]], mask(1, 0, 1)), lambda: cache.prefill([[1, 2]], mask(0, 2)),
                lambda: cache.prefill([[1, 2]], mask(1)), lambda: cache.prefill(np.ones((1, 1, 2))),
                lambda: cache.prefill(np.ones(41)), lambda: cache.step([row], [-1]),
                lambda: cache.step([row], [1, 2]), lambda: cache.step([], []),
                lambda: cache.step([row, row], [1, 2]), lambda: cache.step([row + 1], [1]),
                lambda: cache.fork([row, 99]), lambda: cache.free([row, row]), lambda: cache.free([9])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        cache.fork([row, row, row])                       # rows
    assert cache.fork([]) == [] and cache.lengths() == {row: 3}
    long, _ = cache.prefill(np.ones(40))
    with pytest.raises(ValueError):
        cache.step(long, [1])


@pytest.mark.gpu
def test_more_rows_than_a_call_takes():
    """Where sequences may be so long that attention does not take all rows at once, a call
    of too many is refused before anything runs, and its rows go on."""
    import dataclasses

    from qdc_amd import _lib, backbone
    from qdc_amd.cache import BackboneCache
    from qdc_amd.config import synthetic_inference_config
    from qdc_amd.graphs import StepGraphs
    from qdc_amd.weights import random_weights
    cfg = dataclasses.replace(synthetic_inference_config(), layer_types=("full_attention",),
                              rotary_dim=0)
    model = backbone.QwenBackbone.from_weights(random_weights(cfg, seed=2), cfg)
    tokens, rows = 2 ** 26, 300
    takes = lambda n, t=tokens: _lib.lib().qdc_paged_attention_workspace(  # noqa: E731
        n, cfg.heads, cfg.kv_heads, 64, t // 256, 256, _lib.QDC_F32) >= 0
    assert takes(150) and not takes(rows) and not takes(1, 2 ** 31)
    cache = BackboneCache(model, rows=rows, pages=rows, page_size=256, max_tokens=tokens)
    ids = np.arange(rows)[:, None] % cfg.vocab
    held, _ = cache.prefill(ids[:150])
    held += cache.prefill(ids[150:])[0]
    for call in (lambda: cache.step(held, ids), lambda: StepGraphs(cache)(held, ids)):
        with pytest.raises(ValueError, match="at most 150"):
            call()
        assert cache.lengths() == {r: 1 for r in range(rows)}
    got = cache.step(held[100:250], ids[100:250])
    assert np.isfinite(got).all() and cache.book.lengths.tolist() == [
        1 + (r in held[100:250]) for r in range(rows)]
    cache.free(held)
    with pytest.raises(ValueError, match="at most 150"):
        cache.prefill(ids)
    for many in (ids, np.tile(ids, (2, 1))):              # more than are free, than there are
        with pytest.raises(RuntimeError, match="free rows"):
            BackboneCache(model, rows=150, pages=rows, page_size=256).prefill(many)
    assert not cache.lengths() and cache.free_page_count() == rows
    with pytest.raises(ValueError, match="max_tokens"):
        BackboneCache(model, rows=1, pages=1, page_size=256, max_tokens=2 ** 31)


@pytest.mark.gpu
def test_made_on_another_stream(monkeypatch):
    """A cache made on a stream that has much to do, then used on another one: it is whole
    before the first call."""
    import dataclasses

    from qdc_amd import backbone
    from qdc_amd import cache as module
    from qdc_amd.config import synthetic_inference_config
    from qdc_amd.weights import random_weights
    # (no attention layer: the upload of rotation tables would wait for the stream)
    cfg = dataclasses.replace(synthetic_inference_config(), layer_types=("linear_attention",) * 2)
    model = backbone.QwenBackbone.from_weights(random_weights(cfg, seed=2), cfg)
    ids = np.arange(40)
    want = whole(model, ids)
    new = lambda: module.BackboneCache(model, rows=3, pages=8, page_size=16)  # noqa: E731
    new()                                                 # (new memory might wait as well)
    big, busy, table = torch.randn(8192, 8192, device="cuda:0"), torch.cuda.Event(), \
        module.cache_ops.page_table

    def slow(*args):
        out, x = table(*args), big
        for _ in range(30):
            x = x @ big * 1e-3
        busy.record()
        return out

    slow(3, 8, 8, 16, "cuda:0")
    torch.cuda.synchronize()
    monkeypatch.setattr(module.cache_ops, "page_table", slow)
    cache = new()
    assert busy.query()
    with torch.cuda.stream(torch.cuda.Stream()):
        (row,), got = cache.prefill(ids[:-1])
        got = cache.step([row], ids[-1:])
        assert cache.free_page_count() == 5
    assert normwise(got[0], want) <= BARS["f32"]


@pytest.mark.gpu
@pytest.mark.parametrize("kinds", [("full_attention",), ("linear_attention", "linear_attention")])
def test_one_kind_of_layer(kinds):
    """Models with no state to keep, or with no pages."""
    import dataclasses

    from qdc_amd import backbone
    from qdc_amd.cache import BackboneCache
    from qdc_amd.config import synthetic_inference_config
    from qdc_amd.weights import random_weights
    cfg = dataclasses.replace(synthetic_inference_config(), layer_types=kinds)
    model = backbone.QwenBackbone.from_weights(random_weights(cfg, seed=2), cfg)
    cache = BackboneCache(model, rows=4, pages=16, page_size=16)
    rng = np.random.default_rng(4)
    ids = rng.integers(0, cfg.vocab, 21).tolist()
    (row,), got = cache.prefill(ids)
    assert normwise(got[0], whole(model, ids)) <= BARS["f32"]
    kid, = cache.fork([row])
    cache.compact()
    for t in rng.integers(0, cfg.vocab, 4).tolist():
        ids.append(t)
        got = cache.step([kid, row], [t, t])
        assert np.array_equal(got[0], got[1])
        assert normwise(got[0], whole(model, ids)) <= BARS["f32"]


def test_packed_integers():
    """Host vectors to the device in one copy, each starting on 16 bytes."""
    from types import SimpleNamespace

    from qdc_amd.cache import BackboneCache
    self = SimpleNamespace(model=SimpleNamespace(device="cpu"))
    a, b, c = BackboneCache._ints(self, np.arange(5), np.array([[7, 8], [9, -1]]), np.array([3]))
    assert a.tolist() == [0, 1, 2, 3, 4] and b.tolist() == [7, 8, 9, -1] and c.tolist() == [3]
    assert b.data_ptr() - a.data_ptr() == 32 and c.data_ptr() - b.data_ptr() == 16
