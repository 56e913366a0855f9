"""The operators of the paged cache whose speed is measured, over the sizes, data
types and lengths they are used at: one token's attention over cache pages, q/k
norms with the rotation and the page store, one token of the linear-attention
recurrence, and the pages' own bookkeeping and copies.

``listed()`` names the cases, ``draw(rng)`` gives one more of the same ranges,
``prepare`` makes what a program holds before the call, ``run`` is one pass: the
operators in plain torch, or with ``own`` the calls that a program makes of
``qdc_amd.cache_ops``.  ``exact`` is the same result in 64 bits from the definition.

A cache: pages ``[pages, kv_heads, page_size, head_dim]`` (for several layers one
pool ``[planes, pages, ...]``, K and V a plane each); ``table[row, j]`` the page that
holds a row's positions ``j * page_size ..``, -1 behind its last; ``lengths``;
``refs``, how many rows share a page; ``free``, a count and a stack of free pages.
Places that hold no token hold NaN here, as nothing may read them.
"""
import math
import os
import sys

import numpy as np
import torch

own = False
DEVICE = "cuda:0"
EPS = 1e-6
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
# query heads, KV heads, head size, rotated values
HEADS = {"decision": (4, 2, 64, 16), "0.8b": (8, 2, 256, 64), "wide": (16, 4, 256, 64),
         "128": (12, 4, 128, 32), "one-kv": (4, 1, 64, 16)}
# key heads, value heads, key size, value size
DELTA = {"decision": (2, 4, 128, 128), "0.8b": (16, 16, 128, 128), "wide": (16, 32, 128, 128)}
TAPS = 4


def _framework():
    """The framework's operators, imported at the first call and not at each."""
    ops = sys.modules.get("qdc_amd.cache_ops")
    if ops is None:
        package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                               "qwendecisioncore.jl_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        from qdc_amd import cache_ops as ops
    return ops


# -------------------------------------------------------------------- cases --
def listed():
    return [
        # The small decision model scoring one more token of one prompt: launches
        # and latency are all of it.
        _attend("attend_1x411_f32", "decision", "f32", 16, 1, 411, 411, 0.0),
        # A step of a batch of equal prompts.
        _attend("attend_8x2048_bf16", "0.8b", "bf16", 64, 8, 2048, 2048, 0.0),
        # A serving batch: prompts of very different lengths, some rows empty.
        _attend("attend_96_ragged_bf16", "0.8b", "bf16", 32, 96, 1, 16384, 0.1),
        # Two long documents, odd length.
        _attend("attend_2x100003_wide_bf16", "wide", "bf16", 64, 2, 100003, 100003, 0.0),
        # q and k of one new token, into its page.
        _store("store_step_1_f32", "decision", "f32", 16, 1, 1, 411),
        # Eight left-padded prompts stored while they are run.
        _store("store_8x2048_bf16", "0.8b", "bf16", 64, 8, 2048, 0),
        # The recurrence's step of one row, of a batch, of a wider layer's large batch.
        _delta("delta_1_f32", "decision", "f32", 1),
        _delta("delta_64_bf16", "0.8b", "bf16", 64),
        _delta("delta_151_wide_bf16", "wide", "bf16", 151),
        # One prompt forked into its candidate answers, small and large model; the
        # candidates of the pass before are freed first.
        {"name": "fork_1_to_5_f32", "kind": "fork", "heads": "decision", "dtype": "f32",
         "page": 16, "layers": 1, "states": 3, "parents": 1, "each": 5, "low": 411, "high": 411},
        {"name": "fork_8_to_40_bf16", "kind": "fork", "heads": "0.8b", "dtype": "bf16",
         "page": 64, "layers": 6, "states": 18, "parents": 8, "each": 5, "low": 100, "high": 3000},
        # Prompts that come and go: new rows get pages, the old ones are freed, and
        # the pages that are left move together.
        {"name": "turnover_32_bf16", "kind": "turnover", "heads": "0.8b", "dtype": "bf16",
         "page": 64, "layers": 6, "rows": 32, "low": 20, "high": 2500},
    ]


def _attend(name, heads, dtype, page, rows, low, high, empty):
    """``rows`` queries, lengths log-uniform in low..high, a share of them empty."""
    return {"name": name, "kind": "attend", "heads": heads, "dtype": dtype, "page": page,
            "rows": rows, "low": low, "high": high, "empty": empty}


def _store(name, heads, dtype, page, rows, tokens, at):
    """``tokens`` new tokens of each row: one at position ``at``, or a whole prompt."""
    return {"name": name, "kind": "store", "heads": heads, "dtype": dtype, "page": page,
            "rows": rows, "tokens": tokens, "at": at}


def _delta(name, heads, dtype, rows):
    return {"name": name, "kind": "delta", "heads": heads, "dtype": dtype, "rows": rows}


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "store", "delta", "delta", "fork", "turnover"])
    dtype = rng.choice(["f32", "bf16", "bf16"])
    page = rng.choice([16, 32, 64, 128])
    heads = rng.choice(list(HEADS))
    if kind == "attend":
        rows = _log_int(rng, 1, 200)
        H, KV, hd, _ = HEADS[heads]
        # at most the keys of the largest listed case, in bytes of one row's heads
        most = 200000 * 4 * 256 // (KV * hd * (2 if dtype == "f32" else 1)) // rows
        high = _log_int(rng, 1, min(100003, most))
        low = rng.choice([1, high, max(1, high // 2)])
        empty = rng.choice([0.0, 0.0, 0.2]) if rows > 7 else 0.0
        case = _attend("", heads, dtype, page, rows, low, high, empty)
    elif kind == "store":
        if rng.random() < 0.5:
            case = _store("", heads, dtype, page, _log_int(rng, 1, 256), 1, rng.randint(0, 5000))
        else:
            rows = _log_int(rng, 1, 8)
            most = 8192 if dtype == "f32" or heads == "wide" else 16384
            case = _store("", heads, dtype, page, rows, _log_int(rng, 2, most // rows), 0)
    elif kind == "delta":
        case = _delta("", rng.choice(list(DELTA)), dtype, _log_int(rng, 1, 151))
    elif kind == "fork":
        case = {"kind": kind, "heads": heads, "dtype": dtype, "page": page,
                "layers": rng.randint(1, 4), "states": rng.randint(1, 6),
                "parents": _log_int(rng, 1, 8), "each": rng.randint(1, 5),
                "low": _log_int(rng, 1, 100), "high": _log_int(rng, 101, 2000)}
    else:
        case = {"kind": kind, "heads": heads, "dtype": dtype, "page": page,
                "layers": rng.randint(1, 3), "rows": _log_int(rng, 1, 32),
                "low": _log_int(rng, 1, 50), "high": _log_int(rng, 51, 1500)}
    case.pop("name", None)
    return case


# ------------------------------------------------------------------- inputs --
def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _ints(values):
    return torch.from_numpy(np.ascontiguousarray(values, np.int32)).to(DEVICE)


def _sizes(case, rows):
    """Lengths spread evenly over the logarithm of low..high, the same ones for every
    seed (so that the pools are of one size), a share of them nothing."""
    low, high = case["low"], case["high"]
    n = np.exp(math.log(low) + (np.arange(rows) + 0.5) / rows * math.log(high / low))
    n = np.clip(np.rint(n).astype(np.int64), low, high)
    n[:round(rows * case.get("empty", 0.0))] = 0
    return n


def _lengths(rng, case, rows):
    return rng.permutation(_sizes(case, rows))


def _table(rng, lengths, page, width=None, spare=0):
    """A table whose rows' pages lie anywhere, and how many pages there are."""
    blocks = -(-lengths // page)
    used = int(blocks.sum())
    pages = max(1, used + spare)
    table = np.full((len(lengths), width or max(1, int(blocks.max()))), -1, np.int64)
    table[np.arange(table.shape[1]) < blocks[:, None]] = rng.permutation(pages)[:used]
    return table, pages


def _held(table, lengths, pages, page):
    """``[pages, page]``: whether a place holds a token."""
    held = np.zeros((pages, page), bool)
    at = np.arange(table.shape[1]) * page
    filled = np.clip(lengths[:, None] - at, 0, page)
    keep = table >= 0
    held[table[keep]] = np.arange(page) < filled[keep][:, None]
    return torch.from_numpy(held).to(DEVICE)


def _pool(g, planes, held, kv, dim, dtype):
    pages, page = held.shape
    pool = torch.randn((planes, pages, kv, page, dim), generator=g, device=DEVICE,
                       dtype=torch.float32 if dtype == torch.float32 else torch.bfloat16)
    return pool.masked_fill_(~held[:, None, :, None], float("nan"))


def _rope(n, rotary):
    freq = (1e7 ** (-np.arange(0, rotary, 2) / rotary)).astype(np.float32)
    angle = (np.arange(n, dtype=np.float32)[:, None] * freq).astype(np.float64)
    return tuple(torch.from_numpy(f(angle).astype(np.float32)).to(DEVICE) for f in (np.cos, np.sin))


def _randn(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device=DEVICE) * scale).to(dtype)


def _prepare_attend(case, rng, g):
    H, KV, hd, _ = HEADS[case["heads"]]
    dtype, n = TYPES[case["dtype"]], case["rows"]
    lengths = _lengths(rng, case, n)
    table, pages = _table(rng, lengths, case["page"], spare=3)
    k, v = _pool(g, 2, _held(table, lengths, pages, case["page"]), KV, hd, dtype)
    order = rng.permutation(n)             # the batch takes the cache's rows in any order
    gate = _randn(g, n, 2, H, hd, dtype=dtype)
    return {"q": _randn(g, n, H, hd, dtype=dtype, scale=1.5), "k": k, "v": v,
            "gate": gate[:, 1], "table": _ints(table), "rows": _ints(order),
            "positions": _ints(lengths[order] - 1), "scale": hd ** -0.5}


def _prepare_store(case, rng, g):
    H, KV, hd, rotary = HEADS[case["heads"]]
    dtype, page, B, S = TYPES[case["dtype"]], case["page"], case["rows"], case["tokens"]
    if S == 1:
        positions = np.maximum(0, case["at"] - rng.integers(0, 1 + case["at"] // 4, B))
        rows = rng.permutation(B)
        lengths = np.empty(B, np.int64)
        lengths[rows] = positions + 1
    else:                                   # left padding of up to a third
        first = rng.permutation((np.arange(B) + 0.5) / B * (S / 3)).astype(np.int64)
        at = np.arange(S) - first[:, None]
        positions, rows = np.where(at < 0, -1, at).reshape(-1), np.repeat(np.arange(B), S)
        lengths = S - first
    table, pages = _table(rng, lengths, page, spare=2)
    pool = _randn(g, 2, pages, KV, page, hd, dtype=dtype)
    T = B * S
    proj = _randn(g, T, (2 * H + 2 * KV) * hd, dtype=dtype)
    q, k, v, _ = (x.unflatten(1, (-1, hd)) for x in
                  proj.split([H * hd, KV * hd, KV * hd, H * hd], 1))
    return {"q": q, "k": k, "v": v, "prompt": S > 1, "rotary": rotary,
            "q_norm": _randn(g, hd, scale=0.1, dtype=dtype),
            "k_norm": _randn(g, hd, scale=0.1, dtype=dtype),
            "rope": _rope(int(lengths.max()), rotary), "rows": _ints(rows),
            "positions": _ints(positions), "table": _ints(table),
            "k_pages": pool[0], "v_pages": pool[1]}


def _prepare_delta(case, rng, g):
    KH, H, kd, vd = DELTA[case["heads"]]
    dtype, n = TYPES[case["dtype"]], case["rows"]
    rows = n + 3
    channels = 2 * KH * kd + H * vd
    width = channels + H * vd + 2 * H
    dt = torch.empty(H, device=DEVICE).uniform_(math.log(1e-3), math.log(0.1), generator=g).exp()
    return {"proj": _randn(g, n, -(-width // 256) * 256, dtype=dtype),
            "conv": _randn(g, channels, TAPS, scale=0.4), "sizes": (KH, kd, H, vd),
            "a_decay": -torch.empty(H, device=DEVICE).uniform_(1.0, 16.0, generator=g),
            "dt_bias": dt + torch.log(-torch.expm1(-dt)),
            "norm": 1.0 + _randn(g, vd, scale=0.1, dtype=dtype),
            "ring": _randn(g, rows, TAPS, channels, dtype=dtype),
            "state": _randn(g, rows, H, vd, kd, scale=0.1),
            "rows": _ints(rng.permutation(rows)[:n]),
            # a row's first tokens among them, whose window reaches before its start
            "positions": _ints(np.where(rng.random(n) < 0.2, rng.integers(0, 4, n),
                                        rng.integers(4, 5000, n)))}


def _prepare_fork(case, rng, g):
    _, KV, hd, _ = HEADS[case["heads"]]
    page, n, each = case["page"], case["parents"], case["each"]
    rows = n * (1 + each)
    lengths = np.zeros(rows, np.int64)
    where = rng.permutation(rows)
    parents, children = where[:n], where[n:]
    lengths[parents] = _lengths(rng, case, n)
    table, pages = _table(rng, lengths, page, width=-(-case["high"] // page) + 1,
                          spare=n * each + 5)
    pool = _pool(g, 2 * case["layers"], _held(table, lengths, pages, page), KV, hd,
                 TYPES[case["dtype"]])
    refs = np.zeros(pages, np.int64)
    refs[table[table >= 0]] = 1
    KH, H, kd, vd = DELTA["decision" if hd == 64 else "0.8b"]
    return {"table": _ints(table), "lengths": _ints(lengths), "refs": _ints(refs),
            "free": _ints(_stack(refs)), "page": page, "pool": pool,
            "parents": _ints(np.repeat(parents, each)), "children": _ints(children),
            "states": _randn(g, case["states"], rows, H, vd, kd)}


def _stack(refs):
    """The lowest free page on top."""
    unused = np.flatnonzero(refs == 0)[::-1]
    return np.concatenate([[len(unused)], unused, np.zeros(len(refs) - len(unused), np.int64)])


def _prepare_turnover(case, rng, g):
    _, KV, hd, _ = HEADS[case["heads"]]
    page, n = case["page"], case["rows"]
    # n rows that stay, n that the next pass frees, n that it admits
    sizes = [_lengths(rng, case, n) for _ in range(3)]
    rows = rng.permutation(3 * n).reshape(3, n)
    lengths = np.zeros(3 * n, np.int64)
    lengths[rows[0]], lengths[rows[1]] = sizes[0], sizes[1]
    coming = int((-(-sizes[2] // page)).sum())
    # the rows' pages fill the low end, mixed; what comes is above them
    low, used = _table(rng, lengths, page, width=-(-case["high"] // page))
    pages = used + coming + 7
    refs = np.zeros(pages, np.int64)
    refs[low[low >= 0]] = 1
    pool = _randn(g, 2 * case["layers"], pages, KV, page, hd, dtype=TYPES[case["dtype"]])
    return {"table": _ints(low), "lengths": _ints(lengths), "refs": _ints(refs),
            "free": _ints(_stack(refs)), "page": page, "pool": pool,
            "turns": [(_ints(rows[1]), _ints(rows[2]), _ints(sizes[2])),
                      (_ints(rows[2]), _ints(rows[1]), _ints(sizes[1]))]}


_PREPARE = {"attend": _prepare_attend, "store": _prepare_store, "delta": _prepare_delta,
            "fork": _prepare_fork, "turnover": _prepare_turnover}


def prepare(case, seed):
    state = _PREPARE[case["kind"]](case, np.random.default_rng(seed), _generator(seed))
    state["kind"] = case["kind"]
    return state


# --------------------------------------------------------------------- runs --
def run(s):
    if own:
        return _OWN[s["kind"]](_framework(), s)
    return _PLAIN[s["kind"]](s)


def _book(ops, s):
    return ops.PageTable(s["table"], s["lengths"], s["refs"], s["free"], s["page"])


def _own_attend(ops, s):
    return ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["rows"], s["positions"],
                               s["scale"], gate=s["gate"])


def _own_store(ops, s):
    k_out = torch.empty(s["k"].shape, dtype=s["k"].dtype, device=DEVICE) if s["prompt"] else None
    q = ops.prepare_paged(s["q"], s["k"], s["v"], s["q_norm"], s["k_norm"], s["rope"],
                          s["rotary"], EPS, s["rows"], s["positions"], s["table"],
                          s["k_pages"], s["v_pages"], k_out=k_out)
    return [x for x in (q, k_out, s["k_pages"], s["v_pages"]) if x is not None]


def _own_delta(ops, s):
    KH, kd, H, vd = s["sizes"]
    out = ops.delta_step(s["proj"], s["conv"], s["a_decay"], s["dt_bias"], s["norm"], EPS,
                         s["ring"], s["state"], s["rows"], s["positions"], KH, kd, H, vd)
    return out, s["state"], s["ring"]


def _own_fork(ops, s):
    book = _book(ops, s)
    ops.free_pages(book, s["children"])
    ops.fork_pages(book, s["parents"], s["children"], s["pool"])
    ops.copy_pages(s["states"], s["parents"], s["children"])
    return s["table"], s["lengths"], s["refs"], s["free"][0], s["pool"], s["states"]


def _own_turnover(ops, s):
    book = _book(ops, s)
    old, new, counts = s["turns"][0]
    s["turns"].reverse()
    positions = ops.extend_pages(book, new, counts)
    ops.free_pages(book, old)
    ops.compact_pages(book, s["pool"])
    return positions, s["table"], s["lengths"], s["refs"], s["free"], s["pool"]


_OWN = {"attend": _own_attend, "store": _own_store, "delta": _own_delta, "fork": _own_fork,
        "turnover": _own_turnover}


def _plain_attend(s):
    q, n_keys = s["q"].float(), s["positions"] + 1
    n, H, hd = q.shape
    KV, page = s["k"].shape[1], s["k"].shape[2]
    blocks = s["table"][s["rows"].long()]
    at = torch.arange(blocks.shape[1] * page, device=DEVICE)
    seen = at < n_keys[:, None]                                   # [n, keys]
    index = blocks.clamp(min=0).long()

    def gathered(pages):                                          # [n, KV, keys, hd]
        x = pages[index].transpose(1, 2).reshape(n, KV, at.numel(), hd).float()
        return x.masked_fill(~seen[:, None, :, None], 0.0)

    scores = torch.matmul(q.view(n, KV, H // KV, hd), gathered(s["k"]).transpose(2, 3)) * s["scale"]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights, gathered(s["v"])) / total.clamp(min=1e-30)
    out = out.reshape(n, H, hd) / (1.0 + torch.exp(-s["gate"].float()))
    return out.reshape(n, H * hd).to(s["q"].dtype)


def _plain_norm_rope(x, weight, cos, sin):
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1.0 + weight.float())
    half = cos.shape[-1]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)


def _plain_store(s):
    page, dtype = s["k_pages"].shape[2], s["q"].dtype
    at = s["positions"].long()
    stored = at >= 0
    # a token without a position is normalised, not rotated
    cos = torch.where(stored[:, None], s["rope"][0][at.clamp(min=0)], 1.0)[:, None]
    sin = torch.where(stored[:, None], s["rope"][1][at.clamp(min=0)], 0.0)[:, None]
    q = _plain_norm_rope(s["q"], s["q_norm"], cos, sin).to(dtype)
    k = _plain_norm_rope(s["k"], s["k_norm"], cos, sin).to(dtype)
    keep = stored.nonzero()[:, 0]
    block, place = at[keep] // page, at[keep] % page
    pages = s["table"][s["rows"][keep].long(), block].long()
    s["k_pages"][pages, :, place] = k[keep]
    s["v_pages"][pages, :, place] = s["v"][keep]
    return [x for x in (q, k if s["prompt"] else None, s["k_pages"], s["v_pages"])
            if x is not None]


def _plain_delta(s):
    KH, kd, H, vd = s["sizes"]
    rows, at, n = s["rows"].long(), s["positions"].long(), s["rows"].numel()
    kw, vw = KH * kd, H * vd
    channels = 2 * kw + vw
    proj = s["proj"].float()
    s["ring"][rows, at % TAPS] = s["proj"][:, :channels]
    lag = torch.arange(TAPS, device=DEVICE) + 1 - TAPS            # of each tap, oldest first
    window = s["ring"][rows[:, None], (at[:, None] + lag) % TAPS].float()   # [n, taps, channels]
    window = window.masked_fill((at[:, None] + lag < 0)[..., None], 0.0)
    x = (window * s["conv"].t()).sum(1)
    x = x / (1.0 + torch.exp(-x))
    q, k, v = x[:, :kw].view(n, KH, kd), x[:, kw:2 * kw].view(n, KH, kd), x[:, 2 * kw:].view(n, H, vd)
    q = q / (torch.sqrt(q.square().sum(-1, keepdim=True) + 1e-6) * math.sqrt(kd))
    k = k / torch.sqrt(k.square().sum(-1, keepdim=True) + 1e-6)
    q, k = (t.repeat_interleave(H // KH, 1) for t in (q, k))
    z = proj[:, channels:channels + vw].view(n, H, vd)
    a, b = proj[:, channels + vw:channels + vw + H], proj[:, channels + vw + H:channels + vw + 2 * H]
    beta = 1.0 / (1.0 + torch.exp(-b))
    step = a + s["dt_bias"]
    rate = step.clamp(min=0.0) + torch.log1p(torch.exp(-step.abs()))
    keep = torch.exp(s["a_decay"] * rate)
    state = s["state"][rows] * torch.where(at > 0, 1.0, 0.0)[:, None, None, None]
    state = state * keep[..., None, None]
    u = beta[..., None] * (v - (state * k[:, :, None]).sum(-1))
    state = state + u[..., None] * k[:, :, None]
    s["state"][rows] = state
    o = (state * q[:, :, None]).sum(-1)
    o = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + EPS) * s["norm"].float()
    o = o * (z / (1.0 + torch.exp(-z)))
    return o.reshape(n, vw).to(s["proj"].dtype), s["state"], s["ring"]


def _plain_free(s, rows):
    """Rows in the order given; of the pages left over, the first listed on top."""
    rows = rows.long()
    pages = s["table"][rows].reshape(-1).long()
    pages = pages[pages >= 0]
    s["refs"].index_add_(0, pages, torch.full_like(pages, -1, dtype=torch.int32))
    # a page that several of these rows held counts where it is listed last
    place = torch.arange(pages.numel(), device=DEVICE)
    last = torch.zeros_like(s["refs"], dtype=torch.int64).scatter_reduce_(0, pages, place, "amax")
    left = pages[(s["refs"][pages] == 0) & (last[pages] == place)]
    n = s["free"][0].long()
    s["free"][n + left.numel() - torch.arange(left.numel(), device=DEVICE)] = left.int()
    s["free"][0] += left.numel()
    s["table"][rows] = -1
    s["lengths"][rows] = 0


def _plain_take(s, need):
    """``need[i]`` pages off the stack for entry i, in order: the first page of each
    entry's run, as an index that falls by one a page."""
    first = s["free"][0].long() - (need.cumsum(0) - need)
    s["free"][0] -= need.sum().int()
    return first


def _plain_fork(s):
    parents, children, page = s["parents"].long(), s["children"].long(), s["page"]
    _plain_free(s, s["children"])
    length = s["lengths"][parents].long()
    full, part = length // page, length % page
    block = torch.arange(s["table"].shape[1], device=DEVICE)
    source = s["table"][parents]
    shared = block < full[:, None]
    s["refs"].index_add_(0, source[shared].long(), torch.ones_like(source[shared]))
    begun = part > 0
    first = _plain_take(s, begun.long())
    new = s["free"][first.clamp(min=0)]
    s["refs"][new[begun].long()] = 1
    s["table"][children] = torch.where(shared, source, -1)
    s["table"][children[begun], full[begun]] = new[begun]
    s["lengths"][children] = length.int()
    old = source.gather(1, full.clamp(max=block.numel() - 1)[:, None])[:, 0]
    src, dst = old[begun].long(), new[begun].long()
    used = torch.arange(page, device=DEVICE) < part[begun][:, None]
    s["pool"][:, dst] = torch.where(used[:, None, :, None], s["pool"][:, src], s["pool"][:, dst])
    s["states"][:, children] = s["states"][:, parents]
    return s["table"], s["lengths"], s["refs"], s["free"][0], s["pool"], s["states"]


def _plain_turnover(s):
    old, new, counts = s["turns"][0]
    s["turns"].reverse()
    page, rows = s["page"], new.long()
    positions = s["lengths"][rows]
    have, want = -(-positions // page), -(-(positions + counts) // page)
    first = _plain_take(s, (want - have).long())
    block = torch.arange(s["table"].shape[1], device=DEVICE)
    fresh = (block >= have[:, None]) & (block < want[:, None])
    pages = s["free"][(first[:, None] - (block - have[:, None])).clamp(min=0)]
    s["table"][rows] = torch.where(fresh, pages, s["table"][rows])
    s["refs"][pages[fresh].long()] = 1
    s["lengths"][rows] = positions + counts
    _plain_free(s, old)
    # the k-th hole among the low pages takes the k-th page above them
    live = s["refs"] > 0
    n = int(live.sum())
    holes, movers = (~live[:n]).nonzero()[:, 0], live[n:].nonzero()[:, 0] + n
    moved = torch.arange(live.numel(), device=DEVICE)
    moved[movers] = holes
    s["pool"][:, holes] = s["pool"][:, movers]
    s["table"].copy_(torch.where(s["table"] >= 0, moved[s["table"].clamp(min=0).long()].int(), -1))
    s["refs"][holes] = s["refs"][movers]
    s["refs"][n:] = 0
    s["free"].zero_()
    s["free"][0] = live.numel() - n
    s["free"][1:1 + live.numel() - n] = torch.arange(live.numel() - 1, n - 1, -1, device=DEVICE).int()
    return positions, s["table"], s["lengths"], s["refs"], s["free"], s["pool"]


_PLAIN = {"attend": _plain_attend, "store": _plain_store, "delta": _plain_delta,
          "fork": _plain_fork, "turnover": _plain_turnover}


# --------------------------------------------------------------- yardsticks --
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    kind = case["kind"]
    if kind == "attend":
        H, KV, hd, _ = HEADS[case["heads"]]
        keys = int(_sizes(case, case["rows"]).sum())
        return {"bytes": 2 * keys * KV * hd * size + 3 * case["rows"] * H * hd * size,
                "flops": 4 * keys * H * hd}
    if kind == "store":
        H, KV, hd, _ = HEADS[case["heads"]]
        T = case["rows"] * case["tokens"]
        kept = 5 / 6 if case["tokens"] > 1 else 1.0        # of a prompt, what is not padding
        rows = T * (2 * H + KV + (KV if case["tokens"] > 1 else 0)) + kept * T * 3 * KV
        return {"bytes": rows * hd * size, "flops": 8 * T * (H + KV) * hd}
    if kind == "delta":
        KH, H, kd, vd = DELTA[case["heads"]]
        n, channels = case["rows"], 2 * KH * kd + H * vd
        return {"bytes": n * (2 * H * kd * vd * 4 + (channels * (TAPS + 1) + 2 * H * vd) * size)
                + channels * TAPS * 4, "flops": 7 * n * H * kd * vd}
    _, KV, hd, _ = HEADS[case["heads"]]
    token = 2 * case["layers"] * KV * hd * size
    if kind == "fork":
        KH, H, kd, vd = DELTA["decision" if hd == 64 else "0.8b"]
        kids = case["parents"] * case["each"]
        states = case["states"] * H * kd * vd * 4
        begun = int((_sizes(case, case["parents"]) % case["page"]).sum())
        # a parent's data read once, each child's written
        return {"bytes": (kids + case["parents"]) * states + (1 + case["each"]) * begun * token,
                "flops": 0}
    # the rows that come lie above all that is freed below them
    blocks = int((-(-_sizes(case, case["rows"]) // case["page"])).sum())
    return {"bytes": 2 * blocks * case["page"] * token, "flops": 0}


# ---------------------------------------------------------- 64-bit reference --
def exact(case, seed):
    return _EXACT[case["kind"]](prepare(case, seed))


def _exact_attend(s):
    n, H, hd = s["q"].shape
    KV, page = s["k"].shape[1], s["k"].shape[2]
    out = torch.zeros(n, H, hd, dtype=torch.float64, device=DEVICE)
    gate = torch.sigmoid(s["gate"].double())
    for i, (row, last) in enumerate(zip(s["rows"].tolist(), s["positions"].tolist())):
        if last < 0:
            continue
        pages = s["table"][row, :last // page + 1].long()
        for g in range(KV):
            k, v = (x[pages, g].reshape(-1, hd)[:last + 1].double() for x in (s["k"], s["v"]))
            heads = slice(g * (H // KV), (g + 1) * (H // KV))
            scores = (k @ s["q"][i, heads].double().t().contiguous()).t() * s["scale"]
            out[i, heads] = torch.softmax(scores, -1) @ v
    return (out * gate).reshape(n, H * hd)


def _exact_store(s):
    page = s["k_pages"].shape[2]
    places = s["positions"].tolist()
    at = s["positions"].double().clamp(min=0).long()
    turned = (s["positions"] >= 0).double()[:, None, None]

    def heads(x, weight):
        x = x.double()
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * (1 + weight.double())
        cos, sin = (t.double()[at][:, None] for t in s["rope"])
        half = cos.shape[-1]
        y = x.clone()
        y[..., :half] = x[..., :half] * cos - x[..., half:2 * half] * sin
        y[..., half:2 * half] = x[..., half:2 * half] * cos + x[..., :half] * sin
        return y * turned + x * (1 - turned)

    q, k = heads(s["q"], s["q_norm"]), heads(s["k"], s["k_norm"])
    table = s["table"].cpu().numpy()
    keep = [t for t, p in enumerate(places) if p >= 0]
    rows = s["rows"].tolist()
    page_of = [int(table[rows[t], places[t] // page]) for t in keep]
    place = [places[t] % page for t in keep]
    keys, values = s["k_pages"].double(), s["v_pages"].double()
    keys[page_of, :, place] = k[keep]
    values[page_of, :, place] = s["v"].double()[keep]
    return [x for x in (q, k if s["prompt"] else None, keys, values) if x is not None]


def _exact_delta(s):
    KH, kd, H, vd = s["sizes"]
    rows, at = s["rows"].tolist(), s["positions"].tolist()
    kw, vw = KH * kd, H * vd
    channels = 2 * kw + vw
    proj, ring, state = s["proj"].double(), s["ring"].double(), s["state"].double()
    out = torch.empty(len(rows), H, vd, dtype=torch.float64, device=DEVICE)
    for i, (row, p) in enumerate(zip(rows, at)):
        ring[row, p % TAPS] = proj[i, :channels]
        x = sum(ring[row, (p - j) % TAPS] * s["conv"][:, TAPS - 1 - j].double()
                for j in range(min(TAPS, p + 1)))
        x = torch.nn.functional.silu(x)
        q, k, v = x[:kw].view(KH, kd), x[kw:2 * kw].view(KH, kd), x[2 * kw:].view(H, vd)
        q = q / ((q * q).sum(-1, keepdim=True) + 1e-6).sqrt() / math.sqrt(kd)
        k = k / ((k * k).sum(-1, keepdim=True) + 1e-6).sqrt()
        of = torch.arange(H, device=DEVICE) // (H // KH)
        q, k = q[of], k[of]
        tail = proj[i, channels:]
        z, a, b = tail[:vw].view(H, vd), tail[vw:vw + H], tail[vw + H:vw + 2 * H]
        rate = torch.nn.functional.softplus(a + s["dt_bias"].double(), threshold=100.0)
        S = state[row] * torch.exp(s["a_decay"].double() * rate)[:, None, None] if p else \
            torch.zeros_like(state[row])
        u = torch.sigmoid(b)[:, None] * (v - (S * k[:, None]).sum(-1))
        S = S + u[:, :, None] * k[:, None, :]
        state[row] = S
        o = (S * q[:, None]).sum(-1)
        o = o / torch.sqrt((o * o).mean(-1, keepdim=True) + EPS) * s["norm"].double()
        out[i] = o * torch.nn.functional.silu(z)
    return out.reshape(len(rows), vw), state, ring


def _exact_fork(s):
    """Only the copies have values of their own; the whole numbers are compared as
    they are."""
    page, pool, states = s["page"], s["pool"], s["states"].double()
    free, lengths, table = (s[x].tolist() for x in ("free", "lengths", "table"))
    top = free[0]
    pool = pool.double()
    for p, c in zip(s["parents"].tolist(), s["children"].tolist()):
        states[:, c] = states[:, p]
        if lengths[p] % page:
            pool[:, free[top], :, :lengths[p] % page] = \
                pool[:, table[p][lengths[p] // page], :, :lengths[p] % page].clone()
            top -= 1
    return None, None, None, None, pool, states


def _exact_turnover(s):
    page, free, table = s["page"], s["free"].tolist(), s["table"].tolist()
    old, new, counts = (x.tolist() for x in s["turns"][0])
    lengths, top = s["lengths"].tolist(), free[0]
    refs = s["refs"].tolist()
    for row, count in zip(new, counts):
        for j in range(-(-lengths[row] // page), -(-(lengths[row] + count) // page)):
            refs[free[top]] += 1
            top -= 1
    for row in old:
        for p in table[row]:
            if p >= 0:
                refs[p] -= 1
    live = [p for p, r in enumerate(refs) if r]
    holes = [p for p in range(len(live)) if not refs[p]]
    movers = [p for p in live if p >= len(live)]
    pool = s["pool"].double()
    pool[:, holes] = pool[:, movers]
    return None, None, None, None, None, pool


_EXACT = {"attend": _exact_attend, "store": _exact_store, "delta": _exact_delta,
          "fork": _exact_fork, "turnover": _exact_turnover}
