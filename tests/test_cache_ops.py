"""The operators of a cache that the backbone decodes from (include/qdc_hip_cache.h,
qdc_amd.cache_ops): their argument checks, which need no GPU, and each against a plain
form in 64 bits, at the lengths, pages, masks and rows where they can go wrong."""
import math
import os
import re

import numpy as np
import pytest
import torch

from conftest import ROOT, normwise
from qdc_amd import _lib, cache_ops, ops

F32, BF16, X2 = _lib.QDC_F32, _lib.QDC_BF16, _lib.QDC_BF16X2
FAKE, FAR = 0x10000, 1 << 56  # aligned addresses never dereferenced by validation
DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}  # half a step, relative


# ---------------------------------------------------------- argument checks --
def test_exports_match_header():
    text = open(os.path.join(ROOT, "include", "qdc_hip_cache.h")).read()
    names = set(re.findall(r"^\s*(?:const\s+)?\w+\s*\*?\s*(qdc_\w+)\s*\(", text, re.M))
    assert names == set(_lib.CACHE_SIGNATURES)
    for name in names:
        assert hasattr(_lib.lib(), name), name
    version = re.search(r'#define\s+QDC_HIP_CACHE_VERSION\s+"([^"]+)"', text).group(1)
    assert _lib.lib().qdc_cache_version().decode() == version


def test_prepare_paged_validation():
    names = ("q_out", "k_out", "k_pages", "v_pages", "q", "k", "v", "q_norm", "k_norm", "cos",
             "sin", "index", "positions", "table")

    def f(dtype=BF16, tokens=4, heads=4, kv=2, hd=64, rd=16, tlen=100, rows=3, width=5, pages=7,
          page=16, q_tok=256, q_head=64, k_tok=128, k_head=64, v_tok=128, v_head=64, flag=None,
          **at):
        ptr = [at.get(n, FAR + (i << 40)) for i, n in enumerate(names)]
        return _lib.lib().qdc_prepare_paged(*ptr, tokens, heads, kv, hd, rd, tlen, rows, width,
                                            pages, page, q_tok, q_head, k_tok, k_head, v_tok,
                                            v_head, 1e-6, dtype, flag, None)

    assert f(dtype=X2) == -3
    assert f(hd=96) == -2 and f(page=8) == -2 and f(page=24) == -2 and f(page=512) == -2
    assert f(rd=15) == -2 and f(rd=66) == -2 and f(heads=0) == -2 and f(kv=0) == -2
    assert f(rows=0) == -2 and f(width=0) == -2 and f(pages=0) == -2 and f(tokens=-1) == -2
    assert f(q_head=32) == -2 and f(k_tok=132) == -2 and f(v_head=68) == -2 and f(q_tok=-8) == -2
    assert f(tokens=1 << 24) == -2                  # grid
    for n in names:
        if n != "k_out":
            assert f(**{n: 0}) == -1, n
    for n in ("q", "k_out", "v_pages", "cos"):
        assert f(**{n: FAR + 8}) == -2, n
    assert f(q=FAR + 64) == -5 and f(k_out=FAR + 64) == -5       # over q_out
    assert f(flag=FAR + (2 << 40)) == -5                         # the flag in a page
    assert f(tokens=0, q=0) == 0


def test_paged_attention_validation():
    names = ("q", "k", "v", "gate", "table", "index", "positions")
    size = _lib.lib().qdc_paged_attention_workspace
    need = size(3, 8, 2, 128, 500, 16, BF16)
    assert need > 0 and size(3, 8, 2, 128, 5, 16, BF16) == 0     # short rows need none
    assert size(3, 8, 3, 128, 5, 16, BF16) == -1 and size(3, 8, 2, 96, 5, 16, BF16) == -1
    assert size(3, 8, 2, 128, 5, 20, BF16) == -1 and size(3, 8, 2, 128, 5, 16, X2) == -1
    assert size(1 << 24, 8, 2, 128, 5, 16, BF16) == -1           # the join's grid
    assert size(1 << 15, 8, 2, 128, 1 << 20, 256, BF16) == -1    # tiles past 31 bits

    def f(dtype=BF16, odt=BF16, n=3, heads=8, kv=2, hd=128, rows=4, width=500, pages=7, page=16,
          q_tok=1024, q_head=128, g_tok=1024, g_head=128, o_tok=1024, scale=0.1, ws=FAR + (9 << 40),
          nbytes=need, out=FAR + (8 << 40), flag=None, **at):
        ptr = [at.get(x, FAR + (i << 40)) for i, x in enumerate(names)]
        return _lib.lib().qdc_paged_attention(out, odt, *ptr, n, heads, kv, hd, rows, width, pages,
                                              page, q_tok, q_head, g_tok, g_head, o_tok, scale,
                                              dtype, ws, nbytes, flag, None)

    assert f(dtype=X2) == -3 and f(odt=9) == -3
    assert f(heads=7) == -2 and f(hd=96) == -2 and f(page=12) == -2 and f(rows=0) == -2
    assert f(pages=0) == -2 and f(width=0) == -2 and f(n=-1) == -2
    assert f(q_head=64) == -2 and f(q_tok=1028) == -2 and f(g_head=120) == -2
    assert f(o_tok=1016) == -2 and f(o_tok=1028) == -2
    assert f(scale=0.0) == -4 and f(scale=-1.0) == -4 and f(scale=float("inf")) == -4
    assert f(scale=float("nan")) == -4 and f(scale=3e38) == -4
    for x in ("q", "k", "v", "table", "index", "positions"):
        assert f(**{x: 0}) == -1, x
    assert f(out=0) == -1 and f(ws=0) == -1
    assert f(q=FAR + 8) == -2 and f(gate=FAR + 4) == -2 and f(ws=FAR + (9 << 40) + 8) == -2
    assert f(nbytes=need - 1) == -2
    assert f(out=FAR + (1 << 40)) == -5 and f(ws=FAR + (8 << 40)) == -5
    assert f(n=0, q=0) == 0 and f(width=5, ws=0, nbytes=0, q=0) == -1


def test_pages_validation():
    lib = _lib.lib()
    T, L, R, S = (FAR + (i << 40) for i in range(4))
    I, P, W, POOL = (FAR + (i << 40) for i in range(4, 8))

    def ext(pos=P, table=T, n=4, rows=5, width=6, pages=7, page=16, index=I, counts=None):
        return lib.qdc_pages_extend(pos, table, L, R, S, index, counts, n, rows, width, pages, page,
                                    None, None)

    for bad in (dict(n=-1), dict(rows=0), dict(rows=1 << 18), dict(width=0), dict(pages=0),
                dict(page=17), dict(n=1 << 24), dict(width=1 << 28, page=256)):
        assert ext(**bad) == -2, bad
    assert ext(pos=None) == -1 and ext(table=None) == -1 and ext(index=None) == -1
    assert ext(pos=T + 4) == -5 and ext(index=L) == -5 and ext(counts=P + 8) == -5
    assert ext(n=0, table=None, index=None, pos=None) == 0
    free = lambda index=I, n=4, page=16: lib.qdc_pages_free(T, L, R, S, index, n, 5, 6, 7, page,  # noqa: E731
                                                            None, None)
    assert free(index=None) == -1 and free(index=R) == -5 and free(page=1) == -2
    assert free(n=0, index=None) == 0

    assert lib.qdc_pages_fork_workspace(4, 16, 2, 2, 128) == 0         # little to copy
    assert lib.qdc_pages_fork_workspace(4, 16, 2, 2, 8192) == 64
    assert lib.qdc_pages_fork_workspace(1025, 16, 1, 1, 16) == 16400
    assert lib.qdc_pages_fork_workspace(5000, 16, 0, 0, 0) == 0

    def fork(par=I, ch=P, n=4, pool=POOL, planes=2, heads=2, token=8192, ws=W, nbytes=64):
        return lib.qdc_pages_fork(T, L, R, S, par, ch, n, 5, 6, 7, 16, pool, planes, heads, token,
                                  ws, nbytes, None, None)

    assert fork(token=120) == -2 and fork(token=0) == -2 and fork(heads=0) == -2
    assert fork(planes=-1) == -2 and fork(planes=1 << 16) == -2 and fork(nbytes=63) == -2
    assert fork(ws=W + 4) == -2 and fork(pool=POOL + 4) == -2 and fork(planes=1 << 14, heads=4) == -2
    assert fork(token=1 << 20) == -2 and fork(n=4000, planes=600, nbytes=1 << 20) == -2
    assert fork(par=None) == -1 and fork(pool=None) == -1 and fork(ws=None) == -1
    assert fork(ws=POOL) == -5 and fork(ch=T) == -5 and fork(n=0, par=None) == 0
    assert fork(token=128, ws=None, nbytes=0, ch=None) == -1

    def compact(table=T, pool=POOL, planes=2, nbytes=4096, pages=7, ws=W, have=100):
        return lib.qdc_pages_compact(table, R, S, 5, 6, pages, pool, planes, nbytes, ws, have, None)

    assert lib.qdc_pages_compact_workspace(7) == 100 and lib.qdc_pages_compact_workspace(0) == 0
    assert compact(pages=0) == -2 and compact(nbytes=4100) == -2 and compact(have=99) == -2
    assert compact(planes=1 << 16) == -2 and compact(ws=W + 8) == -2
    assert compact(table=None) == -1 and compact(pool=None) == -1 and compact(ws=None) == -1
    assert compact(ws=POOL + 16) == -5 and compact(pool=T) == -5

    def copy(pool=POOL, src=I, dst=P, n=4, planes=2, items=7, nbytes=64):
        return lib.qdc_copy_pages(pool, src, dst, n, planes, items, nbytes, None, None)

    assert copy(n=-1) == -2 and copy(n=4097) == -2 and copy(nbytes=8) == -2
    assert copy(items=0) == -2 and copy(pool=POOL + 4) == -2
    assert copy(planes=60000, items=1 << 30, nbytes=1 << 30) == -2 and copy(planes=1 << 16) == -2
    assert copy(pool=None) == -1 and copy(src=None) == -1 and copy(src=POOL + 16) == -5
    assert copy(n=0, pool=None) == 0 and copy(planes=0, pool=None) == 0
    # grids of 2^32 work-items: 4 KB a workgroup of 256, 64 KB and more one of 1024
    assert copy(n=4096, planes=4096, nbytes=4096) == -2
    assert copy(n=4096, planes=1024, nbytes=65536) == -2


def test_pages_largest_counts():
    """Lists of pages are walked 1024 at a time in 32 bits: the sizes that a step past their
    end would leave are refused, the last before them are taken (by what each refuses next:
    a missing index or workspace)."""
    lib, most = _lib.lib(), 2 ** 31 - 1024
    T, L, R, S, W = (FAR << i for i in range(5))
    wide = 2 ** 27 - 1                      # 16 rows of it are 2^31 - 16 places

    def calls(rows, width, pages):
        at = (T, L, R, S)
        size = (rows, width, pages, 16)
        return (lib.qdc_pages_extend(FAKE, *at, None, None, 4, *size, None, None),
                lib.qdc_pages_free(*at, None, 4, *size, None, None),
                lib.qdc_pages_fork(*at, None, None, 4, *size, None, 0, 0, 0, None, 0, None, None))

    assert calls(5, 6, most) == calls(15, wide, 7) == (-1, -1, -1)
    for bad in ((5, 6, most + 1), (5, 6, 2 ** 31 - 2), (16, wide, 7)):
        assert calls(*bad) == (-2, -2, -2), bad
    need = lib.qdc_pages_compact_workspace(most)
    assert need == 16 + 12 * most and lib.qdc_pages_compact_workspace(most + 1) == 0
    compact = lambda pages, nbytes: lib.qdc_pages_compact(T, R, S, 5, 6, pages, None, 0, 0, None,  # noqa: E731
                                                          nbytes, None)
    assert compact(most, need) == -1 and compact(most + 1, 1 << 40) == -2


def test_page_table_limits():
    """A table that the operators would refuse at every call is not made."""
    for rows, width, pages, page in ((2 ** 18, 1, 1, 16), (1, 2 ** 23, 1, 256), (1, 2 ** 27, 1, 16),
                                     (1, 1, 2 ** 31 - 1023, 16), (2 ** 17, 2 ** 14, 1, 16)):
        with pytest.raises(ValueError, match="too many rows"):
            cache_ops.page_table(rows, width, pages, page, "meta")
    for rows, width, pages, page in ((2 ** 18 - 1, 1, 1, 16), (1, 2 ** 23 - 1, 1, 256),
                                     (1, 1, 2 ** 31 - 1024, 16), (2 ** 17, 2 ** 14 - 1, 1, 16)):
        assert cache_ops.page_table(rows, width, pages, page, "meta").table.shape == (rows, width)


def test_delta_step_validation():
    names = ("proj", "conv", "a_decay", "dt_bias", "norm", "ring", "state", "index", "positions")

    def f(odt=BF16, dt=BF16, ld=1024, taps=4, n=3, rows=5, kh=2, kd=64, vh=4, vd=32,
          out=FAR + (12 << 40), flag=None, **at):
        p = {x: at.get(x, FAR + (i << 40)) for i, x in enumerate(names)}
        return _lib.lib().qdc_delta_step(out, odt, p["proj"], dt, ld, p["conv"], taps, p["a_decay"],
                                         p["dt_bias"], p["norm"], p["ring"], p["state"],
                                         p["index"], p["positions"], n, rows, kh, kd, vh, vd, 1e-6,
                                         flag, None)

    assert f(dt=X2) == -3 and f(odt=F32) == -3 and f(odt=X2, dt=F32) == -3
    assert f(kd=96) == -2 and f(vd=24) == -2 and f(vd=272) == -2 and f(vh=3) == -2
    assert f(taps=0) == -2 and f(taps=9) == -2 and f(rows=0) == -2 and f(n=-1) == -2
    assert f(ld=2 * 128 + 128 + 128 + 7) == -2 and f(n=1 << 22) == -2
    assert f(n=1 << 20) == -2           # a workgroup of 1024 for each of its 4 heads: 2^32 threads
    for x in names:
        assert f(**{x: 0}) == -1, x
    assert f(out=0) == -1 and f(state=FAR + 4) == -2
    assert f(out=FAR + 16) == -5 and f(ring=FAR + (6 << 40)) == -5
    assert f(flag=FAR + (6 << 40)) == -5 and f(n=0, proj=0) == 0


def test_delta_scan_state_validation():
    need = _lib.lib().qdc_delta_scan_workspace(2, 33, 4, 64, 32)

    def f(state=FAR + (3 << 40), ws=FAR + (2 << 40), out=FAR + (1 << 40)):
        return _lib.lib().qdc_delta_scan_state(out, F32, state, FAR, FAR, FAR, FAR, FAR, 2, 33, 4, 2,
                                               64, 32, 128, 128, ws, need, None)

    assert f(state=None) == -1 and f(state=FAR + 8) == -2 and f(state=FAR + 16) == -5
    assert f(state=FAR + (2 << 40)) == -5 and f(state=FAR + (1 << 40) - 16) == -5


def test_host_tensors_are_refused():
    """Every operator needs device tensors, and a page table's are checked together."""
    z = lambda *s, dt=torch.float32: torch.zeros(s, dtype=dt)  # noqa: E731
    i = z(2, dt=torch.int32)
    book = cache_ops.page_table(2, 3, 4, 16, "cpu")
    assert book.free.tolist() == [4, 3, 2, 1, 0]
    calls = [lambda: cache_ops.prepare_paged(z(2, 4, 64), z(2, 2, 64), z(2, 2, 64), z(64), z(64),
                                             None, 0, 1e-6, i, i, book.table, z(4, 2, 16, 64),
                                             z(4, 2, 16, 64)),
             lambda: cache_ops.paged_attention(z(2, 4, 64), z(4, 2, 16, 64), z(4, 2, 16, 64),
                                               book.table, i, i, 0.1),
             lambda: cache_ops.extend_pages(book, i), lambda: cache_ops.free_pages(book, i),
             lambda: cache_ops.fork_pages(book, i, i), lambda: cache_ops.compact_pages(book),
             lambda: cache_ops.copy_pages(z(1, 4, 16), i, i),
             lambda: cache_ops.delta_step(z(2, 600), z(384, 4), z(4), z(4), z(32), 1e-6,
                                          z(2, 4, 384), z(2, 4, 32, 64), i, i, 2, 64, 4, 32)]
    for call in calls:
        with pytest.raises(ValueError, match="device tensors required"):
            call()
    for bad in ((0, 1, 1, 16), (1, 0, 1, 16), (1, 1, 0, 16), (1, 1, 1, 24)):
        with pytest.raises(ValueError):
            cache_ops.page_table(*bad, "cpu")
    for call in (lambda: cache_ops.copy_pages([1.0], i, i), lambda: cache_ops.free_pages((i, 2, 3, 4, 5), i),
                 lambda: cache_ops.delta_step(z(2, 600), z(384, 4), z(4), z(4), z(32), 1e-6,
                                              z(2, 4, 384), z(2, 4, 32, 64), i, i, 2.5, 64, 4, 32),
                 lambda: cache_ops.paged_attention(None, i, i, i, i, i, 0.1)):
        with pytest.raises((TypeError, ValueError)):      # no tensor, no integer
            call()
    with pytest.raises(ValueError, match="split output"):
        cache_ops.delta_step(z(2, 600), z(384, 4), z(4), z(4), z(32), 1e-6, z(2, 4, 384),
                             z(2, 4, 32, 64), i, i, 2, 64, 4, 32, out_dtype=ops.BF16X2)


# ------------------------------------------------------------------ helpers --
def ints(values):
    return torch.tensor(np.asarray(values, np.int32).reshape(-1), device=DEV)


def flag():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def scattered(rng, lengths, page, spare=2, width=None):
    """A table whose rows' pages lie anywhere among ``pages``."""
    blocks = [-(-n // page) for n in lengths]
    pages = sum(blocks) + spare
    table = np.full((len(lengths), width or max(1, *blocks)), -1, np.int32)
    order = iter(rng.permutation(pages))
    for row, b in zip(table, blocks):
        row[:b] = [next(order) for _ in range(b)]
    return table, pages


# ------------------------------------------------------------ prepare_paged --
# heads, KV heads, head size, rotated values (none, all, halves that are no whole
# 16-byte piece), page size
PREPARE = [(4, 2, 64, 16, 16), (1, 1, 64, 0, 32), (3, 1, 64, 6, 16), (8, 2, 256, 64, 64),
           (6, 6, 128, 128, 16), (2, 1, 256, 20, 256), (5, 5, 128, 24, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,hd,rd,page", PREPARE)
@pytest.mark.parametrize("T", [1, 37])
def test_prepare_paged(T, H, KV, hd, rd, page, dtype):
    """Against 64 bits.  fp32: the sum of squares is off by at most head_dim half
    steps, its root and the products by a few, and a rotated value is a sum of two
    such: (head_dim + 16) 2^-24 of the row's largest value.  bf16 adds its own half
    step.  What is not stored is left as it was, bit for bit."""
    rng = np.random.default_rng(T * 1000 + H * 100 + hd + rd)
    rows, reach = 3, 150
    table, pages = scattered(rng, [reach] * rows, page)
    # distinct places; some entries no token, in each of the ways
    places = rng.permutation(rows * reach)[:T]
    index, pos = places // reach, places % reach
    if T > 9:
        pos[3], index[5] = -1, -1
        index[6] = rows                               # no row of the cache
        pos[7] = table.shape[1] * page                # behind the table
        gone = (int(index[8]), int(pos[8]) // page)
        table[gone] = pages                           # no page
    t = lambda *s: torch.from_numpy(rng.standard_normal(s, dtype=np.float32)).to(dtype)  # noqa: E731
    qg, kv = t(T, H, 2, hd), t(T, 2, KV + 1, hd)      # q beside a gate, k and v in wider rows
    qn, kn = t(hd) * 0.1, t(hd) * 0.1
    old = torch.full((2, pages, KV, page, hd), float("nan"), dtype=dtype)
    tables = ops.rope_tables(max(1, table.shape[1] * page), rd, 1e4, DEV) if rd else None
    d = lambda x: x.to(DEV)  # noqa: E731
    qd, kvd, store, f = d(qg), d(kv), d(old), flag()
    k_out = torch.empty((T, KV, hd), dtype=dtype, device=DEV) if T > 1 else None
    got_q = cache_ops.prepare_paged(qd[:, :, 0], kvd[:, 0, :KV], kvd[:, 1, 1:], d(qn), d(kn), tables,
                                    rd, 1e-6, ints(index), ints(pos), d(torch.from_numpy(table)),
                                    store[0], store[1], k_out=k_out, error_flag=f)

    live = [index[i] >= 0 and 0 <= pos[i] < table.shape[1] * page and index[i] < rows
            and table[index[i], pos[i] // page] < pages for i in range(T)]
    at = np.where(live, pos, 0)

    def expect(x, w):
        x, w = x.double(), w.double()
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (1 + w)
        top = x.abs().amax(-1, keepdim=True)
        if rd:
            cos, sin = (c.double().cpu()[at][:, None] for c in tables)
            keep = torch.tensor(live)[:, None, None]
            cos, sin = torch.where(keep, cos, 1.0), torch.where(keep, sin, 0.0)
            a, b = x[..., :rd // 2], x[..., rd // 2:rd]
            x = torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rd:]], -1)
        tol = (hd + 16) * 2.0 ** -24 * top
        return x, tol if dtype == torch.float32 else tol + HALF[dtype] * x.abs()

    def near(got, pair):
        exp, tol = pair
        assert ((got.double().cpu() - exp).abs() <= tol).all()

    near(got_q, expect(qg[:, :, 0], qn))
    k = expect(kv[:, 0, :KV], kn)
    if k_out is not None:
        near(k_out, k)
    got = store.cpu()
    touched = torch.zeros(pages, page, dtype=torch.bool)
    for i in range(T):
        if live[i]:
            p, o = int(table[index[i], pos[i] // page]), int(pos[i]) % page
            touched[p, o] = True
            near(got[0, p, :, o], (k[0][i], k[1][i]))
            assert torch.equal(got[1, p, :, o], kv[i, 1, 1:])
    assert torch.isnan(got.float()[:, ~touched.unsqueeze(1).expand(pages, KV, page)]).all()
    bad = T > 9
    assert f.item() == int(bad)


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,KV,hd,rd,dtype", [
    (8209, 8, 2, 256, 64, torch.bfloat16),     # from 32 MB of bf16 queries on four heads at a time
    (2731, 24, 3, 256, 32, torch.bfloat16),
    (11003, 12, 4, 128, 128, torch.bfloat16),
    (43691, 6, 1, 64, 0, torch.bfloat16),      # no multiple of four: two
    (10923, 6, 2, 128, 16, torch.float32)])
def test_prepare_paged_many_tokens(T, H, KV, hd, rd, dtype):
    """As above with the tolerance of above, for prompts of tens of MB."""
    assert T * H * hd * dtype.itemsize >= 32 << 20
    g = torch.Generator(device=DEV).manual_seed(T)
    page, rows = 32, 7
    reach = -(-T // rows)
    table, pages = scattered(np.random.default_rng(T), [reach] * rows, page)
    table = torch.from_numpy(table).to(DEV)
    t = lambda *s: torch.randn(s, generator=g, device=DEV).to(dtype)  # noqa: E731
    qg, kv, qn, kn = t(T, H, 2, hd), t(T, 2, KV, hd), t(hd) * 0.1, t(hd) * 0.1
    place = torch.randperm(T, generator=g, device=DEV)
    index, pos = (place // reach).int(), (place % reach).int()
    pos[7::1000], index[9::1000] = -1, -1
    live = (index >= 0) & (pos >= 0)
    tables = ops.rope_tables(reach, rd, 1e4, DEV) if rd else None
    store = torch.full((2, pages, KV, page, hd), float("nan"), dtype=dtype, device=DEV)
    k_out, f = torch.empty((T, KV, hd), dtype=dtype, device=DEV), flag()
    got = cache_ops.prepare_paged(qg[:, :, 0], kv[:, 0], kv[:, 1], qn, kn, tables, rd, 1e-6, index, pos,
                                  table, store[0], store[1], k_out=k_out, error_flag=f)

    def near(got, x, w):
        x = x.double()
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (1 + w.double())
        tol = (hd + 16) * 2.0 ** -24 * x.abs().amax(-1, keepdim=True)
        if rd:
            keep = live[:, None, None]
            cos, sin = (c.double()[torch.where(live, pos, 0).long()][:, None] for c in tables)
            cos, sin = torch.where(keep, cos, 1.0), torch.where(keep, sin, 0.0)
            a, b = x[..., :rd // 2], x[..., rd // 2:rd]
            x = torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rd:]], -1)
        if dtype == torch.bfloat16:
            tol = tol + HALF[dtype] * x.abs()
        assert ((got.double() - x).abs() <= tol).all()

    near(got, qg[:, :, 0], qn)
    near(k_out, kv[:, 0], kn)
    assert f.item() == 0
    at, row = pos[live].long(), index[live].long()
    p, o = table[row, at // page].long(), at % page
    assert torch.equal(store[0, p, :, o], k_out[live]) and torch.equal(store[1, p, :, o], kv[live, 1])
    store[:, p, :, o] = float("nan")
    assert torch.isnan(store).all()


@pytest.mark.gpu
def test_prepare_paged_refusals():
    z = lambda *s, dt=torch.float32: torch.zeros(s, dtype=dt, device=DEV)  # noqa: E731
    i, q, k, n, pg = ints([0, 1]), z(2, 4, 64), z(2, 2, 64), z(64), z(4, 2, 16, 64)
    table = z(2, 3, dt=torch.int32)
    ok = dict(q=q, k=k, v=k.clone(), q_norm=n, k_norm=n, tables=None, rotary_dim=0, eps=1e-6,
              rows=i, positions=i, table=table, k_pages=pg, v_pages=pg.clone())
    cache_ops.prepare_paged(**ok)
    empty = dict(ok, q=q[:0], k=k[:0], v=k[:0], rows=i[:0], positions=i[:0])
    assert cache_ops.prepare_paged(**empty).shape == (0, 4, 64)
    for bad in (dict(q=q[:1]), dict(v=z(2, 1, 64)), dict(q=q.bfloat16()), dict(q_norm=z(32)),
                dict(rows=i.long()), dict(positions=ints([0])), dict(table=table.float()),
                dict(k_pages=z(4, 1, 16, 64)), dict(v_pages=pg.bfloat16()),
                dict(k_pages=pg.transpose(0, 1)), dict(rotary_dim=16),
                dict(q=z(2, 4, 96), k=z(2, 2, 96), v=z(2, 2, 96), q_norm=z(96), k_norm=z(96),
                     k_pages=z(4, 2, 16, 96), v_pages=z(4, 2, 16, 96)),
                dict(k_pages=z(4, 2, 24, 64), v_pages=z(4, 2, 24, 64)),
                dict(q_out=q), dict(k_out=z(2, 2, 64, dt=torch.bfloat16)), dict(v_pages=pg),
                dict(error_flag=z(1)), dict(error_flag=torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(ValueError):
            cache_ops.prepare_paged(**dict(ok, **bad))


# ---------------------------------------------------------- paged_attention --
def attend_exact(q, k, v, table, index, pos, scale, gate, page):
    """64 bits, and per element what the result may differ by before its own rounding.

    A score is a sum of head_dim fp32 products and a multiply: off by at most
    (head_dim + 2) 2^-24 of scale sum |q k|, and the exponent taken from it by 2 steps
    of its own size; a weight exp() of that by as much relatively, with 4 half steps of
    the exponential; sums of n weights and products by 2 n half steps at worst, in
    chains of a tile's and of the tiles' lengths, n <= 2 (32 + tiles); the two terms of
    a weight are 2^-16 off (the first is cut to 8 bits, the rest below 2^-7 of it rounded to
    8 bits).  All of it times the weighted mean of |v|."""
    n, H, hd = q.shape
    KV = k.shape[1]
    out, tol = torch.zeros(n, H, hd, dtype=torch.float64), torch.zeros(n, H, hd, dtype=torch.float64)
    for i in range(n):
        if index[i] < 0 or pos[i] < 0 or index[i] >= len(table):
            continue
        places = [(int(table[index[i], j // page]), j % page)
                  for j in range(min(int(pos[i]) + 1, table.shape[1] * page))]
        places = [x for x in places if 0 <= x[0] < k.shape[0]]
        if not places:
            continue
        p, o = (torch.tensor(x) for x in zip(*places))
        for g in range(KV):
            kk, vv = k[p, g, o].double(), v[p, g, o].double()
            for h in range(g * (H // KV), (g + 1) * (H // KV)):
                qq = q[i, h].double()
                s = (kk * qq).sum(-1) * scale
                w = torch.softmax(s, 0)
                out[i, h] = (w[:, None] * vv).sum(0)
                size = float((kk.abs() * qq.abs()).sum(-1).max()) * scale
                top = float(s.abs().max())
                rel = 2 * ((hd + 2) * size + 4 * top + 4 + 2 * (32 + len(places) / 16)) * 2.0 ** -24
                tol[i, h] = (rel + 2.0 ** -16) * (w[:, None] * vv.abs()).sum(0)
    if gate is not None:
        s = torch.sigmoid(gate.double())
        out, tol = out * s, tol * s + out.abs() * s * 2.0 ** -21
    return out.reshape(n, H * hd), tol.reshape(n, H * hd)


def attend_case(seed, H, KV, hd, page, lengths, dtype, order=None, spread=1.5):
    """q, gate, pages that hold NaN wherever no token is, table, lengths."""
    rng = np.random.default_rng(seed)
    table, pages = scattered(rng, lengths, page)
    t = lambda *s: torch.from_numpy(rng.standard_normal(s, dtype=np.float32)).to(dtype)  # noqa: E731
    kv = t(2, pages, KV, page, hd)
    held = np.zeros((pages, page), bool)
    for row, n in zip(table, lengths):
        for j in range(n):
            held[row[j // page], j % page] = True
    kv[:, ~torch.from_numpy(held).unsqueeze(1).expand(pages, KV, page)] = float("nan")
    index = np.arange(len(lengths)) if order is None else np.asarray(order)
    return t(len(index), H, hd) * spread, t(len(index), H, 2, hd)[:, :, 0], kv[0], kv[1], table, index


def attend_check(case, pos, page, dtype, out_dtype, gated=True, table=None):
    q, gate, k, v, real, index = case
    table = real if table is None else table
    scale = q.shape[2] ** -0.5
    f = flag()
    got = cache_ops.paged_attention(q.to(DEV), k.to(DEV), v.to(DEV), torch.from_numpy(table).to(DEV),
                                    ints(index), ints(pos), scale,
                                    gate=gate.to(DEV) if gated else None, out_dtype=out_dtype,
                                    error_flag=f)
    exp, tol = attend_exact(q, k, v, table, index, pos, scale, gate if gated else None, page)
    if out_dtype == ops.BF16X2:
        got, tol = ops.join_split(got), tol + 2.0 ** -17 * exp.abs()
    elif out_dtype == torch.bfloat16 or (out_dtype is None and dtype == torch.bfloat16):
        tol = tol + HALF[torch.bfloat16] * (exp.abs() + tol)
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    assert ((got - exp).abs() <= tol).all(), float(((got - exp).abs() / tol.clamp(min=1e-30)).max())
    return f.item()


# query heads of a KV head on both sides of 4 (a pass of the join) and 16 (a group);
# lengths around the tiles (16, 32), the pages and the four wavefronts' share
LENGTHS = [1, 0, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 200, 300]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,hd,page", [(4, 2, 64, 16), (8, 2, 256, 64), (5, 1, 128, 32),
                                          (16, 1, 64, 16), (20, 1, 128, 16), (3, 3, 256, 128),
                                          (34, 2, 64, 256)])
def test_paged_attention(H, KV, hd, page, dtype):
    case = attend_case(H * hd + page, H, KV, hd, page, LENGTHS, dtype,
                       order=np.random.default_rng(H).permutation(len(LENGTHS)))
    pos = np.array(LENGTHS)[case[-1]] - 1
    for out, gated in ((None, True), (torch.float32, False), (ops.BF16X2, True)):
        if out == ops.BF16X2 and dtype == torch.float32 and hd == 64:
            out = torch.bfloat16
        assert attend_check(case, pos, page, dtype, out, gated) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_attention_many_entries(dtype):
    """More entries than a wavefront sees at once, several of one row at positions of
    their own, and entries that are no token among them."""
    rng = np.random.default_rng(5)
    lengths = [int(x) for x in rng.integers(0, 90, 40)]
    order = rng.integers(0, 40, 151)
    case = attend_case(6, 4, 2, 64, 16, lengths, dtype, order=order)
    pos = np.array([rng.integers(-1, lengths[r]) if lengths[r] else -1 for r in order])
    index = case[-1]
    index[[3, 70, 150]] = -1
    assert attend_check(case, pos, 16, dtype, None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,hd,lengths", [(4, 1, 64, [9000]), (8, 2, 256, [3001, 2, 777]),
                                             (12, 4, 128, [0, 1, 5000, 0, 33])])
def test_paged_attention_long(H, KV, hd, lengths, dtype):
    """One row's keys over many workgroups, and very different rows beside each other."""
    case = attend_case(hd, H, KV, hd, 64, lengths, dtype, spread=3.0)
    assert attend_check(case, np.array(lengths) - 1, 64, dtype, None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,hd,lengths", [
    (8, 2, 256, [1000] * 8),                # an even share each, the last tile not full
    (4, 2, 64, [700] * 64), (4, 2, 64, [700] * 65),   # as many as a wavefront sees, one more
    (16, 16, 64, [20 + i for i in range(60)] + [2500]),  # more units than workgroups
    (40, 2, 64, [1500, 0, 1, 1033]),        # two groups of heads a KV head, one not full
    (12, 3, 64, [(37 * i) % 700 for i in range(181)]),   # all heads of an entry joined together
    (8, 2, 256, [16001])])                  # many pieces of one row
def test_paged_attention_dealt(H, KV, hd, lengths, dtype):
    """Keys that go to the workgroups in even shares and as one line."""
    case = attend_case(len(lengths) + hd, H, KV, hd, 16, lengths, dtype)
    assert attend_check(case, np.array(lengths) - 1, 16, dtype, None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,hd", [(8, 2, 256), (4, 2, 64), (12, 4, 128), (10, 2, 64)])
def test_paged_attention_shared_pages(H, KV, hd, dtype):
    """Rows that hold the same pages, some only the first of them, beside one that does not."""
    lengths = [900, 900, 611, 900, 640]
    case = attend_case(hd + H, H, KV, hd, 16, lengths, dtype)
    table = case[4].copy()
    table[1] = table[0]
    table[4, :20] = table[0, :20]
    pos = np.array(lengths) - 1
    pos[1] = 555
    assert attend_check(case, pos, 16, dtype, None, table=table) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_attention_rising_scores(dtype):
    """Scores that rise along the keys by hundreds, so that begun sums are rescaled,
    and a last key far below: its weight is nothing."""
    q, gate, k, v, table, index = case = attend_case(9, 4, 1, 64, 16, [400], dtype)
    for j in range(400):
        k[table[0, j // 16], 0, j % 16] = torch.where(q[0, 0] > 0, 1.0, -1.0) * (j / 40.0)
    k[table[0, 399 // 16], 0, 399 % 16] = -k[table[0, 398 // 16], 0, 398 % 16]
    assert attend_check(case, np.array([399]), 16, dtype, None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_attention_bad_tables(dtype):
    """Pages that are none, positions behind the table and rows that are none: left out
    and flagged, the other entries as they should be."""
    lengths = [100, 130, 64, 40]
    case = attend_case(11, 4, 2, 64, 16, lengths, dtype, order=[0, 1, 2, 3, 9])
    table = case[4].copy()
    table[0, 2], table[0, 6], table[2, :] = -1, case[2].shape[0], 1 << 30
    pos = np.array([99, 129, 63, 39, 10])
    assert attend_check(case, pos, 16, dtype, None, table=table) == 1
    full = table.shape[1] * 16                       # 144: row 1 holds 130, the rest NaN
    short = [144, 144]
    case = attend_case(12, 4, 2, 64, 16, short, dtype)
    assert attend_check(case, np.array([full + 50, 2 ** 31 - 1]), 16, dtype, None) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_attention_nan_and_inf(dtype):
    """A NaN or infinity that a row really holds shows in that row alone; a score of
    minus infinity is a weight of nothing."""
    q, gate, k, v, table, index = attend_case(13, 4, 2, 64, 16, [50, 60, 70, 80], dtype)
    k[table[0, 1], 0, 3, 5] = float("nan")
    v[table[1, 2], 1, 4, 7] = float("inf")
    q[2, 0, 0] = 1.0
    k[table[2, 0], 0, 2, 0] = -float("inf")          # head 0 of entry 2: key 2 masked
    d = lambda x: x.to(DEV)  # noqa: E731
    got = cache_ops.paged_attention(d(q), d(k), d(v), d(torch.from_numpy(table)), ints(index),
                                    ints([49, 59, 69, 79]), 0.125).float().cpu().view(4, 4, 64)
    assert torch.isnan(got[0, :2]).all() and torch.isfinite(got[0, 2:]).all()
    assert torch.isfinite(got[1, :2]).all() and (got[1, 2:, 7] == float("inf")).all()
    assert torch.isfinite(got[1, 2:, :7]).all() and torch.isfinite(got[3]).all()
    exp, _ = attend_exact(q, k, v, table, index, [49, 59, 69, 79], 0.125, None, 16)
    assert normwise(got[2, 0], exp.view(4, 4, 64)[2, 0]) <= 2 * HALF[dtype] + 1e-5


def short(n, H, KV, hd, table, page, dtype):
    """Whether such a call is one launch, of a workgroup for each entry and head group."""
    need = _lib.lib().qdc_paged_attention_workspace(n, H, KV, hd, table.shape[1], page,
                                                    F32 if dtype == torch.float32 else BF16)
    assert need >= 0
    return need == 0


def widen(table, places, page):
    """The same rows in a table of ``places`` positions and more, -1 behind them."""
    more = max(0, -(-places // page) - table.shape[1])
    return np.pad(table, ((0, 0), (0, more)), constant_values=-1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,hd,page", [(4, 2, 64, 16), (8, 2, 256, 64), (5, 1, 128, 32),
                                          (16, 1, 64, 16), (20, 1, 128, 16), (3, 3, 256, 128),
                                          (34, 2, 64, 256), (12, 3, 256, 16)])
def test_paged_attention_rows_of_a_wide_table(H, KV, hd, page, dtype):
    """Short rows whose table could hold long ones: work is dealt out by what is there."""
    case = attend_case(H * hd + page, H, KV, hd, page, LENGTHS, dtype,
                       order=np.random.default_rng(H).permutation(len(LENGTHS)))
    pos, table = np.array(LENGTHS)[case[-1]] - 1, widen(case[4], 2000, page)
    assert not short(len(pos), H, KV, hd, table, page, dtype)
    for out, gated in ((None, True), (torch.float32, False), (ops.BF16X2, True)):
        assert attend_check(case, pos, page, dtype, out, gated, table=table) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,hd,page", [(8, 2, 256, 16), (3, 1, 256, 64), (20, 1, 256, 32),
                                          (12, 4, 128, 16), (17, 1, 128, 128), (6, 1, 64, 32)])
def test_paged_attention_short_rows(H, KV, hd, page, dtype):
    """Tables of so few positions that a workgroup takes a unit whole, up to their last."""
    most = {64: 16, 128: 8, 256: 4}[hd] * 2 * (32 if dtype == torch.bfloat16 else 16)
    lengths = [n for n in LENGTHS if n < most] + [most, most - 1]
    case = attend_case(H * hd + page, H, KV, hd, page, lengths, dtype)
    assert short(len(lengths), H, KV, hd, case[4], page, dtype)
    assert case[4].shape[1] * page == most
    assert not short(1, H, KV, hd, widen(case[4], most + 1, page), page, dtype)
    for out, gated in ((None, True), (torch.float32, False), (ops.BF16X2, True)):
        assert attend_check(case, np.array(lengths) - 1, page, dtype, out, gated) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,hd,rows,n", [
    (4, 2, 64, 40, 65),          # one entry more than a wavefront sees
    (8, 2, 256, 30, 151),
    (12, 4, 128, 60, 171),       # 2052 heads: all of an entry joined by one workgroup
    (8, 1, 64, 90, 300),
    (20, 1, 64, 50, 128)])       # the same, two groups of heads
def test_paged_attention_many_entries_of_a_wide_table(H, KV, hd, rows, n, dtype):
    """More entries than a wavefront sees at once, dealt out as one line, several of one
    row at positions of their own, entries that are no token among them."""
    rng = np.random.default_rng(n + hd)
    lengths = [int(x) for x in rng.integers(0, 90, rows)]
    lengths[:3] = [700, 1, 0]
    order = rng.integers(0, rows, n)
    order[:2] = 0
    case = attend_case(n, H, KV, hd, 16, lengths, dtype, order=order)
    pos = np.array([rng.integers(-1, lengths[r]) if lengths[r] else -1 for r in order])
    pos[0] = 699
    case[-1][[3, 63, 64, n - 1]] = -1
    table = widen(case[4], 1100, 16)
    assert not short(n, H, KV, hd, table, 16, dtype)
    assert attend_check(case, pos, 16, dtype, None, table=table) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,hd,n,out", [(2, 1, 64, 4095, None), (2, 1, 64, 4096, ops.BF16X2),
                                           (3, 3, 128, 6201, None)])
def test_paged_attention_thousands_of_entries(H, KV, hd, n, out, dtype):
    """Entries on both sides of where a call is launched in slices, each of its own row of
    the arguments."""
    rng = np.random.default_rng(n)
    lengths = [int(x) for x in rng.integers(0, 40, 50)]
    lengths[0] = 300
    order = rng.integers(1, 50, n)
    order[[0, n // 2, n - 1]] = 0
    case = attend_case(n, H, KV, hd, 16, lengths, dtype, order=order)
    pos = np.array([lengths[r] - 1 for r in order])
    case[-1][rng.integers(1, n // 2, 20)] = -1
    table = widen(case[4], 1100, 16)
    assert not short(n, H, KV, hd, table, 16, dtype)
    assert attend_check(case, pos, 16, dtype, out, table=table) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_attention_widest_table(dtype):
    """A row of 2^31 - 16 keys, all but the last 20 of them one page again and again.  The
    last page's scores are 22 and the others' 1 at most, so it has 0.7 of the weight or
    more.  Sums over 2^27 tiles of 2048 wavefronts: chains of 65536 additions, 2^-24 each,
    of the weights and of their products, and as many again for the rescaling: 2^-6."""
    width, hd = 2 ** 27 - 1, 64
    rng = np.random.default_rng(1)
    t = lambda *s: torch.from_numpy(rng.standard_normal(s, dtype=np.float32)).to(dtype)  # noqa: E731
    q = torch.ones(1, 1, hd, dtype=dtype)
    k, v = t(3, 1, 16, hd) * 0.05, t(3, 1, 16, hd)
    k[2] = 2.75                                             # 64 of it / 8: 22
    table = torch.zeros((1, width), dtype=torch.int32, device=DEV)
    table[0, -2], table[0, -1] = 1, 2
    last = width * 16 - 1 - 12                              # 4 keys of the last page
    f = flag()
    got = cache_ops.paged_attention(q.to(DEV), k.to(DEV), v.to(DEV), table, ints([0]), ints([last]),
                                    0.125, out_dtype=torch.float32, error_flag=f)
    assert f.item() == 0
    s = (k.double()[:, 0].sum(-1) * 0.125)                  # [3, 16]
    assert s[:2].max() < 1 and (s[2] == 22).all()
    times = torch.ones(3, 16, dtype=torch.float64)
    times[0], times[2, 4:] = width - 2, 0
    w = times * torch.exp(s)
    w /= w.sum()
    assert 0.7 < w[2].sum() < 0.95
    exp = (w[..., None] * v.double()[:, 0]).sum((0, 1))
    tol = (2.0 ** -6 + 2.0 ** -16) * (w[..., None] * v.double()[:, 0].abs()).sum((0, 1))
    assert ((got.double().cpu()[0] - exp).abs() <= tol).all()


@pytest.mark.gpu
def test_paged_attention_time_of_many_entries():
    """Eight times the entries take eight times as long, not sixty-four."""
    pages = torch.zeros(64, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    table = torch.full((64, 80), -1, dtype=torch.int32, device=DEV)
    table[:, 0] = torch.arange(64, device=DEV)

    def best(n):
        q = torch.zeros(n, 4, 64, dtype=torch.bfloat16, device=DEV)
        rows, pos = ints(np.arange(n) % 64), ints(np.arange(n) % 16)
        times = []
        for _ in range(4):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            cache_ops.paged_attention(q, pages, pages, table, rows, pos, 0.1)
            end.record()
            end.synchronize()
            times.append(start.elapsed_time(end))
        return min(times)

    few, many = best(8192), best(65536)     # whole: 0.45 and 17.3 ms
    assert many < 16 * few, (few, many)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,hd", [(4, 2, 64), (8, 2, 256), (10, 1, 128)])
def test_paged_attention_shared_pages_of_a_wide_table(H, KV, hd, dtype):
    """Rows that hold the same pages, in the kernel that keeps those in the caches."""
    lengths = [900, 900, 611, 900, 640, 900]
    case = attend_case(hd + H, H, KV, hd, 16, lengths, dtype)
    table = widen(case[4], 1100, 16)
    table[1] = table[0]
    table[4, :20] = table[0, :20]
    pos = np.array(lengths) - 1
    pos[1], pos[5] = 555, -1
    assert not short(len(pos), H, KV, hd, table, 16, dtype)
    assert attend_check(case, pos, 16, dtype, None, table=table) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,hd,n", [(4, 1, 64, 1500), (8, 1, 256, 2500), (20, 1, 128, 1100)])
def test_paged_attention_rising_scores_over_pieces(H, KV, hd, n, dtype):
    """Scores that rise along the keys by hundreds, from piece to piece of a row, and a
    last key far below."""
    q, gate, k, v, table, index = case = attend_case(9, H, KV, hd, 16, [n], dtype)
    for j in range(n):
        k[table[0, j // 16], 0, j % 16] = torch.where(q[0, 0] > 0, 1.0, -1.0) * (j * 10.0 / n)
    k[table[0, (n - 1) // 16], 0, (n - 1) % 16] *= -1
    assert not short(1, H, KV, hd, table, 16, dtype)
    assert attend_check(case, np.array([n - 1]), 16, dtype, None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,hd", [(4, 2, 64), (8, 2, 256), (17, 1, 128)])
@pytest.mark.parametrize("others", [0, 61])
def test_paged_attention_bad_long_tables(H, KV, hd, others, dtype):
    """Pages that are none within long rows, a row of nothing but such, positions behind
    the table and rows that are none: left out and flagged, in the shares of few entries
    and in the line of many."""
    lengths = [1500, 1300, 700, 40, 9] + [7] * others
    n = len(lengths)
    order = np.arange(n)
    order[4] = n + 3                                        # no row
    case = attend_case(11, H, KV, hd, 16, lengths, dtype, order=order)
    table = widen(case[4], 1600, 16)
    assert not short(n, H, KV, hd, table, 16, dtype)
    table[0, 2], table[0, 70:], table[2, :] = -1, case[2].shape[0], 1 << 30
    pos = np.array(lengths) - 1
    pos[4] = 10
    assert attend_check(case, pos, 16, dtype, None, table=table) == 1
    full = [1600, 1600, 33]                                 # every place of the table held
    case = attend_case(12, H, KV, hd, 16, full, dtype)
    assert attend_check(case, np.array([1650, 2 ** 31 - 1, 32]), 16, dtype, None) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,hd", [(4, 2, 64), (8, 2, 256), (6, 2, 128)])
def test_paged_attention_nan_and_inf_in_long_rows(H, KV, hd, dtype):
    """A NaN or infinity in one piece of a long row shows in that row's heads alone; a score
    of minus infinity is a weight of nothing."""
    lengths = [1500, 1600, 1700, 1100]
    q, gate, k, v, table, index = attend_case(13, H, KV, hd, 16, lengths, dtype)
    k[table[0, 41], 0, 3, 5] = float("nan")
    v[table[1, 52], 1, 4, 7] = float("inf")
    q[2, 0, 0] = 1.0
    k[table[2, 60], 0, 2, 0] = -float("inf")          # head 0 of entry 2: one key masked
    assert not short(4, H, KV, hd, table, 16, dtype)
    d, scale, G = lambda x: x.to(DEV), hd ** -0.5, H // KV  # noqa: E731
    pos = [x - 1 for x in lengths]
    got = cache_ops.paged_attention(d(q), d(k), d(v), d(torch.from_numpy(table)), ints(index),
                                    ints(pos), scale).float().cpu().view(4, H, hd)
    assert torch.isnan(got[0, :G]).all() and torch.isfinite(got[0, G:]).all()
    assert torch.isfinite(got[1, :G]).all() and (got[1, G:, 7] == float("inf")).all()
    rest = [i for i in range(hd) if i != 7]
    assert torch.isfinite(got[1, G:][:, rest]).all() and torch.isfinite(got[3]).all()
    exp, _ = attend_exact(q, k, v, table, index, pos, scale, None, 16)
    exp = exp.view(4, H, hd)
    for i, h in ((2, 0), (1, 0), (3, H - 1)):
        assert normwise(got[i, h], exp[i, h]) <= 2 * HALF[dtype] + 1e-5


@pytest.mark.gpu
def test_paged_attention_refusals():
    z = lambda *s, dt=torch.float32: torch.zeros(s, dtype=dt, device=DEV)  # noqa: E731
    i, q, pg, table = ints([0, 1]), z(2, 4, 64), z(4, 2, 16, 64), z(2, 3, dt=torch.int32)
    ok = dict(q=q, k_pages=pg, v_pages=pg, table=table, rows=i, positions=i, scale=0.1)
    cache_ops.paged_attention(**ok)
    assert cache_ops.paged_attention(**dict(ok, q=q[:0], rows=i[:0], positions=i[:0])).shape == (0, 256)
    for bad in (dict(q=q[0]), dict(q=q.half()), dict(q=z(2, 3, 64)), dict(v_pages=pg[:2]),
                dict(k_pages=pg.bfloat16(), v_pages=pg.bfloat16()), dict(table=table.long()),
                dict(rows=ints([0])), dict(positions=i.long()), dict(scale=0.0),
                dict(scale=float("nan")), dict(gate=q[:1]), dict(gate=q.bfloat16()),
                dict(out_dtype=torch.float16), dict(out_dtype="f8"),
                dict(q=z(2, 4, 32), k_pages=z(4, 2, 16, 32), v_pages=z(4, 2, 16, 32)),
                dict(k_pages=z(4, 2, 10, 64), v_pages=z(4, 2, 10, 64)),
                dict(table=z(2, 3, dt=torch.int32).cpu()), dict(error_flag=i.long())):
        with pytest.raises(ValueError):
            cache_ops.paged_attention(**dict(ok, **bad))


# -------------------------------------------------------------------- pages --
class Model:
    """The page table in plain Python, as the operators' documentation has it."""

    def __init__(self, rows, width, pages, page):
        self.rows, self.width, self.pages, self.page = rows, width, pages, page
        self.table = [[] for _ in range(rows)]
        self.lengths, self.refs = [0] * rows, [0] * pages
        self.stack = list(range(pages - 1, -1, -1))

    def good(self, rows):
        rows = [r for r in rows if r >= 0]
        return len(set(rows)) == len(rows) and all(r < self.rows for r in rows)

    def extend(self, rows, counts):
        live = [(r, c) for r, c in zip(rows, counts) if r >= 0]
        if not self.good(rows) or any(c < 0 or self.lengths[r] + c > self.width * self.page
                                      for r, c in live):
            return [-1] * len(rows), True
        need = [-(-(self.lengths[r] + c) // self.page) - len(self.table[r]) for r, c in live]
        if sum(need) > len(self.stack):
            return [-1] * len(rows), True
        out = []
        need = iter(need)
        for r, c in zip(rows, counts):
            out.append(-1 if r < 0 else self.lengths[r])
            if r >= 0:
                for _ in range(next(need)):
                    self.table[r].append(self.stack.pop())
                    self.refs[self.table[r][-1]] = 1
                self.lengths[r] += c
        return out, False

    def free(self, rows):
        if not self.good(rows):
            return True
        listed = [p for r in rows if r >= 0 for p in self.table[r]]
        for p in listed:
            self.refs[p] -= 1
        last = {p: i for i, p in enumerate(listed)}
        left = [p for i, p in enumerate(listed) if self.refs[p] == 0 and last[p] == i]
        self.stack += left[::-1]
        for r in rows:
            if r >= 0:
                self.table[r], self.lengths[r] = [], 0
        return False

    def fork(self, parents, children, data=None):
        live = [(p, c) for p, c in zip(parents, children) if p >= 0 and c >= 0]
        kids = [c for _, c in live]
        if not self.good(kids) or any(p >= self.rows or p in kids for p, _ in live) or \
                any(self.lengths[c] for c in kids):
            return True
        if sum(self.lengths[p] % self.page > 0 for p, _ in live) > len(self.stack):
            return True
        for p, c in live:
            full, part = divmod(self.lengths[p], self.page)
            self.table[c], self.lengths[c] = self.table[p][:full], self.lengths[p]
            for x in self.table[c]:
                self.refs[x] += 1
            if part:
                new = self.stack.pop()
                self.refs[new] = 1
                self.table[c].append(new)
                if data is not None:
                    data[:, new, :, :part] = data[:, self.table[p][full], :, :part]
        return False

    def compact(self, data=None):
        live = [p for p in range(self.pages) if self.refs[p] > 0]
        m = len(live)
        holes = [p for p in range(m) if self.refs[p] <= 0]
        to = dict(zip([p for p in live if p >= m], holes))
        for src, dst in to.items():
            self.refs[dst], self.refs[src] = self.refs[src], 0
            if data is not None:
                data[:, dst] = data[:, src]
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        self.stack = list(range(self.pages - 1, m - 1, -1))

    def check(self, book):
        table = [row + [-1] * (self.width - len(row)) for row in self.table]
        assert book.table.tolist() == table
        assert book.lengths.tolist() == self.lengths and book.refs.tolist() == self.refs
        free = book.free.tolist()
        assert free[0] == len(self.stack) and free[1:1 + free[0]] == self.stack


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,pages,page,dtype,dim", [(12, 6, 40, 16, torch.float32, 4),
                                                             (7, 3, 11, 64, torch.bfloat16, 64),
                                                             (10, 3, 40, 64, torch.float32, 256),
                                                             (30, 9, 300, 32, torch.bfloat16, 8)])
def test_pages_life(rows, width, pages, page, dtype, dim):
    """Rows that grow, fork, end and move together in any order, whole numbers and
    copies exact after every call; calls that cannot be done whole among them."""
    rng = np.random.default_rng(rows * page)
    book, ref = cache_ops.page_table(rows, width, pages, page, DEV), Model(rows, width, pages, page)
    data = torch.from_numpy(rng.standard_normal((3, pages, 2, page, dim), dtype=np.float32)).to(dtype)
    pool = data.to(DEV)
    refused = {"extend": 0, "fork": 0, "free": 0}
    for step in range(60):
        f = flag()
        what = rng.choice(["extend", "extend", "extend", "fork", "fork", "free", "compact"])
        n = int(rng.integers(1, rows // 2 + 2))
        some = rng.permutation(rows)[:n].tolist()
        if rng.random() < 0.15:
            some[rng.integers(n)] = int(rng.choice([-1, rows, some[0]]))
        if what == "extend":
            counts = [int(c) for c in rng.choice([0, 1, 1, page - 1, page, 2 * page + 3], len(some))]
            if rng.random() < 0.1:
                counts[-1] = -1
            got = cache_ops.extend_pages(book, ints(some), ints(counts), error_flag=f)
            exp, bad = ref.extend(some, counts)
            assert got.tolist() == exp
        elif what == "fork":
            empty = [r for r in range(rows) if not ref.lengths[r]]
            rng.shuffle(empty)
            kids = (empty + some)[:n]
            parents = [int(x) for x in rng.integers(-1, rows, len(kids))]
            cache_ops.fork_pages(book, ints(parents), ints(kids), pool, error_flag=f)
            bad = ref.fork(parents, kids, data)
        elif what == "free":
            cache_ops.free_pages(book, ints(some), error_flag=f)
            bad = ref.free(some)
        else:
            cache_ops.compact_pages(book, pool)
            ref.compact(data)
            bad = False
        refused[what] = refused.get(what, 0) + bool(bad)
        assert f.item() == int(bad), (step, what)
        ref.check(book)
        assert torch.equal(pool.cpu(), data), (step, what)
    assert refused["extend"] and refused["fork"]


@pytest.mark.gpu
def test_pages_many_rows():
    """More rows in a call than the bookkeeping takes at once, pages that hundreds of
    rows share, and rows that free them in one call."""
    rows, width, pages, page = 2600, 4, 6000, 16
    book, ref = cache_ops.page_table(rows, width, pages, page, DEV), Model(rows, width, pages, page)
    rng = np.random.default_rng(3)
    some = rng.permutation(rows)[:1300].tolist()
    counts = [int(c) for c in rng.integers(1, width * page + 1, 1300)]
    got, (exp, bad) = cache_ops.extend_pages(book, ints(some), ints(counts)), ref.extend(some, counts)
    assert got.tolist() == exp and not bad
    ref.check(book)
    kids = [r for r in range(rows) if not ref.lengths[r]][:1200]
    parents = [some[i % 3] for i in range(len(kids))]
    cache_ops.fork_pages(book, ints(parents), ints(kids))
    assert not ref.fork(parents, kids)
    ref.check(book)
    gone = rng.permutation(some[:900] + kids[:1100]).tolist()
    cache_ops.free_pages(book, ints(gone))
    assert not ref.free(gone)
    ref.check(book)
    cache_ops.compact_pages(book)
    ref.compact()
    ref.check(book)


@pytest.mark.gpu
def test_fork_and_free_give_the_stack_back():
    book = cache_ops.page_table(9, 8, 50, 16, DEV)
    cache_ops.extend_pages(book, ints([4, 2]), ints([50, 17]))
    before = [t.clone() for t in book[:4]]
    for _ in range(3):
        cache_ops.fork_pages(book, ints([4, 2, 4, 4]), ints([0, 8, 1, 3]))
        cache_ops.free_pages(book, ints([0, 8, 1, 3]))
        for a, b in zip(before, book[:4]):
            assert torch.equal(a, b)
    # a parent that ends before its children: they keep its pages
    cache_ops.fork_pages(book, ints([4]), ints([0]))
    cache_ops.free_pages(book, ints([4]))
    assert book.lengths.tolist() == [50, 0, 17, 0, 0, 0, 0, 0, 0]
    assert sorted(book.refs.tolist())[-6:] == [1] * 6 and book.free[0].item() == 50 - 6


@pytest.mark.gpu
def test_copy_pages():
    rng = np.random.default_rng(1)
    for shape, dtype in (((2, 9, 4), torch.float32), ((1, 300, 3, 40), torch.bfloat16),
                         ((5, 20, 1025, 4), torch.float32)):
        data = torch.from_numpy(rng.standard_normal(shape, dtype=np.float32)).to(dtype)
        pool, f = data.to(DEV), flag()
        order = rng.permutation(shape[1])
        src, dst = order[:3].tolist() * 2, order[3:9].tolist()
        cache_ops.copy_pages(pool, ints(src), ints(dst), error_flag=f)
        data[:, dst] = data[:, src]
        assert torch.equal(pool.cpu(), data) and f.item() == 0
        # dst twice: the first; dst that is a src, src and dst out of range: not at all;
        # a negative index: left out
        a, b, c, d, e = order[:5].tolist()
        n = shape[1]
        cache_ops.copy_pages(pool, ints([a, b, c, n, a, -1]), ints([d, d, a, e, n, e]), error_flag=f)
        data[:, d] = data[:, a]
        assert torch.equal(pool.cpu(), data) and f.item() == 1
    cache_ops.copy_pages(pool, ints([]), ints([]))
    # one item, whose stride may be anything
    data = torch.zeros(3, 1, 8, device=DEV).as_strided((3, 1, 8), (8, 12345, 1))
    data += torch.arange(24, device=DEV).view(3, 1, 8)
    assert data.is_contiguous()
    f.zero_()
    cache_ops.copy_pages(data, ints([0]), ints([0]), error_flag=f)
    assert f.item() == 1 and torch.equal(data.flatten(), torch.arange(24.0, device=DEV))
    # more pairs of one src than a workgroup writes at once, bad ones between them
    data = torch.from_numpy(rng.standard_normal((2, 400, 260), dtype=np.float32))
    pool, f = data.to(DEV), flag()
    order = rng.permutation(400).tolist()
    src = [order[int(x)] for x in rng.integers(0, 3, 300)]
    dst = order[3:303]
    dst[17], dst[40], dst[41] = order[1], dst[39], 400    # a src, an earlier dst, none
    src[100] = -1
    cache_ops.copy_pages(pool, ints(src), ints(dst), error_flag=f)
    for i, (a, b) in enumerate(zip(src, dst)):
        if i not in (17, 40, 41, 100):
            data[:, b] = data[:, a]
    assert torch.equal(pool.cpu(), data) and f.item() == 1
    with pytest.raises(ValueError):
        cache_ops.copy_pages(pool, ints([0] * 4097), ints([1] * 4097))


@pytest.mark.gpu
def test_pages_refusals():
    book = cache_ops.page_table(3, 4, 5, 16, DEV)
    i, pool = ints([0, 1]), torch.zeros(2, 5, 2, 16, 8, device=DEV)
    for bad in (lambda: cache_ops.extend_pages(book, i.long()),
                lambda: cache_ops.extend_pages(book, i, ints([1])),
                lambda: cache_ops.extend_pages(book, i, positions=ints([1])),
                lambda: cache_ops.extend_pages(book._replace(page_size=20), i),
                lambda: cache_ops.extend_pages(book._replace(free=book.free[1:]), i),
                lambda: cache_ops.extend_pages(book._replace(lengths=book.refs), i),
                lambda: cache_ops.free_pages(book, i.cpu()),
                lambda: cache_ops.fork_pages(book, i, ints([2])),
                lambda: cache_ops.fork_pages(book, i, i, pool[:, :4]),
                lambda: cache_ops.fork_pages(book, i, i, pool.transpose(2, 3)),
                lambda: cache_ops.fork_pages(book, i, i, torch.zeros(2, 5, 2, 16, 6, device=DEV,
                                                                     dtype=torch.bfloat16)),
                lambda: cache_ops.compact_pages(book, pool[:, :4]),
                lambda: cache_ops.copy_pages(pool[:, :, 0], i, i),
                lambda: cache_ops.copy_pages(torch.zeros(2, 5, 3, device=DEV), i, i),
                lambda: cache_ops.copy_pages(pool, i, ints([2]))):
        with pytest.raises(ValueError):
            bad()
    assert book.lengths.tolist() == [0, 0, 0]


# --------------------------------------------------------------- delta_step --
# key heads, value heads, key size, value size, taps
STEP = [(2, 4, 128, 128, 4), (1, 1, 32, 16, 1), (2, 2, 64, 48, 2), (1, 4, 128, 256, 4),
        (4, 8, 32, 80, 8), (3, 3, 64, 144, 3)]


def step_exact(s, KH, kd, H, vd, taps):
    """64 bits on the CPU; rows are updated in place."""
    kw, vw = KH * kd, H * vd
    cq = 2 * kw + vw
    out = torch.zeros(len(s["rows"]), H, vd, dtype=torch.float64)
    proj, ring, state = s["proj"].double(), s["ring"].double(), s["state"].double()
    done = set()
    for i, (row, p) in enumerate(zip(s["rows"], s["pos"])):
        if row < 0 or p < 0 or row >= len(ring) or row in done:
            continue
        done.add(row)
        ring[row, p % taps] = proj[i, :cq]
        x = torch.zeros(cq, dtype=torch.float64)
        for lag in range(min(taps, p + 1)):
            x += ring[row, (p - lag) % taps] * s["conv"][:, taps - 1 - lag].double()
        x = x * torch.sigmoid(x)
        q, k, v = x[:kw].view(KH, kd), x[kw:2 * kw].view(KH, kd), x[2 * kw:].view(H, vd)
        q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + 1e-6) / math.sqrt(kd)
        k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + 1e-6)
        q, k = (t.repeat_interleave(H // KH, 0) for t in (q, k))
        tail = proj[i, cq:]
        z, a, b = tail[:vw].view(H, vd), tail[vw:vw + H], tail[vw + H:vw + 2 * H]
        f = torch.exp(s["a_decay"].double() *
                      torch.nn.functional.softplus(a + s["dt_bias"].double(), threshold=200.0))
        S = state[row] * f[:, None, None] if p else torch.zeros_like(state[row])
        u = torch.sigmoid(b)[:, None] * (v - (S * k[:, None]).sum(-1))
        S = S + u[..., None] * k[:, None]
        state[row] = S
        o = (S * q[:, None]).sum(-1)
        o = o / torch.sqrt((o * o).mean(-1, keepdim=True) + 1e-6) * s["norm"].double()
        out[i] = o * z * torch.sigmoid(z)
    return out.view(-1, vw), ring, state


def step_case(seed, KH, H, kd, vd, taps, n, rows, dtype):
    rng = np.random.default_rng(seed)
    t = lambda *s: torch.from_numpy(rng.standard_normal(s, dtype=np.float32))  # noqa: E731
    cq = 2 * KH * kd + H * vd
    return {"proj": t(n, cq + H * vd + 2 * H + 5).to(dtype), "conv": t(cq, taps) * 0.5,
            "a_decay": -torch.exp(t(H)), "dt_bias": t(H), "norm": (1 + 0.1 * t(vd)).to(dtype),
            "ring": t(rows, taps, cq).to(dtype), "state": t(rows, H, vd, kd) * 0.3,
            "rows": [int(r) for r in rng.permutation(rows)[:n]],
            "pos": [int(p) for p in rng.integers(0, 2 * taps + 3, n)]}


def step_run(s, KH, H, kd, vd, out_dtype=None, error_flag=None):
    d = {k: v.to(DEV) for k, v in s.items() if isinstance(v, torch.Tensor)}
    out = cache_ops.delta_step(d["proj"], d["conv"], d["a_decay"], d["dt_bias"], d["norm"], 1e-6,
                               d["ring"], d["state"], ints(s["rows"]), ints(s["pos"]), KH, kd, H, vd,
                               out_dtype=out_dtype, error_flag=error_flag)
    return out, d["ring"], d["state"]


def step_near(got, exp, KH, kd, vd, dtype, split=False):
    """fp32 throughout: a state is one product and sum after dot products of kd terms,
    off by at most (kd + 40) half steps of the largest value in its head (u and the
    gates take some tens of operations); an output row is normalised, so its values
    are off by as much of the row's largest, then rounded to its type."""
    (out, ring, state), (eo, er, es) = got, exp
    assert torch.equal(ring.double().cpu(), er)
    top = es.abs().amax((-1, -2), keepdim=True).clamp(min=1.0)
    assert ((state.double().cpu() - es).abs() <= (kd + 40) * 2.0 ** -24 * top).all()
    out = (ops.join_split(out) if split else out).double().cpu()
    rows = eo.view(len(eo), -1, vd)
    size = rows.abs().amax(-1, keepdim=True).expand_as(rows).reshape_as(eo)
    half = 2.0 ** -17 if split else HALF[dtype]
    # the norm divides by the row's size: relative errors of its values come out alike
    tol = 4 * (kd + vd + 40) * 2.0 ** -24 * size + half * eo.abs()
    assert ((out - eo).abs() <= tol).all(), float(((out - eo).abs() / tol.clamp(min=1e-30)).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("KH,H,kd,vd,taps", STEP)
def test_delta_step(KH, H, kd, vd, taps, dtype):
    s = step_case(kd + vd, KH, H, kd, vd, taps, 7, 9, dtype)
    f = flag()
    got = step_run(s, KH, H, kd, vd, error_flag=f)
    step_near(got, step_exact(s, KH, kd, H, vd, taps), KH, kd, vd, dtype)
    assert f.item() == 0
    if dtype == torch.bfloat16:
        got = step_run(s, KH, H, kd, vd, out_dtype=ops.BF16X2)
        step_near(got, step_exact(s, KH, kd, H, vd, taps), KH, kd, vd, dtype, split=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_delta_step_rows(dtype):
    """Rows at position 0 start empty whatever they held, NaN too; entries that are no
    token, a row named twice and one that is none: zeros, and the cache as it was."""
    KH, H, kd, vd, taps = 2, 4, 64, 32, 4
    s = step_case(3, KH, H, kd, vd, taps, 9, 12, dtype)
    s["pos"] = [0, 2, -1, 9, 5, 6, 7, 1, 3]
    r0, r1 = s["rows"][0], s["rows"][1]
    s["ring"][r0], s["state"][r0] = float("nan"), float("nan")
    s["ring"][r1, 3] = float("nan")             # position -1 of a row at position 2
    s["rows"][4], s["rows"][5], s["rows"][6] = -1, s["rows"][3], 12
    f = flag()
    got = step_run(s, KH, H, kd, vd, error_flag=f)
    exp = step_exact(s, KH, kd, H, vd, taps)
    assert f.item() == 1 and (got[0][[2, 4, 5, 6]] == 0).all()
    assert torch.isnan(got[1].float().cpu()[r0, 1:]).all()
    assert torch.isfinite(got[2][r0]).all()
    exp = (exp[0], torch.nan_to_num(exp[1]), exp[2])
    step_near((got[0], torch.nan_to_num(got[1].double()), got[2]), exp, KH, kd, vd, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("taps", [3, 4, 8])
def test_delta_step_last_positions(taps):
    """The largest positions there are: the window's slots are those of the tokens before,
    whatever their sum with the taps passes."""
    KH, H, kd, vd, n = 2, 4, 32, 32, 9
    s = step_case(taps, KH, H, kd, vd, taps, n, n, torch.float32)
    s["pos"] = [2 ** 31 - 1 - i for i in range(n)]
    s["rows"] = list(range(n))          # the largest in the first row
    f = flag()
    got = step_run(s, KH, H, kd, vd, error_flag=f)
    step_near(got, step_exact(s, KH, kd, H, vd, taps), KH, kd, vd, torch.float32)
    assert f.item() == 0


@pytest.mark.gpu
def test_delta_step_large_state():
    """A state of 128 MB and more is streamed: the same bits as rows a few at a time."""
    KH, H, kd, vd, n = 16, 32, 128, 128, 70
    g = torch.Generator(device=DEV).manual_seed(5)
    t = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    cq = 2 * KH * kd + H * vd
    assert n * H * vd * kd * 4 >= 128 << 20
    args = [t(n, cq + H * vd + 2 * H), t(cq, 4) * 0.5, -t(H).exp(), t(H), 1 + 0.1 * t(vd), 1e-6,
            t(n + 1, 4, cq), t(n + 1, H, vd, kd) * 0.3]
    rows, pos = torch.randperm(n + 1, generator=g, device=DEV)[:n].int(), ints(range(n))
    rows[7], rows[9], pos[11] = -1, rows[3], -1
    ring, state, f = args[6].clone(), args[7].clone(), flag()
    out = cache_ops.delta_step(*args[:6], ring, state, rows, pos, KH, kd, H, vd, error_flag=f)
    assert f.item() == 1 and (out[[7, 9, 11]] == 0).all()
    rows[9] = -1
    for i in range(0, n, 10):
        few = cache_ops.delta_step(args[0][i:i + 10], *args[1:], rows[i:i + 10].contiguous(),
                                   pos[i:i + 10].contiguous(), KH, kd, H, vd)
        assert torch.equal(few, out[i:i + 10])
    assert torch.equal(ring, args[6]) and torch.equal(state, args[7])


@pytest.mark.gpu
@pytest.mark.parametrize("S,KH,H,kd,vd", [(5, 2, 4, 128, 128), (40, 1, 2, 64, 48), (70, 16, 64, 32, 32)])
def test_steps_continue_a_scan(S, KH, H, kd, vd):
    """A prompt through the prologue, the scan (with its last state) and the gated norm,
    and then tokens one by one: the same as the whole sequence at once, to the fp32 bar
    of 1e-5 that both forms hold."""
    taps, more, dtype = 4, 6, torch.float32
    rng = np.random.default_rng(S)
    kw, vw = KH * kd, H * vd
    cq = 2 * kw + vw
    width = -(-(cq + vw + 2 * H) // 4) * 4
    B = 9 if H == 64 else 2                # both forms of the scan
    d = lambda x: torch.from_numpy(np.asarray(x, np.float32)).to(DEV)  # noqa: E731
    proj = d(rng.standard_normal((B, S + more, width)))
    conv, norm = d(rng.standard_normal((cq, taps)) * 0.5), d(1 + 0.1 * rng.standard_normal(vd))
    decay, bias = d(-np.exp(rng.standard_normal(H))), d(rng.standard_normal(H) - 2)

    def whole(n):
        p = proj[:, :n].reshape(B * n, width).contiguous()
        q, k, v, beta, dec = ops.delta_prologue(p, conv, decay, bias, n, KH, kd, H, vd,
                                                interleaved=True)
        shape = lambda t: t.view(B, n, *t.shape[1:])  # noqa: E731
        return [shape(t) for t in (q, k, v, beta, dec)]

    state = torch.empty(B, H, vd, kd, device=DEV)
    out = ops.delta_scan(*whole(S), state=state)
    assert normwise(out.cpu(), ops.delta_scan(*whole(S)).cpu()) <= 1e-6
    ring = torch.full((B, taps, cq), float("nan"), device=DEV)
    for p in range(max(0, S - taps), S):
        ring[:, p % taps] = proj[:, p, :cq]
    steps = []
    for p in range(S, S + more):
        steps.append(cache_ops.delta_step(proj[:, p], conv, decay, bias, norm, 1e-6, ring, state,
                                          ints(range(B)), ints([p] * B), KH, kd, H, vd))
    full = ops.delta_scan(*whole(S + more)).view(-1, H, vd)
    z = proj[..., cq:cq + vw].reshape(-1, H, vd).contiguous()
    exp = ops.native_gated_rms(full, z, norm, 1e-6).view(B, S + more, vw)[:, S:]
    assert normwise(torch.stack(steps, 1).cpu(), exp.cpu()) <= 1e-5
    last = torch.empty_like(state)
    ops.delta_scan(*whole(S + more), state=last)
    assert normwise(state.cpu(), last.cpu()) <= 1e-5


@pytest.mark.gpu
def test_delta_step_refusals():
    KH, H, kd, vd = 2, 4, 64, 32
    s = step_case(1, KH, H, kd, vd, 4, 2, 3, torch.float32)
    d = {k: v.to(DEV) for k, v in s.items() if isinstance(v, torch.Tensor)}
    ok = dict(d, eps=1e-6, rows=ints([0, 1]), positions=ints([0, 1]), key_heads=KH, key_dim=kd,
              value_heads=H, value_dim=vd)
    cache_ops.delta_step(**ok)
    for bad in (dict(proj=d["proj"][:, :519]), dict(proj=d["proj"].bfloat16()),
                dict(conv=d["conv"][:5]), dict(conv=d["conv"].t()), dict(state=d["state"].bfloat16()),
                dict(state=d["state"][:2]), dict(ring=d["ring"][:, :3]), dict(norm=d["norm"][:8]),
                dict(a_decay=d["a_decay"][:2]), dict(rows=ints([0])),
                dict(positions=ints([0, 1]).long()), dict(out_dtype=torch.bfloat16),
                dict(out_dtype=ops.BF16X2), dict(key_heads=3), dict(state=d["ring"])):
        with pytest.raises(ValueError):
            cache_ops.delta_step(**dict(ok, **bad))
    with pytest.raises(ValueError):       # a state where the scan keeps none
        q = torch.zeros(1, 4, 1, 96, device=DEV)
        g = torch.zeros(1, 4, 1, device=DEV)
        ops.delta_scan(q, q, q, g, g, state=torch.zeros(1, 1, 96, 96, device=DEV))


# ---------------------------------------------------------- how they are run --
def decode_inputs(seed=0, n=6, dtype=torch.bfloat16):
    rng = np.random.default_rng(seed)
    H, KV, hd, page, pages, width = 4, 2, 64, 16, 60, 8
    t = lambda *s: torch.from_numpy(rng.standard_normal(s, dtype=np.float32)).to(dtype).to(DEV)  # noqa: E731
    book = cache_ops.page_table(n + 2, width, pages, page, DEV)
    rows = ints(rng.permutation(n + 2)[:n])
    cache_ops.extend_pages(book, rows, ints(rng.integers(1, 60, n)))
    return dict(q=t(n, H, hd), k=t(n, KV, hd), v=t(n, KV, hd), gate=t(n, H, hd), norm=t(hd) * 0.1,
                pool=t(2, pages, KV, page, hd), book=book, rows=rows,
                tables=ops.rope_tables(width * page, 16, 1e4, DEV))


def decode_step(s, positions=None):
    """The attention layer's part of a step: a place for the token, q and k prepared
    and stored, attention over the row."""
    pos = cache_ops.extend_pages(s["book"], s["rows"], positions=positions)
    q = cache_ops.prepare_paged(s["q"], s["k"], s["v"], s["norm"], s["norm"], s["tables"], 16, 1e-6,
                                s["rows"], pos, s["book"].table, s["pool"][0], s["pool"][1])
    return cache_ops.paged_attention(q, s["pool"][0], s["pool"][1], s["book"].table, s["rows"], pos,
                                     0.125, gate=s["gate"])


@pytest.mark.gpu
def test_captured_step():
    """A step recorded into a graph and replayed, with eager work between, gives what
    the eager steps give: the positions move on the device."""
    a, b = decode_inputs(), decode_inputs()
    pos = torch.empty(6, dtype=torch.int32, device=DEV)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        decode_step(b)                          # lazy initialisation outside the capture
        eager = [decode_step(a)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = decode_step(b, pos)
    for _ in range(5):
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        eager.append(decode_step(a))
        assert torch.equal(got, eager[-1])
        assert torch.equal(a["book"].table, b["book"].table)
        assert torch.equal(a["pool"], b["pool"])
    assert not torch.equal(eager[1], eager[2])


@pytest.mark.gpu
def test_two_captured_graphs():
    """Two caches' graphs that end, fork, move and continue rows through workspaces of
    their own, replayed in turn, with eager work between."""
    H, KV, hd, page, width, pages = 8, 2, 256, 64, 12, 60
    parents, children, rows = ints([0, 1, 2]), ints([3, 4, 5]), ints(range(6))

    def inputs(seed):
        rng = np.random.default_rng(seed)
        t = lambda *s: torch.from_numpy(rng.standard_normal(s, dtype=np.float32)).bfloat16().to(DEV)  # noqa: E731
        book = cache_ops.page_table(6, width, pages, page, DEV)
        cache_ops.extend_pages(book, parents, ints([300, 511, 70 + seed]))
        return dict(q=t(6, H, hd), k=t(6, KV, hd), v=t(6, KV, hd), gate=t(6, H, hd),
                    norm=t(hd) * 0.1, pool=t(2, pages, KV, page, hd), book=book, rows=rows,
                    tables=ops.rope_tables(width * page, 16, 1e4, DEV), flag=flag())

    def cycle(s):
        cache_ops.free_pages(s["book"], children, error_flag=s["flag"])
        cache_ops.fork_pages(s["book"], parents, children, s["pool"], error_flag=s["flag"])
        cache_ops.compact_pages(s["book"], s["pool"])
        cache_ops.copy_pages(s["pool"], ints_50, ints_51, error_flag=s["flag"])
        return decode_step(s)

    ints_50, ints_51 = ints([0, -1, 7]), ints([51, 3, 52])     # pages beyond those in use
    lib = _lib.lib()
    assert lib.qdc_pages_fork_workspace(3, page, 2, KV, 2 * hd) > 0
    assert lib.qdc_paged_attention_workspace(6, H, KV, hd, width, page, BF16) > 0
    twins, held = [inputs(0), inputs(1)], [inputs(0), inputs(1)]
    stream = torch.cuda.Stream()
    graphs, outs, eager = [], [], []
    with torch.cuda.stream(stream):
        for h, w in zip(held, twins):
            cycle(h)
            eager.append(cycle(w))
    torch.cuda.synchronize()
    for h in held:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(cycle(h))
        graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
        got = [o.clone() for o in outs]
        torch.cuda.synchronize()
        for g, h, w in zip(got, held, twins):
            assert torch.equal(g, cycle(w)) and torch.isfinite(g).all()
            for x, y in zip(h["book"][:4], w["book"][:4]):
                assert torch.equal(x, y)
            assert torch.equal(h["pool"], w["pool"])
            assert h["flag"].item() == w["flag"].item() == 0
    assert not torch.equal(got[0], got[1])


@pytest.mark.gpu
def test_other_stream_and_same_results():
    """On a side stream the kernels wait for that stream's work alone, and two runs give
    the same bits."""
    want = decode_step(decode_inputs(7))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        s = decode_inputs(7)
        big = torch.randn(4096, 4096, device=DEV)
        for _ in range(20):
            big = big @ big * 1e-3
        s["q"] = s["q"] + 0.0 * big[0, 0].bfloat16()     # behind the products
        got = decode_step(s)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(want, got)


@pytest.mark.gpu
def test_two_threads():
    """Two host threads, each with a stream and a cache of its own."""
    from concurrent.futures import ThreadPoolExecutor

    def steps(seed):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            s = decode_inputs(seed)
            out = [decode_step(s) for _ in range(30)]
        stream.synchronize()
        return torch.stack(out)

    want = [steps(3), steps(4)]
    with ThreadPoolExecutor(2) as pool:
        got = list(pool.map(steps, (3, 4)))
    assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Pages whose byte offsets, and element offsets, pass 2^32."""
    hd, page, KV = 256, 256, 2
    pages = (1 << 32) // (KV * page * hd) + 3             # 4.3e9 elements of bf16 a tensor
    free = torch.cuda.mem_get_info()[0]
    if free < 5 * pages * KV * page * hd:
        pytest.skip("needs 22 GB of device memory")
    k = torch.zeros((pages, KV, page, hd), dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    rng = np.random.default_rng(0)
    t = lambda *s: torch.from_numpy(rng.standard_normal(s, dtype=np.float32)).bfloat16().to(DEV)  # noqa: E731
    table = ints([pages - 1, 0, pages - 2]).view(1, 3)
    T = 600
    q, kn, vn, norm = t(T, 4, hd), t(T, KV, hd), t(T, KV, hd), t(hd) * 0.1
    rows, pos = ints([0] * T), ints(range(T))
    qp = cache_ops.prepare_paged(q, kn, vn, norm, norm, None, 0, 1e-6, rows, pos, table, k, v)
    got = cache_ops.paged_attention(qp[-3:], k, v, table, rows[-3:], pos[-3:], 0.0625)
    small = torch.stack([x[[pages - 1, 0, pages - 2]] for x in (k, v)])
    want = cache_ops.paged_attention(qp[-3:], small[0], small[1], ints([0, 1, 2]).view(1, 3),
                                     rows[-3:], pos[-3:], 0.0625)
    assert torch.equal(got, want) and torch.isfinite(want).all() and want.abs().max() > 0
    assert torch.equal(small[1].transpose(1, 2).reshape(-1, KV, hd)[:T], vn)
