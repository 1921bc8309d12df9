"""The 4-bit K/V cache and attention over it on the GPU, against numpy in 64 bits: the cache to the
bit, attention within what the roundings of its definition allow (kvref.tolerance)."""
import ctypes
import sys

import numpy as np
import pytest

import arf_amd
import kvref
from arf_amd import arfq

pytestmark = pytest.mark.gpu


def _say(*a):
    print("case:", *a, flush=True)
    sys.stdout.flush()


class Batch:
    """Sequences of `lens` cached tokens whose last `news` are the step's, on shuffled pages."""

    def __init__(self, ctx, lens, news, page, rng, use_start=True, spare=0):
        self.lens, self.news, self.page = lens, news, page
        need = [-(-max(ln, 0) // page) for ln in lens]
        self.n_pages = max(1, sum(need) + spare)
        ids = rng.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((len(lens), max(1, max(need))), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = ids[at:at + n]
            at += n
        self.start = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        self.tokens = int(self.start[-1])
        self.d_table, self.d_len = ctx.to_device(self.table), ctx.to_device(np.array(lens, np.int32))
        self.d_start = ctx.to_device(self.start)
        self.seqs = arf_amd.KVSeqs(self.d_table, self.d_len, self.d_start if use_start else None,
                                   self.tokens if use_start else None)
        whole = np.concatenate([[0], np.cumsum(np.maximum(lens, 0))]).astype(np.int32)
        self.whole_start = whole
        self.d_whole = ctx.to_device(whole)
        self.whole = arf_amd.KVSeqs(self.d_table, self.d_len, self.d_whole, int(whole[-1]))

    def cached(self, b):
        return slice(self.whole_start[b], self.whole_start[b + 1])


def _rows(rng, n, heads, dim, dtype, outliers=True):
    x = rng.standard_normal((n, heads, dim)).astype(np.float32)
    if outliers:
        x[:, :, rng.integers(0, dim, 3)] *= 8
    return x.astype(dtype)


def _filled(ctx, kv, batch, rng, dtype=np.float16):
    rows = int(batch.whole_start[-1])
    k, v = (_rows(rng, rows, kv.heads, kv.head_dim, dtype, o) for o in (True, False))
    ctx.kv_write(kv, batch.whole, ctx.to_device(k), ctx.to_device(v))
    return kvref.held_pair(k, v)


def _attend(ctx, kv, batch, q, out_dtype, scale, **kw):
    tokens, hq, dim = q.shape
    out = ctx.to_device(np.full(q.shape, 7, out_dtype))
    ctx.kv_attention(kv, batch.seqs, ctx.to_device(q), out, hq, scale, **kw)
    return out.numpy()


def _check(batch, got, q, hk, hv, scale, absent=None, **kw):
    f16 = got.dtype == np.float16 and q.dtype == np.float16
    worst = 0.0
    for b, (ln, n) in enumerate(zip(batch.lens, batch.news)):
        rows = slice(batch.start[b], batch.start[b + 1])
        c = batch.cached(b)
        want, mag, eps, floor = kvref.attention(q[rows], hk[c], hv[c], scale, absent=None if absent is None else absent[b], **kw)
        g = got[rows].astype(np.float64)
        assert np.array_equal(np.isnan(g), np.isnan(want)), (b, ln, n)
        ok = ~np.isnan(want)
        tol = kvref.tolerance(want, mag, eps, floor, max(ln, 0), f16)
        if got.dtype == np.float16 and not f16:
            tol = tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
        off = np.abs(g - want)
        worst = max(worst, float((off / tol)[ok].max()) if ok.any() else 0.0)
        assert (off[ok] <= tol[ok]).all(), (b, ln, n, float((off / tol)[ok].max()))
    print("largest share of the tolerance", worst, flush=True)


# ---- the cache ----

@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,page,dtype", [(1, 16, np.float32), (3, 48, np.float16), (8, 256, np.float32)])
def test_write_and_read_to_the_bit(gpu_ctx, dim, heads, page, dtype):
    _say("write/read", dim, heads, page, np.dtype(dtype).name)
    rng = np.random.default_rng(dim + heads + page)
    batch = Batch(gpu_ctx, [1, 300, 0, 17, 97], [1, 300, 1, 5, 97], page, rng, spare=2)
    kv = gpu_ctx.kv_cache(heads, dim, page, batch.n_pages)
    k, v = (_rows(rng, batch.tokens, heads, dim, dtype) for _ in "kv")
    # small, large, zero and tiny rows; exact halves of a step; +-0
    k[3] *= 1e-3
    k[4] = 0
    k[5] = (np.arange(dim) % 17 - 8) / 2.0
    v[6] *= 100
    v[7] = dtype(-0.0)
    if dtype == np.float32:
        k[8] *= 1e-7
        v[9] *= 1e6  # held as +-65280
        v[10] *= 1e30
        k[11] *= 1e-38
    gpu_ctx.kv_write(kv, batch.seqs, gpu_ctx.to_device(k), gpu_ctx.to_device(v))
    hk, hv = kvref.held_pair(k, v)
    nowhere = batch.start[2]  # the idle slot's row
    for out in (np.float32, np.float16):
        dk, dv = (gpu_ctx.to_device(np.full(k.shape, 5, out)) for _ in "kv")
        gpu_ctx.kv_read(kv, batch.seqs, dk, dv)
        for got, want in ((dk.numpy(), hk), (dv.numpy(), hv)):
            assert (got[nowhere] == 5).all()
            rest = np.arange(batch.tokens) != nowhere
            assert np.array_equal(got[rest].astype(np.float64), want[rest])


def test_scales_over_every_exponent(gpu_ctx):
    # one row for every exponent of f32 and some mantissas: scales' ties, f16's subnormals, the largest
    _say("scales")
    rng = np.random.default_rng(3)
    top = np.exp2(np.arange(-60, 40, dtype=np.float64))[:, None] * (1 + np.array([0, 1, 2, 3, 127, 128, 129, 255]) / 256
                                                                 + np.array([0, 1, -1])[:, None] * 2.0 ** -23).ravel()
    top = top.ravel().astype(np.float32)
    x = (rng.uniform(-1, 1, (top.size, 1, 64)) * top[:, None, None]).astype(np.float32)
    x[:, 0, ::32] = top[:, None] * np.where(np.arange(top.size) % 2, 1, -1)[:, None]
    x[:, 0, 5::32] = x[:, 0, ::32] * 0.5  # q = -4, and ties where the scale was rounded
    batch = Batch(gpu_ctx, [top.size], [top.size], 64, rng)
    kv = gpu_ctx.kv_cache(1, 64, 64, batch.n_pages)
    dx = gpu_ctx.to_device(x)
    gpu_ctx.kv_write(kv, batch.seqs, dx, dx)
    dk, dv = gpu_ctx.empty(x.shape, np.float32), gpu_ctx.empty(x.shape, np.float32)
    gpu_ctx.kv_read(kv, batch.seqs, dk, dv)
    want = kvref.held(x)
    assert np.array_equal(dk.numpy().astype(np.float64), want)
    assert np.array_equal(dv.numpy().astype(np.float64), want)


def test_strided_rows_and_untouched_neighbours(gpu_ctx):
    # k and v as columns of a fused qkv product; what is not a row's stays
    _say("strides")
    rng = np.random.default_rng(4)
    heads, dim, hq = 2, 96, 6
    width = (hq + 2 * heads) * dim
    batch = Batch(gpu_ctx, [40, 33], [3, 33], 16, rng)
    kv = gpu_ctx.kv_cache(heads, dim, 16, batch.n_pages)
    qkv = rng.standard_normal((batch.tokens + 2, width)).astype(np.float32)  # two rows of no sequence behind
    d = gpu_ctx.to_device(qkv)
    seqs = arf_amd.KVSeqs(batch.d_table, batch.d_len, batch.d_start, batch.tokens + 2)
    gpu_ctx.kv_write(kv, seqs, d.columns(hq * dim), d.columns((hq + heads) * dim), width, width)
    full = gpu_ctx.to_device(np.full((batch.tokens + 2, width), 9, np.float32))
    gpu_ctx.kv_read(kv, seqs, full.columns(hq * dim), full.columns((hq + heads) * dim), width, width)
    got = full.numpy()
    assert (got[batch.tokens:] == 9).all() and (got[:, :hq * dim] == 9).all()
    k = qkv[:batch.tokens, hq * dim:(hq + heads) * dim].reshape(-1, heads, dim)
    v = qkv[:batch.tokens, (hq + heads) * dim:].reshape(-1, heads, dim)
    want = np.concatenate([kvref.held(k).reshape(batch.tokens, -1), kvref.held(v).reshape(batch.tokens, -1)], 1)
    assert np.array_equal(got[:batch.tokens, hq * dim:].astype(np.float64), want)
    # the other tokens of the first sequence were never written: zeros
    dk, dv = (gpu_ctx.empty((73, heads, dim), np.float32) for _ in "kv")
    gpu_ctx.kv_read(kv, batch.whole, dk, dv)
    assert (dk.numpy()[:37] == 0).all() and (dv.numpy()[:37] == 0).all()
    assert np.array_equal(dk.numpy()[37:40].astype(np.float64), kvref.held(k[:3]))
    # attention reads q from the same rows, and leaves rows of no sequence
    out = gpu_ctx.to_device(np.full((batch.tokens + 2, hq * dim + 32), 9, np.float32))
    gpu_ctx.kv_attention(kv, seqs, d, out, hq, 0.1, q_stride=width, out_stride=hq * dim + 32)
    o = out.numpy()
    assert (o[batch.tokens:] == 9).all() and (o[:, hq * dim:] == 9).all()
    q = qkv[:batch.tokens, :hq * dim].reshape(-1, hq, dim)
    _check(batch, np.ascontiguousarray(o[:batch.tokens, :hq * dim]).reshape(q.shape), q, dk.numpy().astype(np.float64),
           dv.numpy().astype(np.float64), 0.1)


def test_values_that_are_not_finite(gpu_ctx):
    # a NaN or an infinity in a row: its key is NaN, rows that attend to it are, others are not
    _say("not finite")
    rng = np.random.default_rng(5)
    heads, dim = 2, 64
    batch = Batch(gpu_ctx, [90], [70], 16, rng)
    kv = gpu_ctx.kv_cache(heads, dim, 16, batch.n_pages)
    k, v = (_rows(rng, 90, heads, dim, np.float16) for _ in "kv")
    k[60, 0, 5], v[75, 1, 40], v[80, 0, 3], k[85, 1, 63] = np.nan, np.inf, -np.inf, np.inf
    gpu_ctx.kv_write(kv, batch.whole, gpu_ctx.to_device(k), gpu_ctx.to_device(v))
    dk, dv = (gpu_ctx.empty(k.shape, np.float32) for _ in "kv")
    gpu_ctx.kv_read(kv, batch.whole, dk, dv)
    hk, hv = kvref.held_pair(k, v)
    assert np.array_equal(dk.numpy().astype(np.float64), hk, equal_nan=True) and np.isnan(hk[75, 1]).all()
    assert np.array_equal(dv.numpy().astype(np.float64), hv)
    for dtype in (np.float16, np.float32):
        q = _rows(rng, 70, 4, dim, dtype)
        got = _attend(gpu_ctx, kv, batch, q, dtype, 0.125)
        _check(batch, got, q, hk, hv, 0.125)
        assert not np.isnan(got[:40]).any() and np.isnan(got[40:, :2]).all() and np.isnan(got[55:, 2:]).all()
        # the window leaves them behind
        got = _attend(gpu_ctx, kv, batch, q, dtype, 0.125, window=3)
        _check(batch, got, q, hk, hv, 0.125, window=3)
        assert not np.isnan(got[69]).any()
    q = _rows(rng, 70, 4, dim, np.float32)
    q[3, 1, 2], q[8, 2, 0] = np.nan, np.inf
    got = _attend(gpu_ctx, kv, batch, q, np.float32, 0.125, window=2)
    bad = np.isnan(got).any(-1)
    assert bad[3, 1] and bad[8, 2] and bad[:40].sum() == 2


def test_page_ids_outside_the_cache_name_nothing(gpu_ctx):
    _say("bad pages")
    rng = np.random.default_rng(6)
    heads, dim, page = 2, 128, 16
    batch = Batch(gpu_ctx, [200, 77], [4, 1], page, rng)
    kv = gpu_ctx.kv_cache(heads, dim, page, batch.n_pages)
    hk, hv = _filled(gpu_ctx, kv, batch, rng)
    absent = [np.zeros(200, bool), np.zeros(77, bool)]
    table = batch.table.copy()
    for b, p, i in [(0, 0, -1), (0, 3, batch.n_pages), (0, 7, 2 ** 31 - 1), (1, 4, -2 ** 31)]:
        table[b, p] = i
        absent[b][p * page:(p + 1) * page] = True
    batch.d_table.upload(table)
    for dtype in (np.float16, np.float32):
        q = _rows(rng, 5, 8, dim, dtype)
        _check(batch, _attend(gpu_ctx, kv, batch, q, dtype, 0.09), q, hk, hv, 0.09, absent=absent)
    # rows that would go to such a page are not written, or read
    k = gpu_ctx.to_device(_rows(rng, 277, heads, dim, np.float16))
    gpu_ctx.kv_write(kv, batch.whole, k, k)
    dk, dv = (gpu_ctx.to_device(np.full((277, heads, dim), 5, np.float32)) for _ in "kv")
    gpu_ctx.kv_read(kv, batch.whole, dk, dv)
    gone = np.concatenate(absent)
    assert (dk.numpy()[gone] == 5).all() and not (dk.numpy()[~gone] == 5).all(-1).any()


def test_malformed_batches_reach_nothing(gpu_ctx):
    # lengths, starts and tables that contradict each other: rows that name nothing
    _say("malformed")
    rng = np.random.default_rng(7)
    heads, dim, page = 2, 64, 32
    kv = gpu_ctx.kv_cache(heads, dim, page, 4)
    table = gpu_ctx.to_device(np.array([[0, 1], [2, 3], [1, 0]], np.int32))
    for lens, start in [([2 ** 31 - 1, -2 ** 31, 64], [0, 1, 2, 3]), ([64, 64, 64], [0, 5, 2, 6]),
                        ([64, 64, 64], [-3, 2, 4, 99]), ([10 ** 9, 64, -5], [6, 6, 6, 6]), ([1000, 1, 65], [0, 2, 4, 6])]:
        seqs = arf_amd.KVSeqs(table, gpu_ctx.to_device(np.array(lens, np.int32)),
                              gpu_ctx.to_device(np.array(start, np.int32)), 6)
        x = gpu_ctx.to_device(_rows(rng, 6, heads, dim, np.float32))
        gpu_ctx.kv_write(kv, seqs, x, x)
        y, z = (gpu_ctx.to_device(np.full((6, heads, dim), 5, np.float32)) for _ in "kv")
        gpu_ctx.kv_read(kv, seqs, y, z)
        out = gpu_ctx.to_device(np.full((6, 4, dim), 5, np.float32))
        q = gpu_ctx.to_device(_rows(rng, 6, 4, dim, np.float32))
        gpu_ctx.kv_attention(kv, seqs, q, out, 4, 0.1)
        o = out.numpy()
        rows = np.zeros(6, bool)  # of a sequence whose rows lie in the batch
        for b in range(3):
            if 0 <= start[b] < start[b + 1] <= 6:
                rows[start[b]:start[b + 1]] = True
        assert (o[~rows] == 5).all() and np.isfinite(o).all()


# ---- attention ----

LENS = [1, 2, 15, 16, 17, 31, 33, 64, 100, 255, 257, 513]


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,group,page", [(2, 1, 16), (1, 5, 48), (3, 8, 64), (1, 17, 32)])
def test_decode(gpu_ctx, dtype, dim, heads, group, page):
    _say("decode", np.dtype(dtype).name, dim, heads, group, page)
    rng = np.random.default_rng(dim + heads * 7 + group)
    batch = Batch(gpu_ctx, LENS + [0], [1] * (len(LENS) + 1), page, rng, use_start=group != 5)
    kv = gpu_ctx.kv_cache(heads, dim, page, batch.n_pages)
    hk, hv = _filled(gpu_ctx, kv, batch, rng)
    q = _rows(rng, batch.tokens, heads * group, dim, dtype)
    scale = dim ** -0.5
    got = _attend(gpu_ctx, kv, batch, q, dtype, scale)
    _check(batch, got, q, hk, hv, scale)
    assert (got[-1] == 0).all()  # the idle slot


@pytest.mark.parametrize("dtype,out", [(np.float16, np.float16), (np.float32, np.float32), (np.float16, np.float32),
                                       (np.float32, np.float16)])
@pytest.mark.parametrize("kw", [{}, dict(window=1), dict(window=37), dict(window=256, softcap=20.0), dict(causal=False),
                                dict(causal=False, window=40)])
def test_several_tokens_a_sequence(gpu_ctx, dtype, out, kw):
    _say("several", np.dtype(dtype).name, np.dtype(out).name, kw)
    rng = np.random.default_rng(11)
    heads, group, dim, page = 2, 3, 128, 16
    # some with more rows than cached tokens (the first rows are at negative positions)
    batch = Batch(gpu_ctx, [1, 40, 300, 0, 65, 129, 7], [1, 40, 9, 3, 33, 2, 12], page, rng)
    kv = gpu_ctx.kv_cache(heads, dim, page, batch.n_pages)
    hk, hv = _filled(gpu_ctx, kv, batch, rng, np.float32)
    q = _rows(rng, batch.tokens, heads * group, dim, dtype)
    got = _attend(gpu_ctx, kv, batch, q, out, 0.088, **kw)
    _check(batch, got, q, hk, hv, 0.088, **kw)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("dim,heads,group,n,length", [(64, 1, 4, 333, 333), (96, 2, 3, 150, 700), (128, 1, 5, 257, 1100),
                                                      (128, 2, 1, 400, 400), (256, 1, 2, 130, 390), (128, 1, 16, 70, 5000)])
def test_prompts(gpu_ctx, dtype, dim, heads, group, n, length):
    _say("prompt", np.dtype(dtype).name, dim, heads, group, n, length)
    rng = np.random.default_rng(n + length)
    batch = Batch(gpu_ctx, [length, 20], [n, 1], 32, rng)
    kv = gpu_ctx.kv_cache(heads, dim, 32, batch.n_pages)
    hk, hv = _filled(gpu_ctx, kv, batch, rng)
    q = _rows(rng, batch.tokens, heads * group, dim, dtype)
    scale = dim ** -0.5
    for kw in ({}, dict(window=100), dict(softcap=15.0, causal=False)):
        _check(batch, _attend(gpu_ctx, kv, batch, q, dtype, scale, **kw), q, hk, hv, scale, **kw)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("group", [1, 6])
def test_long_sequences_beside_short_ones(gpu_ctx, dtype, group):
    _say("long", np.dtype(dtype).name, group)
    rng = np.random.default_rng(13)
    batch = Batch(gpu_ctx, [40001, 3, 2000, 70], [1, 1, 2, 1], 64, rng)
    kv = gpu_ctx.kv_cache(1, 128, 64, batch.n_pages)
    hk, hv = _filled(gpu_ctx, kv, batch, rng)
    q = _rows(rng, batch.tokens, group, 128, dtype) * dtype(2)
    _check(batch, _attend(gpu_ctx, kv, batch, q, dtype, 0.09), q, hk, hv, 0.09)


def test_many_sequences(gpu_ctx):
    # more than a wave of them, some without rows of their own
    _say("many")
    rng = np.random.default_rng(14)
    lens = [int(x) for x in rng.integers(0, 90, 150)]
    news = [int(min(n, ln + 1)) for n, ln in zip(rng.integers(0, 4, 150), lens)]
    batch = Batch(gpu_ctx, lens, news, 16, rng)
    kv = gpu_ctx.kv_cache(2, 64, 16, batch.n_pages)
    hk, hv = _filled(gpu_ctx, kv, batch, rng)
    q = _rows(rng, batch.tokens, 4, 64, np.float32)
    _check(batch, _attend(gpu_ctx, kv, batch, q, np.float32, 0.125), q, hk, hv, 0.125)


@pytest.mark.parametrize("factor,scale", [(1e-30, 0.1), (1e4, 0.1), (1e4, 1e-5), (1e30, 1e-30), (1.0, -0.1), (1.0, 0.0)])
def test_magnitudes_of_q(gpu_ctx, factor, scale):
    # f32 q is scaled to f16's range by row: any size of it works; a negative and a zero scale
    _say("magnitudes", factor, scale)
    rng = np.random.default_rng(15)
    batch = Batch(gpu_ctx, [300], [3], 16, rng)
    kv = gpu_ctx.kv_cache(1, 64, 16, batch.n_pages)
    hk, hv = _filled(gpu_ctx, kv, batch, rng)
    q = (_rows(rng, 3, 2, 64, np.float32) * np.float32(factor)).astype(np.float32)
    q[1, 1] = 0
    _check(batch, _attend(gpu_ctx, kv, batch, q, np.float32, scale), q, hk, hv, scale)


def test_scores_that_rise_along_the_keys(gpu_ctx):
    # the running maximum grows at every step, or falls from the first on
    _say("rising")
    rng = np.random.default_rng(16)
    n = 700
    batch = Batch(gpu_ctx, [n, n], [1, 1], 16, rng)
    kv = gpu_ctx.kv_cache(1, 64, 16, batch.n_pages)
    k = np.zeros((2 * n, 1, 64), np.float16)
    k[:n, 0, 0] = np.arange(n) / 2
    k[n:, 0, 0] = -np.arange(n) / 2
    v = _rows(rng, 2 * n, 1, 64, np.float16)
    gpu_ctx.kv_write(kv, batch.whole, gpu_ctx.to_device(k), gpu_ctx.to_device(v))
    hk, hv = kvref.held_pair(k, v)
    for dtype in (np.float16, np.float32):
        q = np.ones((2, 4, 64), dtype)
        for scale in (0.01, 1.0, 30.0):
            _check(batch, _attend(gpu_ctx, kv, batch, q, dtype, scale), q, hk, hv, scale)


def test_same_bits_again_and_with_a_workspace(gpu_ctx):
    _say("again")
    rng = np.random.default_rng(17)
    batch = Batch(gpu_ctx, [5000, 800, 31], [2, 60, 1], 64, rng)
    kv = gpu_ctx.kv_cache(2, 128, 64, batch.n_pages)
    _filled(gpu_ctx, kv, batch, rng)
    q = _rows(rng, batch.tokens, 8, 128, np.float32)
    first = _attend(gpu_ctx, kv, batch, q, np.float32, 0.1)
    need = gpu_ctx.kv_attention_workspace(kv, batch.seqs, 8)
    ws = gpu_ctx.to_device(np.full(need // 4 + 4, np.nan, np.float32))
    for w in (None, ws, ws):
        assert np.array_equal(_attend(gpu_ctx, kv, batch, q, np.float32, 0.1, workspace=w).view(np.uint32),
                              first.view(np.uint32))
    assert np.isnan(ws.numpy()[need // 4:]).all()


def test_two_contexts_at_once(gpu_ctx):
    # a cache is its own: two contexts (streams) read and write different caches and the same one
    _say("two contexts")
    rng = np.random.default_rng(18)
    with arf_amd.Context(0) as other:
        sides = []
        for ctx in (gpu_ctx, other):
            batch = Batch(ctx, [3000, 900], [1, 1], 32, rng)
            kv = ctx.kv_cache(2, 64, 32, batch.n_pages)
            hk, hv = _filled(ctx, kv, batch, rng)
            q = _rows(rng, 2, 8, 64, np.float16)
            sides.append((ctx, batch, kv, hk, hv, q, ctx.to_device(q), ctx.empty(q.shape, np.float16)))
            ctx.sync()
        for _ in range(10):
            for ctx, batch, kv, hk, hv, q, dq, out in sides:
                ctx.kv_attention(kv, batch.seqs, dq, out, 8, 0.125)
        for ctx, batch, kv, hk, hv, q, dq, out in sides:
            _check(batch, out.numpy(), q, hk, hv, 0.125)
        ctx, batch, kv, hk, hv, q, dq, out = sides[0]
        mine = other.empty(q.shape, np.float16)
        other.kv_attention(kv, batch.seqs, dq, mine, 8, 0.125)
        assert np.array_equal(mine.numpy().view(np.uint16), out.numpy().view(np.uint16))
        for s in sides:
            s[2].free()


def test_refusals(gpu_ctx):
    _say("refusals")
    L, h = arf_amd.load_library(), gpu_ctx.handle
    E = arfq
    p = ctypes.c_void_p()
    for heads, dim, page, pages, want in [(0, 128, 64, 4, E.ARFQ_E_SHAPE), (1025, 128, 64, 4, E.ARFQ_E_SHAPE),
                                          (8, 0, 64, 4, E.ARFQ_E_SHAPE), (8, 80, 64, 4, E.ARFQ_E_UNSUPPORTED),
                                          (8, 512, 64, 4, E.ARFQ_E_UNSUPPORTED), (8, 128, 0, 4, E.ARFQ_E_SHAPE),
                                          (8, 128, 24, 4, E.ARFQ_E_SHAPE), (8, 128, 272, 4, E.ARFQ_E_SHAPE),
                                          (8, 128, 64, 0, E.ARFQ_E_SHAPE), (8, 128, 64, 2 ** 31, E.ARFQ_E_SHAPE),
                                          (1024, 256, 256, 2 ** 31 - 1, E.ARFQ_E_NOMEM)]:
        assert L.arfq_kv_create(h, heads, dim, page, pages, ctypes.byref(p)) == want, (heads, dim, page, pages)
        assert p.value is None and L.arfq_last_error(h).startswith(b"kv_create")
    assert L.arfq_kv_create(h, 8, 128, 64, 4, None) == E.ARFQ_E_INVALID
    kv = gpu_ctx.kv_cache(2, 64, 16, 4)
    assert kv.bytes_num == 4 * 2 * 16 * 2 * (32 + 4)
    table, lens = gpu_ctx.to_device(np.zeros((2, 2), np.int32)), gpu_ctx.to_device(np.array([20, 20], np.int32))
    x = gpu_ctx.to_device(np.zeros((2, 4, 64), np.float32))

    def seqs(batch=2, tokens=2, start=None, ln=lens.ptr, pages=table.ptr, most=2):
        return E._KVSeqsStruct(batch, tokens, start, ln, pages, most)

    def write(s, k=x.ptr, ks=128, v=x.ptr, vs=128, t=0, cache=kv.handle):
        return L.arfq_kv_write(h, cache, ctypes.byref(s) if s else None, k, ks, v, vs, t)

    def attend(s, hq=4, q=x.ptr, qs=256, o=x.ptr, os=256, t=0, scale=1.0, cap=0.0, win=0, ws=None, wb=0, ot=0):
        return L.arfq_kv_attention(h, kv.handle, ctypes.byref(s) if s else None, hq, q, qs, t, o, os, ot, scale, cap, win, 1,
                                   ws, wb)

    assert write(seqs()) == E.ARFQ_OK and attend(seqs()) == E.ARFQ_OK
    for s, want in [(None, E.ARFQ_E_INVALID), (seqs(ln=None), E.ARFQ_E_INVALID), (seqs(pages=None), E.ARFQ_E_INVALID),
                    (seqs(batch=-1), E.ARFQ_E_SHAPE), (seqs(tokens=-1), E.ARFQ_E_SHAPE), (seqs(most=-1), E.ARFQ_E_SHAPE),
                    (seqs(tokens=3), E.ARFQ_E_SHAPE), (seqs(most=2 ** 25 + 1), E.ARFQ_E_SHAPE),
                    (seqs(batch=2 ** 25), E.ARFQ_E_SHAPE), (seqs(batch=16385), E.ARFQ_E_SHAPE),
                    (seqs(tokens=2 ** 30, start=lens.ptr), E.ARFQ_E_SHAPE)]:
        assert write(s) == want and attend(s) == want
        assert L.arfq_kv_read(h, kv.handle, ctypes.byref(s) if s else None, x.ptr, 128, x.ptr, 128, 0) == want
    # nothing to do: nothing is looked at
    for s in (seqs(tokens=0), seqs(batch=0, tokens=0, ln=None, pages=None)):
        assert write(s, k=None) == E.ARFQ_OK and attend(s, q=None) == E.ARFQ_OK
    for kw, want in [(dict(k=None), E.ARFQ_E_INVALID), (dict(v=None), E.ARFQ_E_INVALID), (dict(t=2), E.ARFQ_E_INVALID),
                     (dict(ks=127), E.ARFQ_E_SHAPE), (dict(vs=130), E.ARFQ_E_INVALID), (dict(k=x.ptr + 4), E.ARFQ_E_INVALID),
                     (dict(ks=2 ** 41), E.ARFQ_E_SHAPE), (dict(cache=None), E.ARFQ_E_INVALID)]:
        assert write(seqs(), **kw) == want, kw
    nan, inf = float("nan"), float("inf")
    for kw, want in [(dict(hq=3), E.ARFQ_E_SHAPE), (dict(hq=0), E.ARFQ_E_SHAPE), (dict(q=None), E.ARFQ_E_INVALID),
                     (dict(o=None), E.ARFQ_E_INVALID), (dict(qs=255), E.ARFQ_E_SHAPE), (dict(os=258), E.ARFQ_E_INVALID),
                     (dict(t=5), E.ARFQ_E_INVALID), (dict(ot=-1), E.ARFQ_E_INVALID), (dict(scale=nan), E.ARFQ_E_INVALID),
                     (dict(scale=inf), E.ARFQ_E_INVALID), (dict(cap=-1.0), E.ARFQ_E_INVALID), (dict(cap=inf), E.ARFQ_E_INVALID),
                     (dict(win=-1), E.ARFQ_E_SHAPE)]:
        assert attend(seqs(), **kw) == want, kw
        assert L.arfq_last_error(h).startswith(b"kv_attention")
    # a workspace for more keys than one piece has
    assert attend(seqs(most=2 ** 20), ws=x.ptr, wb=16) == E.ARFQ_E_SHAPE and b"workspace" in L.arfq_last_error(h)
    assert attend(seqs(most=2 ** 20), ws=x.ptr + 4, wb=2 ** 40) == E.ARFQ_E_SHAPE
    with pytest.raises(ValueError):
        gpu_ctx.kv_write(kv, arf_amd.KVSeqs(table, lens), x, gpu_ctx.empty((2, 2, 64), np.float16))
    kv.free()
