"""The 4-bit K/V cache and its attention at the ends of what the header allows: batches that contradict
themselves, the largest calls, extreme factors, every variant that a size selects."""
import ctypes

import numpy as np
import pytest

import arf_amd
import kvref
from arf_amd import arfq
from test_gpu_kv import Batch, _attend, _check, _filled, _rows, _say

pytestmark = pytest.mark.gpu


# ---- a start that decreases ----

@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("first,lens", [([0, 16], [100]), ([0, 3, 16], [20000, 300]), ([0, 3, 3, 15], [300, 7, 5000])])
@pytest.mark.parametrize("heads,group", [(8, 4), (2, 9)])
def test_no_rows_from_where_start_decreases(gpu_ctx, dtype, first, lens, heads, group):
    # `first` rises, and is followed by sequences that name the same 16 rows again and again, some of many
    # keys: more work items than the call's rows make.  The first ones' rows are right, all else is left
    _say("decreasing start", np.dtype(dtype).name, first, lens, heads, group)
    rng = np.random.default_rng(len(first) + heads)
    dim, page, most, tokens, batch = 128, 64, 2048, 16, 90
    n = len(lens)
    good = Batch(gpu_ctx, lens, list(np.diff(first)), page, rng)
    kv = gpu_ctx.kv_cache(heads, dim, page, good.n_pages)
    hk, hv = _filled(gpu_ctx, kv, good, rng)
    table = rng.integers(0, good.n_pages, (batch, most)).astype(np.int32)
    table[:n, :good.table.shape[1]] = good.table
    start = (first + [0, 16] * batch)[:batch + 1]
    every = lens + [100] * (batch - n - 1) + [most * page]
    seqs = arf_amd.KVSeqs(gpu_ctx.to_device(table), gpu_ctx.to_device(np.array(every, np.int32)),
                          gpu_ctx.to_device(np.array(start, np.int32)), tokens)
    q = _rows(rng, tokens, heads * group, dim, dtype)
    dq, out = gpu_ctx.to_device(q), gpu_ctx.to_device(np.full((tokens + 64, heads * group, dim), 9, dtype))
    need = gpu_ctx.kv_attention_workspace(kv, seqs, heads * group)
    ws = gpu_ctx.to_device(np.full(need // 4, 0x7f7f7f7f, np.int32))
    gpu_ctx.kv_attention(kv, seqs, dq, out, heads * group, 0.09, workspace=ws)
    got, rows = out.numpy(), first[-1]
    assert (got[rows:] == 9).all()
    _check(good, got[:rows], q[:rows], hk, hv, 0.09)


def test_rows_written_and_read_where_start_decreases(gpu_ctx):
    _say("decreasing start, write and read")
    rng = np.random.default_rng(41)
    heads, dim, page, batch, tokens = 2, 96, 16, 140, 16
    kv = gpu_ctx.kv_cache(heads, dim, page, 2 * batch)
    table = np.arange(2 * batch, dtype=np.int32).reshape(batch, 2)
    lens = np.full(batch, 20, np.int32)
    for at, first in ((1, [0, 16]), (64, [0] * 64 + [11]), (100, [0] * 30 + [3] * 60 + [14] * 11)):
        start = np.array((first + [0, 16] * batch)[:batch + 1], np.int32)
        seqs = arf_amd.KVSeqs(gpu_ctx.to_device(table), gpu_ctx.to_device(lens), gpu_ctx.to_device(start), tokens)
        k, v = (_rows(rng, tokens, heads, dim, np.float32) for _ in "kv")
        gpu_ctx.kv_write(kv, seqs, gpu_ctx.to_device(k), gpu_ctx.to_device(v))
        rows = first[-1]
        dk, dv = (gpu_ctx.to_device(np.full(k.shape, 5, np.float32)) for _ in "kv")
        gpu_ctx.kv_read(kv, seqs, dk, dv)
        for got, x in ((dk.numpy(), k), (dv.numpy(), v)):
            assert np.array_equal(got[:rows].astype(np.float64), kvref.held(x[:rows])) and (got[rows:] == 5).all()
        # what else the cache holds is as it was: the rows' own places hold them, the others zeros
        whole = arf_amd.KVSeqs(seqs.pages, seqs.lens, gpu_ctx.to_device(np.arange(batch + 1, dtype=np.int32) * 20), batch * 20)
        wk, wv = (gpu_ctx.empty((batch, 20, heads, dim), np.float32) for _ in "kv")
        gpu_ctx.kv_read(kv, whole, wk, wv)
        gk = wk.numpy()
        for b in range(batch):
            n = max(0, start[b + 1] - start[b]) if b < at else 0
            assert not gk[b, :20 - n].any()
            assert n == 0 or np.array_equal(gk[b, 20 - n:].astype(np.float64), kvref.held(k[start[b]:start[b] + n]))
        # (written back to zeros for the next)
        zero = gpu_ctx.to_device(np.zeros((batch * 20, heads, dim), np.float32))
        gpu_ctx.kv_write(kv, whole, zero, zero)
    kv.free()


# ---- the largest calls ----

def _seqs(ctx, table, lens, start, tokens):
    return arf_amd.KVSeqs(ctx.to_device(np.asarray(table, np.int32)), ctx.to_device(np.asarray(lens, np.int32)),
                          ctx.to_device(np.asarray(start, np.int32)), tokens)


@pytest.mark.parametrize("dim,heads", [(64, 1), (96, 2), (128, 1), (256, 4)])
def test_as_many_rows_as_a_call_takes(gpu_ctx, dim, heads):
    # 2^30 rows of k and v, all but the first few of no sequence (so there is no memory behind them):
    # more threads than one dimension of a grid has
    _say("2^30 rows", dim, heads)
    rng = np.random.default_rng(dim)
    L, h = arf_amd.load_library(), gpu_ctx.handle
    kv = gpu_ctx.kv_cache(heads, dim, 16, 8)
    seqs = _seqs(gpu_ctx, [[3, 1], [5, 0]], [20, 9], [2, 22, 31], 2 ** 30 // heads)
    k, v = (_rows(rng, 31, heads, dim, np.float16) for _ in "kv")
    dk, dv, w = gpu_ctx.to_device(k), gpu_ctx.to_device(v), heads * dim
    assert L.arfq_kv_write(h, kv.handle, seqs.ref, dk.ptr, w, dv.ptr, w, 1) == arfq.ARFQ_OK, L.arfq_last_error(h)
    for dtype, t in ((np.float32, 0), (np.float16, 1)):
        ok, ov = (gpu_ctx.to_device(np.full((40, heads, dim), 5, dtype)) for _ in "kv")
        assert L.arfq_kv_read(h, kv.handle, seqs.ref, ok.ptr, w, ov.ptr, w, t) == arfq.ARFQ_OK, L.arfq_last_error(h)
        for got, x in ((ok.numpy(), k), (ov.numpy(), v)):
            assert np.array_equal(got[2:31].astype(np.float64), kvref.held(x[2:])) and (got[:2] == 5).all() and (got[31:] == 5).all()
    kv.free()


def test_rows_behind_the_first_2_32_threads(gpu_ctx):
    # the last rows of a write that takes more than 2^32 threads (k and v the same 64 GiB, most of it of no sequence)
    _say("2^27 rows of 256")
    dim, rows = 256, 2 ** 27 + 9
    if gpu_ctx.memory()[1] < 100 * 2 ** 30:
        pytest.skip("64 GiB of rows")
    L, h = arf_amd.load_library(), gpu_ctx.handle
    rng = np.random.default_rng(42)
    kv = gpu_ctx.kv_cache(1, dim, 16, 2)
    p = ctypes.c_void_p()
    assert L.arfq_dev_malloc(h, rows * dim * 2, ctypes.byref(p)) == arfq.ARFQ_OK
    try:
        x = _rows(rng, 20, 1, dim, np.float16)
        assert L.arfq_copy_h2d(h, p.value + (rows - 20) * dim * 2, x.ctypes.data, x.nbytes) == arfq.ARFQ_OK
        seqs = _seqs(gpu_ctx, [[1, 0]], [20], [0, rows], rows)
        assert L.arfq_kv_write(h, kv.handle, seqs.ref, p.value, dim, p.value, dim, 1) == arfq.ARFQ_OK, L.arfq_last_error(h)
        dk, dv = (gpu_ctx.empty(x.shape, np.float32) for _ in "kv")
        gpu_ctx.kv_read(kv, _seqs(gpu_ctx, [[1, 0]], [20], [0, 20], 20), dk, dv)
        assert np.array_equal(dk.numpy().astype(np.float64), kvref.held(x)) and np.array_equal(dv.numpy(), dk.numpy())
    finally:
        L.arfq_dev_free(h, p.value)
        kv.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_as_many_workgroups_as_attention_takes(gpu_ctx, dtype):
    # 1024 heads, 2048 sequences, 2^30 rows of q: a prompt, a token, and rows of no sequence
    _say("2^30 rows of q", np.dtype(dtype).name)
    heads, dim, batch = 1024, 64, 2048
    rng = np.random.default_rng(43)
    L, h = arf_amd.load_library(), gpu_ctx.handle
    kv = gpu_ctx.kv_cache(heads, dim, 16, 8)
    table = np.full((batch, 6), -1)
    table[0], table[batch - 1, 0] = [4, 1, 7, 0, 2, 6], 3
    lens = np.zeros(batch, np.int32)
    lens[0], lens[-1] = 90, 12
    start = np.full(batch + 1, 80)
    start[0], start[-1] = 0, 81
    filled = _seqs(gpu_ctx, table[[0, -1]], [90, 12], [0, 90, 102], 102)
    k, v = (_rows(rng, 102, heads, dim, np.float16) for _ in "kv")
    gpu_ctx.kv_write(kv, filled, gpu_ctx.to_device(k), gpu_ctx.to_device(v))
    q = _rows(rng, 81, heads, dim, dtype)
    dq, out = gpu_ctx.to_device(q), gpu_ctx.to_device(np.full((96, heads, dim), 9, dtype))
    w, t = heads * dim, int(dtype == np.float16)
    seqs = _seqs(gpu_ctx, table, lens, start, 2 ** 20)
    assert L.arfq_kv_attention(h, kv.handle, seqs.ref, heads, dq.ptr, w, t, out.ptr, w, t, 0.125, 0.0, 0, 1,
                               None, 0) == arfq.ARFQ_OK, L.arfq_last_error(h)
    got = out.numpy()
    assert (got[81:] == 9).all()
    hk, hv = kvref.held_pair(k, v)
    some = [0, 1, 500, 1023]  # heads

    class One:
        lens, news, start = [90, 12], [80, 1], [0, 80, 81]

        @staticmethod
        def cached(b):
            return slice(0, 90) if b == 0 else slice(90, 102)

    _check(One, np.ascontiguousarray(got[:81, some]), np.ascontiguousarray(q[:, some]), hk[:, some], hv[:, some], 0.125)
    kv.free()


# ---- factors of the scores ----

def _filled_batch(ctx, rng, dim):
    batch = Batch(ctx, [300, 700, 20], [3, 40, 1], 16, rng)
    kv = ctx.kv_cache(1, dim, 16, batch.n_pages)
    return batch, kv, *_filled(ctx, kv, batch, rng)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("cap", [1e18, 1.9e19, 1e33, 1e35, 1e37, 2e38, 3.4028234e38])
def test_caps_that_no_score_comes_near(gpu_ctx, dtype, cap):
    # tanh(v) is v: the attention of no cap (kvref with none, within its tolerance of that)
    _say("large cap", np.dtype(dtype).name, cap)
    rng = np.random.default_rng(44)
    batch, kv, hk, hv = _filled_batch(gpu_ctx, rng, 64)
    q = _rows(rng, batch.tokens, 3, 64, dtype)
    q[1, 0] = 0
    for scale in (0.125, -3.0, 1e-30):
        _check(batch, _attend(gpu_ctx, kv, batch, q, dtype, scale, softcap=cap), q, hk, hv, scale)
    kv.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("cap", [1e-45, 1e-40, 1e-38, 1e-20, 1e-3])
def test_caps_that_leave_nothing(gpu_ctx, dtype, cap):
    # every score within cap of 0: the mean of the values
    _say("small cap", np.dtype(dtype).name, cap)
    rng = np.random.default_rng(45)
    batch, kv, hk, hv = _filled_batch(gpu_ctx, rng, 128)
    q = _rows(rng, batch.tokens, 3, 128, dtype)
    q[1, 0] = 0
    for scale in (0.125, -1e30, 0.0):
        _check(batch, _attend(gpu_ctx, kv, batch, q, dtype, scale, softcap=cap), q, hk, hv, scale, softcap=cap)
    kv.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("cap", [0.0, 1.0])
def test_the_largest_scale_of_products_that_are_zero(gpu_ctx, dtype, cap):
    _say("large scale", np.dtype(dtype).name, cap)
    rng = np.random.default_rng(46)
    batch, kv, hk, hv = _filled_batch(gpu_ctx, rng, 96)
    q = np.zeros((batch.tokens, 3, 96), dtype)
    for scale in (3.4e38, -3.4e38):
        _check(batch, _attend(gpu_ctx, kv, batch, q, dtype, scale, softcap=cap), q, hk, hv, scale, softcap=cap)
    kv.free()


# ---- the largest values ----

@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_values_beyond_the_largest_scale(gpu_ctx, dim):
    # of the sign of the group's extreme 65280, of the other 57120 (codes end at 7)
    _say("largest values", dim)
    batch = Batch(gpu_ctx, [4], [4], 16, np.random.default_rng(47))
    kv = gpu_ctx.kv_cache(1, dim, 16, batch.n_pages)
    x = np.zeros((4, 1, dim), np.float32)
    x[0, 0, ::32], x[0, 0, 1::32] = 1e6, -1e6
    x[1, 0, 2::32], x[1, 0, 3::32] = -2e6, 1e6
    x[2, 0, 4::32], x[2, 0, 5::32] = 3e38, -65281
    x[3, 0, 6::32], x[3, 0, 7::32] = -65280, 57121
    want = np.zeros_like(x)
    want[0, 0, ::32], want[0, 0, 1::32] = 65280, -57120
    want[1, 0, 2::32], want[1, 0, 3::32] = -65280, 57120
    want[2, 0, 4::32], want[2, 0, 5::32] = 65280, -57120
    want[3, 0, 6::32], want[3, 0, 7::32] = -65280, 57120
    assert np.array_equal(kvref.held(x), want)
    d = gpu_ctx.to_device(x)
    gpu_ctx.kv_write(kv, batch.seqs, d, d)
    for dtype in (np.float32, np.float16):
        dk, dv = gpu_ctx.empty(x.shape, dtype), gpu_ctx.empty(x.shape, dtype)
        gpu_ctx.kv_read(kv, batch.seqs, dk, dv)
        assert np.array_equal(dk.numpy(), want.astype(dtype)) and np.array_equal(dv.numpy(), want.astype(dtype))
    kv.free()


# ---- every variant that a size selects ----

@pytest.mark.parametrize("dim,heads,rows", [(64, 7, 262144), (96, 3, 131072), (128, 5, 131072), (256, 3, 65536)])
def test_reads_that_fill_the_chip(gpu_ctx, dim, heads, rows):
    # from `rows` rows on a wave reads several sets of rows: just above it, ragged, an idle slot, an odd number of
    # rows, both types; and f32 from 192 MiB on, where the stores pass the caches
    _say("large reads", dim, heads)
    rng = np.random.default_rng(dim + heads)
    for least in (rows, (192 << 20) // (8 * dim)):
        tokens = (least + heads - 1) // heads + 2
        tokens += tokens % 2  # (odd with the idle slot's)
        cuts = np.sort(rng.choice(np.arange(1, tokens), 9, replace=False))
        lens = np.diff(np.concatenate([[0], cuts, [tokens]])).tolist()
        lens[4:4] = [0]  # (its row is nobody's)
        news = [max(1, n) for n in lens]
        batch = Batch(gpu_ctx, lens, news, 48, rng)
        kv = gpu_ctx.kv_cache(heads, dim, 48, batch.n_pages)
        few = _rows(rng, 997, heads, dim, np.float16)
        pick = rng.integers(0, 997, (2, batch.tokens))
        dk, dv = (gpu_ctx.to_device(few[p]) for p in pick)
        gpu_ctx.kv_write(kv, batch.seqs, dk, dv)
        held = kvref.held(few)
        nowhere = batch.start[4]
        rest = np.arange(batch.tokens) != nowhere
        for dtype in (np.float32, np.float16):
            dk, dv = (gpu_ctx.to_device(np.full((batch.tokens, heads, dim), 5, dtype)) for _ in "kv")
            gpu_ctx.kv_read(kv, batch.seqs, dk, dv)
            for d, p in ((dk, pick[0]), (dv, pick[1])):
                got = d.numpy()
                assert (got[nowhere] == 5).all() and np.array_equal(got[rest], held.astype(dtype)[p[rest]])
        kv.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("n,length,kw", [(1153, 1153, {}), (2100, 2100, {}), (1100, 1400, dict(window=500)),
                                         (1500, 1600, dict(causal=False))])
def test_one_prompt_of_more_tiles_than_units(gpu_ctx, dtype, n, length, kw):
    # 32 K/V heads: eight workgroups a head at a time, every other round of a prompt's tiles backwards
    _say("tile rounds", np.dtype(dtype).name, n, length, kw)
    rng = np.random.default_rng(n)
    heads, dim, some = 32, 64, [0, 13, 31]
    batch = Batch(gpu_ctx, [length], [n], 64, rng)
    kv = gpu_ctx.kv_cache(heads, dim, 64, batch.n_pages)
    hk, hv = _filled(gpu_ctx, kv, batch, rng)
    q = _rows(rng, n, heads, dim, dtype)
    got = _attend(gpu_ctx, kv, batch, q, dtype, 0.125, **kw)
    assert np.isfinite(got).all() and (got != 7).any(-1).all()
    _check(batch, np.ascontiguousarray(got[:, some]), np.ascontiguousarray(q[:, some]), hk[:, some], hv[:, some], 0.125, **kw)
    kv.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("page", [80, 112, 128, 240, 256])
def test_attention_over_larger_pages(gpu_ctx, dtype, dim, page):
    _say("pages", np.dtype(dtype).name, dim, page)
    rng = np.random.default_rng(page + dim)
    batch = Batch(gpu_ctx, [1, 700, 257, 0, 3000, page, page + 1], [1, 1, 2, 1, 1, 1, 90], page, rng, spare=3)
    kv = gpu_ctx.kv_cache(2, dim, page, batch.n_pages)
    hk, hv = _filled(gpu_ctx, kv, batch, rng)
    q = _rows(rng, batch.tokens, 4, dim, dtype)
    scale = dim ** -0.5
    for kw in ({}, dict(window=130)):
        _check(batch, _attend(gpu_ctx, kv, batch, q, dtype, scale, **kw), q, hk, hv, scale, **kw)
    kv.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_cache_beyond_32_bits_of_bytes(gpu_ctx, dtype, dim):
    # pages on both sides of 2^32 bytes, decode and a prompt
    _say("large cache", np.dtype(dtype).name, dim)
    rng = np.random.default_rng(48)
    heads, page = 32, 256
    bytes_of_page = heads * page * dim * 9 // 8
    n_pages = 2 ** 32 // bytes_of_page + 9
    kv = gpu_ctx.kv_cache(heads, dim, page, n_pages)
    assert kv.bytes_num > 2 ** 32
    batch = Batch(gpu_ctx, [700, 513, 300], [1, 1, 70], page, rng)
    ids = np.concatenate([np.arange(4), n_pages - 1 - np.arange(4)])
    ids = rng.permutation(ids)
    batch.table = np.where(batch.table >= 0, ids[batch.table % 8], -1).astype(np.int32)
    batch.d_table.upload(batch.table)
    hk, hv = _filled(gpu_ctx, kv, batch, rng)
    dk, dv = (gpu_ctx.empty(hk.shape, np.float16) for _ in "kv")
    gpu_ctx.kv_read(kv, batch.whole, dk, dv)
    assert np.array_equal(dk.numpy().astype(np.float64), hk) and np.array_equal(dv.numpy().astype(np.float64), hv)
    q, some = _rows(rng, batch.tokens, heads, dim, dtype), [0, 17, 31]
    got = _attend(gpu_ctx, kv, batch, q, dtype, 0.09)
    _check(batch, np.ascontiguousarray(got[:, some]), np.ascontiguousarray(q[:, some]), hk[:, some], hv[:, some], 0.09)
    kv.free()


# ---- lengths beyond the table ----

@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("causal", [True, False])
def test_tokens_past_the_tables_end(gpu_ctx, dtype, causal):
    # a length of more tokens than max_pages * page_size: those are not written, read or attended to
    _say("past the table", np.dtype(dtype).name, causal)
    rng = np.random.default_rng(49)
    heads, dim, page, most = 2, 128, 16, 3
    kv = gpu_ctx.kv_cache(heads, dim, page, 8)
    table = [[5, 2, 7], [0, 4, 1]]
    k, v = (_rows(rng, 96, heads, dim, np.float16) for _ in "kv")
    gpu_ctx.kv_write(kv, _seqs(gpu_ctx, table, [48, 48], [0, 48, 96], 96), gpu_ctx.to_device(k), gpu_ctx.to_device(v))
    hk, hv = kvref.held_pair(k, v)
    # rows 0..59: of a sequence of 100 (its tokens 40 .. 99), rows 60..61 of one of 2^31 - 1
    seqs = _seqs(gpu_ctx, table, [100, 2 ** 31 - 1], [0, 60, 62], 62)
    nk, nv = (_rows(rng, 62, heads, dim, np.float16) for _ in "kv")
    gpu_ctx.kv_write(kv, seqs, gpu_ctx.to_device(nk), gpu_ctx.to_device(nv))
    new = kvref.held_pair(nk, nv)
    for old, n in ((hk, new[0]), (hv, new[1])):
        old[40:48] = n[:8]
    dk, dv = (gpu_ctx.to_device(np.full((62, heads, dim), 5, np.float32)) for _ in "kv")
    gpu_ctx.kv_read(kv, seqs, dk, dv)
    assert np.array_equal(dk.numpy()[:8].astype(np.float64), new[0][:8]) and (dk.numpy()[8:] == 5).all()
    assert np.array_equal(dv.numpy()[:8].astype(np.float64), new[1][:8]) and (dv.numpy()[8:] == 5).all()
    q, out = _rows(rng, 62, 6, dim, dtype), gpu_ctx.empty((62, 6, dim), dtype)
    gpu_ctx.kv_attention(kv, seqs, gpu_ctx.to_device(q), out, 6, 0.09, causal=causal)
    got = out.numpy()
    f16 = dtype == np.float16
    for t in range(62):
        # as the last token of what the table holds of it
        n, at = (min(41 + t, 48) if causal else 48, 0) if t < 60 else (48, 48)
        want, mag, eps, floor = kvref.attention(q[t:t + 1], hk[at:at + n], hv[at:at + n], 0.09)
        assert (np.abs(got[t] - want[0]) <= kvref.tolerance(want, mag, eps, floor, n, f16)[0]).all(), t
    kv.free()
