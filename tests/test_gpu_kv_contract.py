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
