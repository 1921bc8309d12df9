"""The 4-bit K/V cache and its attention as a program uses them: behind and before quantised products,
token by token, on a stream of the caller's, captured into graphs, with exact workspaces."""
import contextlib
import ctypes

import numpy as np
import pytest

import arf_amd
import kvref
from arf_amd import QType, arfq, synth
from conftest import rel_err
from test_gpu_kv import Batch, _attend, _check, _filled, _rows, _say

pytestmark = pytest.mark.gpu


# ---- HIP's own calls, from the runtime that the library is linked with ----

def _hip(name, *args):
    st = getattr(arf_amd.load_library(), name)(*args)
    assert st == 0, (name, st)


@contextlib.contextmanager
def _stream_ctx():
    """A context on a stream of the caller's."""
    s = ctypes.c_void_p()
    with arf_amd.Context(0):  # (the device is set up)
        _hip("hipStreamCreate", ctypes.byref(s))
    with arf_amd.Context(0, s.value) as ctx:
        assert arf_amd.load_library().arfq_ctx_stream(ctx.handle) == s.value
        yield ctx, s
        ctx.sync()
    _hip("hipStreamDestroy", s)


class Graph:
    """What `calls` enqueues on the stream, captured."""

    def __init__(self, stream, calls):
        self.stream, graph, self.run = stream, ctypes.c_void_p(), ctypes.c_void_p()
        _hip("hipStreamBeginCapture", stream, 2)  # (relaxed: a temporary array may be freed meanwhile)
        try:
            calls()
        finally:
            _hip("hipStreamEndCapture", stream, ctypes.byref(graph))
        _hip("hipGraphInstantiate", ctypes.byref(self.run), graph, None, None, ctypes.c_size_t(0))
        _hip("hipGraphDestroy", graph)

    def launch(self):
        _hip("hipGraphLaunch", self.run, self.stream)

    def free(self):
        _hip("hipGraphExecDestroy", self.run)


# ---- a layer's attention block ----

@pytest.mark.parametrize("qtype,heads,group,dim", [("q8_0", 2, 4, 64), ("q4_k", 1, 2, 128), ("q6_k", 2, 1, 128)])
def test_attention_block_prompt_then_tokens(gpu_ctx, qtype, heads, group, dim):
    # qkv product -> cache -> attention -> output product: two prompts, then tokens one at a time (one
    # sequence idles a step, and a third joins late), every stage against 64 bits of the stage before
    _say("block", qtype, heads, group, dim)
    rng = np.random.default_rng(heads + dim)
    hq, hidden, page, slots = heads * group, 512, 16, 3
    width, wq = (hq + 2 * heads) * dim, hq * dim
    qt = QType[qtype.upper()]
    raw = [gpu_ctx.upload(qt, synth.weight(qtype, n, k, seed=s), n, k) for n, k, s in ((width, hidden, 5), (hidden, wq, 6))]
    dense = [gpu_ctx.dequant(w).numpy().reshape(w.n, w.k).astype(np.float64) for w in raw]
    kv = gpu_ctx.kv_cache(heads, dim, page, 16)
    table = rng.permutation(15).astype(np.int32).reshape(slots, 5)
    d_table = gpu_ctx.to_device(table)
    d_len, d_start = gpu_ctx.empty((slots,), np.int32), gpu_ctx.empty((slots + 1,), np.int32)
    lens = np.zeros(slots, np.int32)
    keys = [(np.zeros((0, heads, dim)),) * 2 for _ in range(slots)]
    for news in ([37, 5, 0], [1, 1, 0], [1, 0, 20], [1, 1, 1], [1, 3, 1]):
        news = np.array(news, np.int32)
        lens += news
        start = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        m = int(start[-1])
        d_len.upload(lens)
        d_start.upload(start)
        seqs = arf_amd.KVSeqs(d_table, d_len, d_start, m)
        x = synth.activations(m, hidden, seed=int(lens.sum()))
        dx, qkv = gpu_ctx.to_device(x), gpu_ctx.empty((m, width), np.float32)
        att, y = gpu_ctx.empty((m, wq), np.float32), gpu_ctx.empty((m, hidden), np.float32)
        gpu_ctx.matmul(raw[0], dx, m, qkv)
        gpu_ctx.kv_write(kv, seqs, qkv.columns(wq), qkv.columns(wq + heads * dim), width, width)
        gpu_ctx.kv_attention(kv, seqs, qkv, att, hq, dim ** -0.5, q_stride=width)
        gpu_ctx.matmul(raw[1], att, m, y)
        qkv_h, att_h = qkv.numpy(), att.numpy()
        assert rel_err(qkv_h, x.astype(np.float64) @ dense[0].T) < 2e-3
        assert rel_err(y.numpy(), att_h.astype(np.float64) @ dense[1].T) < 2e-3
        q, k, v = (np.ascontiguousarray(a).reshape(m, -1, dim) for a in np.split(qkv_h, [wq, wq + heads * dim], 1))
        hk, hv = kvref.held_pair(k, v)
        for b in range(slots):
            r = slice(start[b], start[b + 1])
            keys[b] = tuple(np.concatenate([old, new[r]]) for old, new in zip(keys[b], (hk, hv)))
            want, mag, eps, floor = kvref.attention(q[r], *keys[b], dim ** -0.5)
            off = np.abs(att_h[r].reshape(want.shape) - want)
            assert (off <= kvref.tolerance(want, mag, eps, floor, int(lens[b]), False)).all(), (b, lens)
    kv.free()


# ---- streams and graphs ----

@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_captured_and_replayed(dtype):
    # a decode step (write, attention) in one graph and a step of drafts in another, which share a
    # workspace: lengths, pages and rows change between the replays, eager work runs in between
    _say("graph", np.dtype(dtype).name)
    rng = np.random.default_rng(31)
    heads, group, dim, page, slots, most = 2, 4, 128, 16, 5, 200
    with _stream_ctx() as (ctx, stream):
        d_table, d_len = ctx.empty((slots, most), np.int32), ctx.empty((slots,), np.int32)
        steps = []
        for tokens in (slots, 23):
            arrays = [ctx.to_device(np.zeros((tokens, h, dim), dtype)) for h in (heads, heads, heads * group, heads * group)]
            start = ctx.to_device(np.zeros(slots + 1, np.int32))
            steps.append((arf_amd.KVSeqs(d_table, d_len, start, tokens), start, arrays, ctx.kv_cache(heads, dim, page, slots * most)))
        need = max(ctx.kv_attention_workspace(kv, s, heads * group) for s, _, _, kv in steps)
        ws = ctx.empty((need // 4,), np.float32)

        def calls(seqs, arrays, kv, ws):
            k, v, q, out = arrays
            ctx.kv_write(kv, seqs, k, v)
            ctx.kv_attention(kv, seqs, q, out, heads * group, 0.09, workspace=ws)

        graphs = [Graph(stream, lambda: calls(seqs, arrays, kv, ws)) for seqs, _, arrays, kv in steps]
        lens = np.array([3000, 0, 17, 900, 1], np.int32)
        history = ctx.empty((slots * 3000, heads, dim), np.float16)
        history.upload(_rows(rng, slots * 3000, heads, dim, np.float16))
        for turn in range(4):
            d_table.upload(rng.permutation(slots * most).astype(np.int32).reshape(slots, most))
            whole = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
            d_whole = ctx.to_device(whole)
            for i, (seqs, start, arrays, kv) in enumerate(steps):
                d_len.upload(np.diff(whole).astype(np.int32))
                ctx.kv_write(kv, arf_amd.KVSeqs(d_table, d_len, d_whole, int(whole[-1])), history, history)
                tokens = seqs.tokens
                news = np.ones(slots, np.int32) if i == 0 else np.array([9, 0, 4, 8, 2], np.int32)
                lens = np.minimum(lens + news * (lens > 0), most * page)
                d_len.upload(lens)
                start.upload(np.concatenate([[0], np.cumsum(news)]).astype(np.int32))
                for a in arrays[:3]:
                    a.upload(_rows(rng, tokens, a.shape[1], dim, dtype))
                arrays[3].upload(np.full(arrays[3].shape, 7, dtype))
                ctx.sync()
                graphs[i].launch()
                got = arrays[3].numpy()
                calls(seqs, arrays, kv, None)  # (writes the same rows again)
                assert np.array_equal(got.view(np.uint8), arrays[3].numpy().view(np.uint8)), (turn, i)
                graphs[i].launch()
                graphs[1 - i].launch()
                graphs[i].launch()
                assert np.array_equal(got.view(np.uint8), arrays[3].numpy().view(np.uint8)), (turn, i)
        for g in graphs:
            g.free()
        # under capture a workspace is the caller's; a call that wants none runs without
        short = arf_amd.KVSeqs(ctx.to_device(np.zeros((2, 4), np.int32)), ctx.to_device(np.array([40, 9], np.int32)))
        assert ctx.kv_attention_workspace(steps[0][3], short, heads * group) == 0
        q, out = steps[0][2][2:]
        refused = []

        def refused_and_not():
            ctx.kv_attention(steps[0][3], short, q, out, heads * group, 0.09)
            for call in (lambda: ctx.kv_attention(steps[0][3], steps[0][0], q, out, heads * group, 0.09),
                         lambda: ctx.kv_cache(1, 64, 16, 1)):
                with pytest.raises(arf_amd.ArfqError) as e:
                    call()
                refused.append((e.value.status, str(e.value)))

        g = Graph(stream, refused_and_not)
        assert [s for s, _ in refused] == [arfq.ARFQ_E_INVALID] * 2 and "capture" in refused[0][1]
        ctx.kv_attention(steps[0][3], short, q, out, heads * group, 0.09)
        want = out.numpy()[:2]
        for _ in range(3):
            out.upload(np.full(out.shape, 7, dtype))
            ctx.sync()
            g.launch()
            got = out.numpy()
            assert np.array_equal(got[:2].view(np.uint8), want.view(np.uint8)) and (got[2:] == 7).all()
        g.free()
        for *_, kv in steps:
            kv.free()


def test_callers_stream(gpu_ctx):
    # the same work on a stream of the caller's gives the same bits
    _say("stream")
    got = []
    with _stream_ctx() as (other, _):
        for ctx in (gpu_ctx, other):
            rng = np.random.default_rng(33)
            batch = Batch(ctx, [700, 64, 130], [80, 1, 130], 32, rng)
            kv = ctx.kv_cache(2, 96, 32, batch.n_pages)
            _filled(ctx, kv, batch, rng)
            q = _rows(rng, batch.tokens, 6, 96, np.float32)
            got.append(_attend(ctx, kv, batch, q, np.float32, 0.1))
            kv.free()
    assert np.array_equal(got[0].view(np.uint32), got[1].view(np.uint32))


# ---- batches ----

def test_more_than_a_wave_of_prompts_and_tokens(gpu_ctx):
    # 130 sequences, prompts of more rows than the short tiles take among single tokens and idle slots
    _say("mixed")
    rng = np.random.default_rng(34)
    lens = [int(x) for x in rng.integers(1, 60, 130)]
    news = [1] * 130
    for b, (ln, n) in {3: (90, 90), 63: (200, 33), 64: (1500, 40), 65: (0, 0), 100: (77, 77), 129: (700, 35)}.items():
        lens[b], news[b] = ln, n
    batch = Batch(gpu_ctx, lens, news, 16, rng)
    kv = gpu_ctx.kv_cache(2, 64, 16, batch.n_pages)
    hk, hv = _filled(gpu_ctx, kv, batch, rng)
    for dtype in (np.float16, np.float32):
        q = _rows(rng, batch.tokens, 4, 64, dtype)
        for kw in ({}, dict(window=50)):
            _check(batch, _attend(gpu_ctx, kv, batch, q, dtype, 0.125, **kw), q, hk, hv, 0.125, **kw)


@pytest.mark.parametrize("batch,max_pages,heads,group,dim", [(1000, 32, 1, 1, 64), (1, 2000, 8, 8, 128), (300, 40, 2, 65, 64),
                                                             (64, 33, 1, 17, 256), (1, 1, 1, 1, 64), (500, 17, 1, 64, 96)])
def test_workspaces_of_the_size_that_is_asked_for(gpu_ctx, batch, max_pages, heads, group, dim):
    # with and without a start, the caller's workspace gives the bits of the context's scratch
    _say("workspace", batch, max_pages, heads, group, dim)
    rng = np.random.default_rng(batch + max_pages)
    kv = gpu_ctx.kv_cache(heads, dim, 16, 64)
    x = gpu_ctx.to_device(_rows(rng, 1024, heads, dim, np.float16))
    every = arf_amd.KVSeqs(gpu_ctx.to_device(np.arange(64, dtype=np.int32)[None]), gpu_ctx.to_device(np.array([1024], np.int32)),
                           gpu_ctx.to_device(np.array([0, 1024], np.int32)), 1024)
    gpu_ctx.kv_write(kv, every, x, x)
    table = gpu_ctx.to_device(rng.integers(0, 64, (batch, max_pages)).astype(np.int32))
    lens = gpu_ctx.to_device(rng.integers(0, 16 * max_pages + 1, batch).astype(np.int32))
    one = gpu_ctx.to_device(np.arange(batch + 1, dtype=np.int32))
    q = _rows(rng, batch, heads * group, dim, np.float16)
    dq, out = gpu_ctx.to_device(q), gpu_ctx.empty(q.shape, np.float16)
    for start in (None, one):
        seqs = arf_amd.KVSeqs(table, lens, start, None if start is None else batch)
        need = gpu_ctx.kv_attention_workspace(kv, seqs, heads * group)
        ws = gpu_ctx.empty((max(16, need),), np.uint8)
        got = []
        for w in (None, ws):
            out.upload(np.full(q.shape, 7, np.float16))
            gpu_ctx.kv_attention(kv, seqs, dq, out, heads * group, 0.1, workspace=w)
            got.append(out.numpy())
        assert np.array_equal(got[0].view(np.uint16), got[1].view(np.uint16)) and np.isfinite(got[0]).all()
    kv.free()


def test_sequences_that_share_pages(gpu_ctx):
    # a page of two tables is read by both; a sequence of the batch may be named twice
    _say("shared pages")
    rng = np.random.default_rng(35)
    batch = Batch(gpu_ctx, [100, 100], [1, 2], 32, rng)
    batch.table[1] = batch.table[0]
    batch.d_table.upload(batch.table)
    kv = gpu_ctx.kv_cache(1, 128, 32, batch.n_pages)
    k, v = (_rows(rng, 100, 1, 128, np.float32) for _ in "kv")
    gpu_ctx.kv_write(kv, batch.whole, *(gpu_ctx.to_device(np.concatenate([a, a])) for a in (k, v)))
    hk, hv = (np.concatenate([a, a]) for a in kvref.held_pair(k, v))
    q = _rows(rng, 3, 4, 128, np.float32)
    got = _attend(gpu_ctx, kv, batch, q, np.float32, 0.09)
    _check(batch, got, q, hk, hv, 0.09)


def test_workspace_does_not_grow_with_a_prompt(gpu_ctx):
    # parts are kept only of rows whose keys are cut, and a step with many tiles cuts none
    kv = gpu_ctx.kv_cache(8, 128, 64, 4)
    table, lens, start = (gpu_ctx.to_device(np.zeros(n, np.int32)) for n in ((1, 1000), 1, 2))
    sizes = [gpu_ctx.kv_attention_workspace(kv, arf_amd.KVSeqs(table, lens, start, t), 32) for t in (1, 8192, 32768, 2 ** 20)]
    assert 0 < sizes[0] < sizes[1] == sizes[2] == sizes[3] < 2 ** 27
    kv.free()
