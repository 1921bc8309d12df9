"""The operators of a serving step as a program uses them: one behind another between quantised products, token by
token with drafts taken back, captured into graphs that share a workspace, on a stream of the caller's."""
import numpy as np
import pytest

import arf_amd
import kvref
import stepref
from arf_amd import QType, synth
from conftest import rel_err
from test_gpu_kv import _say
from test_gpu_kv_use import Graph, _stream_ctx

pytestmark = pytest.mark.gpu


class State:
    """What a program keeps of its requests: two steps that take each other's lengths, and the cache behind them."""

    def __init__(self, ctx, batch, most, page, n_pages, tokens, heads, dim):
        i32 = lambda *s: ctx.to_device(np.zeros(s, np.int32))
        self.ctx, self.add, self.tokens = ctx, i32(batch), tokens
        pages, free = ctx.to_device(np.full((batch, most), -1, np.int32)), ctx.to_device(np.arange(n_pages, dtype=np.int32)[::-1].copy())
        held, n_free = (i32(batch), i32(batch)), (ctx.to_device(np.array([n_pages], np.int32)), i32(1))
        self.steps = [arf_amd.KVStep(page, self.add, held[i], held[1 - i], pages, free, n_free[i], n_free[1 - i], i32(batch + 1), i32(batch),
                                     i32(batch + 1), i32(batch + 1), i32(tokens), ctx.to_device(np.zeros(tokens, np.int64))) for i in (0, 1)]
        self.kv = ctx.kv_cache(heads, dim, page, n_pages)
        self.bounds = ctx.to_device(np.zeros((n_pages, heads, 2, dim), np.float16))


@pytest.mark.parametrize("qtype,heads,group,dim", [("q8_0", 2, 4, 64), ("q4_k", 1, 2, 128)])
def test_attention_block_of_many_requests(gpu_ctx, qtype, heads, group, dim):
    # page tables -> qkv product -> adapters -> rotary positions -> cache and bounds -> chosen blocks -> output product:
    # prompts, tokens, drafts taken back, a request that ends and another in its slot; each stage against 64
    # bits of the stage before
    _say("block", qtype, heads, group, dim)
    ctx, rng = gpu_ctx, np.random.default_rng(heads + dim)
    hq, hidden, page, slots, tokens = heads * group, 512, 16, 3, 150
    width, wq, rank = (hq + 2 * heads) * dim, hq * dim, 16
    qt = QType[qtype.upper()]
    w = [ctx.upload(qt, synth.weight(qtype, n, k, seed=s), n, k) for n, k, s in ((width, hidden, 5), (hidden, wq, 6))]
    dense = [ctx.dequant(x).numpy().reshape(x.n, x.k).astype(np.float64) for x in w]
    la, lb = (rng.standard_normal((2, rank, hidden)) / 23).astype(np.float16), rng.standard_normal((2, width, rank)).astype(np.float16)
    lora = arf_amd.Lora(ctx.to_device(la), ctx.to_device(lb))
    rope = arf_amd.Rope.sections([dim // 4, dim // 8, dim // 8], 1000.0, "cycle")
    state = State(ctx, slots, 16, page, 24, tokens, heads, dim)
    kv, count = state.kv, 4
    keys = [(np.zeros((0, heads, dim)),) * 2 for _ in range(slots)]
    held = np.zeros(slots, np.int32)
    x, ids = ctx.empty((tokens, hidden), np.float32), ctx.empty((tokens,), np.int32)
    pos3 = ctx.empty((3, tokens), np.int32)
    qkv, both = ctx.empty((tokens, width), np.float32), ctx.empty((tokens, width), np.float32)
    att, y = ctx.empty((tokens, wq), np.float32), ctx.empty((tokens, hidden), np.float32)
    chosen = ctx.empty((tokens, heads, count), np.int32)
    for i, add in enumerate(([100, 45, 0], [1, 1, 0], [5, 0, 30], [-3, 1, 1], [1, -46, 1], [1, 17, 1], [200, 1, 1], [1, 1, 1])):
        add = np.array(add, np.int32)
        step = state.steps[i % 2]
        state.add.upload(add)
        ctx.kv_plan(step)
        grown = step.held_next.numpy()
        fits = (add <= 0) | (held + add <= 16 * page) & (np.cumsum(np.maximum(add, 0)) <= tokens)
        assert np.array_equal(grown, np.where(fits, held + add, held))
        start, pos, lens = step.start.numpy(), step.positions.numpy(), step.lens.numpy()
        assert np.array_equal(lens, np.where(fits, grown, 0))
        m = int(start[-1])
        hx = synth.activations(tokens, hidden, seed=100 + i)
        which = rng.integers(-1, 2, slots)[np.searchsorted(start[1:], np.arange(tokens), side="right").clip(max=slots - 1)].astype(np.int32)
        p3 = np.stack([pos, pos // 4, pos % 4]).astype(np.int32)
        x.upload(hx)
        ids.upload(which)
        pos3.upload(p3)
        if m:
            ctx.matmul(w[0], x, m, qkv)
        ctx.lora_add(lora, ids, x, m, both, base=qkv)
        hb = both.numpy()[:m]
        ctx.rope(rope, pos3, both, both, m, hq + heads, dim, x_stride=width, out_stride=width)
        ctx.kv_write(kv, step.seqs, both.columns(wq), both.columns(wq + heads * dim), width, width)
        ctx.kv_bounds(kv, step.seqs, state.bounds)
        ctx.kv_attention_blocks(kv, step.seqs, state.bounds, both, att, hq, dim ** -0.5, count, first=1, last=2, chosen=chosen, q_stride=width)
        if m:
            ctx.matmul(w[1], att, m, y)
        h0, h1, ha, hc, hy = qkv.numpy()[:m], both.numpy()[:m], att.numpy()[:m], chosen.numpy()[:m], y.numpy()[:m]
        if m:
            assert rel_err(h0, hx[:m].astype(np.float64) @ dense[0].T) < 2e-3
            assert rel_err(hy, ha.astype(np.float64) @ dense[1].T) < 2e-3
            want, mags = stepref.lora(hx[:m], which[:m], la, lb, None, h0)
            assert (np.abs(hb - want) <= stepref.lora_tolerance(want, mags, h0, hidden, rank)).all()
            turned = hb[:, :wq + heads * dim].reshape(m, -1, dim)
            want, mag = stepref.rope(turned, p3, rope._freqs, rope._axes, False)
            assert (np.abs(h1[:, :wq + heads * dim].reshape(want.shape) - want) <= stepref.rope_tolerance(want, mag, p3 * 1.0, False)).all()
            assert np.array_equal(h1[:, wq + heads * dim:], hb[:, wq + heads * dim:])
        q, k, v = (np.ascontiguousarray(a).reshape(m, -1, dim) for a in np.split(h1, [wq, wq + heads * dim], 1))
        hk, hv = kvref.held_pair(k, v)
        for b in range(slots):
            r = slice(start[b], start[b + 1])
            if add[b] < 0:
                keys[b] = tuple(old[:grown[b]] for old in keys[b])
            elif not fits[b]:
                assert (ha[r] == 0).all() and (hc[r] == -1).all()
            elif add[b] > 0:
                keys[b] = tuple(np.concatenate([old, new[r]]) for old, new in zip(keys[b], (hk, hv)))
                # (the bounds of a page that tokens were taken back from are formed anew with its next row)
                want, mag, eps, floor, most, blocks = stepref.attend_blocks(q[r], *keys[b], page, dim ** -0.5, count, 1, 2)
                assert np.array_equal(hc[r], blocks)
                off = np.abs(ha[r].reshape(want.shape) - want)
                assert (off <= kvref.tolerance(want, mag, eps, floor, most, False)).all(), (i, b)
        held = grown
    kv.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_captured_and_replayed(dtype):
    # two steps in a graph (the second takes the first's lengths), the operators sharing one workspace: what the step
    # asks for, rows, adapters and pages change between the replays, eager work of another state runs in between and says
    # what is right, to the bit
    _say("graph", np.dtype(dtype).name)
    rng = np.random.default_rng(12)
    heads, group, dim, page, batch, tokens, k, rank, count = 2, 4, 64, 16, 5, 40, 96, 8, 3
    hq = heads * group
    width = (hq + 2 * heads) * dim
    la, lb = rng.standard_normal((3, rank, k)).astype(np.float16), rng.standard_normal((3, width, rank)).astype(np.float16)
    with _stream_ctx() as (ctx, stream), arf_amd.Context(0) as other:
        def program(c, with_workspace):
            s = State(c, batch, 30, page, 80, tokens, heads, dim)
            s.lora, s.rope = arf_amd.Lora(c.to_device(la), c.to_device(lb)), arf_amd.Rope.sections([dim // 2])
            s.x, s.ids = (c.to_device(np.zeros((tokens, k), np.float32)), c.to_device(np.zeros(tokens, np.int32)))
            s.base, s.qkv = (c.to_device(np.zeros((tokens, width), np.float32)) for _ in "bq")
            s.rows = c.to_device(np.zeros((tokens, hq + heads, dim), dtype))
            s.v = c.to_device(np.zeros((tokens, heads, dim), dtype))
            s.out = [c.to_device(np.zeros((tokens, hq, dim), dtype)) for _ in (0, 1)]
            s.chosen = [c.to_device(np.zeros((tokens, heads, count), np.int32)) for _ in (0, 1)]
            s.ws = None
            if with_workspace:
                size = max(c.lora_workspace(s.lora, tokens), c.kv_attention_blocks_workspace(s.kv, s.steps[0].seqs, hq, count))
                s.ws = c.empty((size,), np.uint8)

            def run():
                row = (hq + heads) * dim
                for i, step in enumerate(s.steps):
                    c.kv_plan(step)
                    c.lora_add(s.lora, s.ids, s.x, tokens, s.qkv, base=s.base, workspace=s.ws)
                    c.rope(s.rope, step.positions, s.qkv, s.rows, tokens, hq + heads, dim, x_stride=width)
                    c.kv_write(s.kv, step.seqs, s.rows.columns(hq * dim), s.v, row, heads * dim)
                    c.kv_bounds(s.kv, step.seqs, s.bounds)
                    c.kv_attention_blocks(s.kv, step.seqs, s.bounds, s.rows, s.out[i], hq, 0.125, count, first=1, chosen=s.chosen[i],
                                          q_stride=row, workspace=s.ws)
            s.run = run
            return s
        s, t = program(ctx, True), program(other, False)
        with pytest.raises(arf_amd.ArfqError, match="needs a workspace"):
            big = arf_amd.Lora(ctx.to_device(np.zeros((1, 8, 16392), np.float16)), ctx.to_device(np.zeros((1, 8, 8), np.float16)))
            wide = ctx.to_device(np.zeros((1, 16392), np.float32))
            assert ctx.lora_workspace(big, 1) > 0
            Graph(stream, lambda: ctx.lora_add(big, s.ids, wide, 1, s.qkv))
        with pytest.raises(arf_amd.ArfqError, match="needs a workspace"):
            Graph(stream, lambda: ctx.kv_attention_blocks(s.kv, s.steps[0].seqs, s.bounds, s.rows, s.out[0], hq, 0.125, count))
        graph = Graph(stream, s.run)
        for i, add in enumerate(([9, 4, 0, 8, 1], [1, 1, 1, 1, 1], [3, -5, 20, 1, 0], [-100, 1, 1, 1, 1], [8, 8, 8, 8, 8], [1, 1, 1, 1, 30])):
            inputs = (rng.standard_normal((tokens, k)).astype(np.float32), rng.integers(-1, 3, tokens).astype(np.int32),
                      rng.standard_normal((tokens, width)).astype(np.float32), rng.standard_normal((tokens, heads, dim)).astype(dtype))
            for p in (s, t):
                for d, h in zip((p.x, p.ids, p.base, p.v), inputs):
                    d.upload(h)
                p.add.upload(np.array(add, np.int32))
            graph.launch()
            t.run()
            other.sync()
            ctx.sync()
            for a, b in zip((s.bounds, *s.out, *s.chosen), (t.bounds, *t.out, *t.chosen)):
                assert np.array_equal(a.numpy(), b.numpy()), i
            for p, q in zip(s.steps, t.steps):
                for name in ("held_next", "n_free_next", "lens", "positions", "slots", "pages"):
                    assert np.array_equal(getattr(p, name).numpy(), getattr(q, name).numpy()), (i, name)
        graph.free()


def test_calls_without_work(gpu_ctx):
    # no rows, no sequences: nothing is written
    _say("no work")
    up = gpu_ctx.to_device
    none, x = up(np.zeros(0, np.int32)), up(np.full((4, 64), 3, np.float32))
    gpu_ctx.rope(arf_amd.Rope.sections([32]), none, x, x, 0, 1, 64)
    lora = arf_amd.Lora(up(np.zeros((1, 8, 64), np.float16)), up(np.zeros((1, 64, 8), np.float16)))
    gpu_ctx.lora_add(lora, none, x, 0, x)
    assert gpu_ctx.lora_workspace(lora, 0) == 0
    kv = gpu_ctx.kv_cache(1, 64, 16, 4)
    bounds = up(np.full((4, 1, 2, 64), 9, np.float16))
    for seqs in (arf_amd.KVSeqs(up(np.zeros((0, 4), np.int32)), none), arf_amd.KVSeqs(up(np.zeros((2, 4), np.int32)), up(np.zeros(2, np.int32)), None, 0)):
        gpu_ctx.kv_bounds(kv, seqs, bounds)
        gpu_ctx.kv_attention_blocks(kv, seqs, bounds, x, x, 1, 1.0, 2)
    empty = arf_amd.KVSeqs(up(np.zeros((2, 0), np.int32)), up(np.array([5, 0], np.int32)))  # tables without a page
    out, chosen = up(np.full((2, 64), 3, np.float32)), up(np.full((2, 1, 2), 5, np.int32))
    gpu_ctx.kv_bounds(kv, empty, bounds)
    gpu_ctx.kv_attention_blocks(kv, empty, bounds, x, out, 1, 1.0, 2, chosen=chosen)
    assert (x.numpy() == 3).all() and (bounds.numpy() == 9).all() and (out.numpy() == 0).all() and (chosen.numpy() == -1).all()
    kv.free()
