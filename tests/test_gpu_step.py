"""A step's bookkeeping, adapters, rotary positions and attention over chosen blocks on the GPU, against numpy in 64
bits (stepref): whole numbers equal, others within what the roundings of their definitions allow."""
import ctypes

import numpy as np
import pytest

import arf_amd
import kvref
import stepref
from arf_amd import arfq
from test_gpu_kv import Batch, _filled, _rows, _say

pytestmark = pytest.mark.gpu


# ---- a step's bookkeeping ----

NAMES = ("pages", "free", "held_next", "lens", "start", "taken", "freed", "n_free_next", "positions", "slots")


def _plan(ctx, page, add, held, pages, free, n_free, tokens):
    """The call's arrays; what it may leave as it was starts from 77 (what a step before left there)."""
    n = len(add)
    up = lambda a: ctx.to_device(np.asarray(a, np.int32))
    new = lambda *shape: up(np.full(shape, 77))
    step = arf_amd.KVStep(page, up(add), up(held), new(n), up(pages), up(free), up([n_free]), new(1), new(n + 1),
                          new(n), new(n + 1), new(n + 1), new(tokens), ctx.to_device(np.full(tokens, 77, np.int64)))
    ctx.kv_plan(step)
    got = {name: getattr(step, name).numpy() for name in NAMES}
    assert np.array_equal(step.add.numpy(), add) and np.array_equal(step.held.numpy(), held) and step.n_free.numpy()[0] == n_free
    return got


def _check_plan(ctx, page, add, held, pages, free, n_free, tokens):
    got = _plan(ctx, page, add, held, pages, free, n_free, tokens)
    want = stepref.plan(page, add, held, pages, free, n_free, tokens)
    for name in NAMES:
        assert np.array_equal(got[name], want[name]), name
    return got


def _random_plan(rng, batch, page, longest, most_new, short):
    held = rng.integers(0, longest + 1, batch)
    add = rng.integers(1, most_new + 1, batch)
    kind = rng.integers(0, 6, batch)
    add = np.where(kind == 0, -held, np.where(kind == 1, -np.minimum(held, rng.integers(0, 40, batch)), np.where(kind == 2, 0, add)))
    held = np.where(kind == 3, 0, held)
    add = np.where(kind == 3, np.abs(add), add)
    ceil = lambda n: -(-n // page)
    have, need = ceil(held), ceil(np.maximum(held + add, 0))
    pages = np.full((batch, max(1, int(max(have.max(), need.max())))), -1, np.int32)
    want = int(np.maximum(need - have, 0).sum() - np.maximum(have - need, 0).sum())
    n_free = max(0, want) // 2 if short else max(0, want) + 3
    ids = rng.permutation(int(have.sum()) + n_free + 5).astype(np.int32)
    at = 0
    for b in range(batch):
        pages[b, :have[b]] = ids[at:at + have[b]]
        at += have[b]
    free = np.full(ids.size, -9, np.int32)
    free[:n_free] = ids[at:at + n_free]
    return add.astype(np.int32), held.astype(np.int32), pages, free, n_free, max(1, int(np.maximum(add, 0).sum()))


@pytest.mark.parametrize("short", [False, True])
@pytest.mark.parametrize("batch,page,longest,most_new", [(1, 16, 0, 1), (1, 16, 50, 33), (64, 64, 8192, 1), (63, 1, 40, 5),
                                                         (300, 48, 500, 300), (1024, 16, 64, 3), (1025, 32, 900, 9),
                                                         (5000, 16, 100, 2), (16384, 16, 40, 1), (7, 65536, 200000, 70000)])
def test_plan(gpu_ctx, batch, page, longest, most_new, short):
    _say("plan", batch, page, longest, most_new, short)
    rng = np.random.default_rng(batch + page + longest)
    _check_plan(gpu_ctx, page, *_random_plan(rng, batch, page, longest, most_new, short))


@pytest.mark.parametrize("spare", [0, 5000])  # rows in the sums' workgroup, and in a launch of their own
def test_plan_refuses_what_does_not_fit(gpu_ctx, spare):
    _say("plan refusals", spare)
    pages = np.arange(24, dtype=np.int32).reshape(6, 4)
    free = np.arange(100, 110).astype(np.int32)
    held = np.array([16, 33, 64, 10, 0, 48], np.int32)
    for add, h, n_free, tokens in (
            ([17, 16, 1, 1, 40, 16], held, 4, 91 + spare),     # the fifth does not fit, nor the sixth's page; the third passes the table
            ([17, 16, 0, 1, 40, 16], held, 100, 91 + spare),   # more free pages than places: ten
            ([17, 16, 0, 1, 40, 16], held, -5, 90 + spare),    # fewer than none
            ([1, 1, -64, 1, 1, 1], held, 0, 5 + spare),        # what is given back is taken
            ([1, 50, 1, 1, 1, 1], held, 10, 40),               # rows past the last place, and what follows
            ([2 ** 31 - 1] * 6, held, 10, 64),
            ([-2 ** 31] * 6, held, 3, 1 + spare),              # all end: pages past the stack's places are dropped
            ([1, -1, 2, 0, 1, 1], [-1, 65, 64, 2 ** 31 - 1, -2 ** 31, 5], 10, 6 + spare),  # not lengths
            ([0, 0, 0, 0, 0, 0], held, 5, 1)):
        _check_plan(gpu_ctx, 16, np.array(add, np.int32), np.array(h, np.int32), pages, free, n_free, tokens)


def test_plan_pages_of_one_token(gpu_ctx):
    # more pages wanted than 31 bits count
    _say("plan pages of one")
    pages, free = np.arange(12, dtype=np.int32).reshape(3, 4), np.arange(20, 28).astype(np.int32)
    for add in ([1, 2 ** 31 - 1, 1], [2 ** 31 - 1, 1, 1], [-1, 2, -2 ** 31]):
        _check_plan(gpu_ctx, 1, np.array(add, np.int32), np.array([2, 2, 3], np.int32), pages, free, 5, 1 << 20)


def test_plan_of_nothing(gpu_ctx):
    _say("plan of nothing")
    none = np.zeros(0, np.int32)
    got = _plan(gpu_ctx, 16, none, none, np.zeros((0, 3), np.int32), np.arange(4, dtype=np.int32), 3, 2)
    assert got["n_free_next"][0] == 3 and (got["positions"] == -1).all() and (got["slots"] == -1).all() and got["start"][0] == 0
    pages = np.zeros((2, 0), np.int32)  # tables without a page
    _check_plan(gpu_ctx, 16, np.array([1, 0], np.int32), np.array([0, 0], np.int32), pages, np.arange(4, dtype=np.int32), 3, 2)


def test_plan_step_after_step(gpu_ctx):
    # held and held_next change places; every page has one owner throughout, and rejected rows give the stack back as it was
    _say("plan steps")
    rng = np.random.default_rng(5)
    page, batch, most, total = 16, 20, 9, 60
    held, n_free = np.zeros(batch, np.int32), total
    pages, free = np.full((batch, most), -1, np.int32), rng.permutation(total).astype(np.int32)
    for i in range(60):
        kind = rng.integers(0, 8, batch)
        add = np.where(kind == 0, -held, np.where(kind < 3, -np.minimum(held, rng.integers(0, 20, batch)), rng.integers(0, 30, batch)))
        got = _check_plan(gpu_ctx, page, add.astype(np.int32), held, pages, free, n_free, 400)
        grown, n = got["held_next"], int(got["n_free_next"][0])
        owned = [int(p) for b in range(batch) for p in got["pages"][b, :-(-int(grown[b]) // page)]]
        assert sorted(owned + [int(p) for p in got["free"][:n]]) == list(range(total))
        back = _check_plan(gpu_ctx, page, np.minimum(held - grown, 0).astype(np.int32), grown, got["pages"], got["free"], n, 1)
        if (grown >= held).all():
            assert np.array_equal(back["held_next"], held) and int(back["n_free_next"][0]) == n_free
            assert np.array_equal(back["free"][:n_free], free[:n_free])
        held, pages, free, n_free = grown, got["pages"], got["free"], n


# ---- rotary positions ----

ROPES = [("halves", [16], "chunks"), ("halves", [5, 7, 4], "cycle"), ("neighbours", [16], "chunks"), ("neighbours", [3, 0, 9, 4], "own")]


@pytest.mark.parametrize("pairs,sections,layout", ROPES)
@pytest.mark.parametrize("xt,ot", [(np.float32, np.float32), (np.float16, np.float16), (np.float32, np.float16), (np.float16, np.float32)])
@pytest.mark.parametrize("tokens,heads,dim", [(1, 1, 32), (5, 3, 40), (67, 13, 128), (3, 2, 1024), (300, 5, 80)])
def test_rope(gpu_ctx, pairs, sections, layout, xt, ot, tokens, heads, dim):
    _say("rope", pairs, sections, layout, np.dtype(xt).name, np.dtype(ot).name, tokens, heads, dim)
    rng = np.random.default_rng(tokens + dim)
    rope = arf_amd.Rope.sections(sections, 500.0, layout, pairs, gain=1.25)
    pos = rng.integers(-1000, 100000, (len(sections), tokens + 3)).astype(np.int32)
    xs, os_ = heads * dim + 16, heads * dim + 8
    x = rng.standard_normal((tokens, xs)).astype(xt)
    rows = x[:, :heads * dim].reshape(tokens, heads, dim)
    want, mag = stepref.rope(rows, pos, rope._freqs, rope._axes, pairs == "neighbours", 1.25)
    d_pos, dx = gpu_ctx.to_device(pos), gpu_ctx.to_device(x)
    out = gpu_ctx.to_device(np.full((tokens, os_), 7, ot))
    gpu_ctx.rope(rope, d_pos, dx, out, tokens, heads, dim, x_stride=xs, out_stride=os_)
    got = out.numpy()
    assert (got[:, heads * dim:] == 7).all()
    tol = stepref.rope_tolerance(want, mag, pos[:, :tokens] * 1.0, ot == np.float16)
    assert (np.abs(got[:, :heads * dim].reshape(rows.shape) - want) <= tol).all()
    if xt == ot:
        # in place, to the bit; and back
        gpu_ctx.rope(rope, d_pos, dx, dx, tokens, heads, dim, x_stride=xs, out_stride=xs)
        turned = dx.numpy()
        assert np.array_equal(turned[:, :heads * dim], got[:, :heads * dim]) and np.array_equal(turned[:, heads * dim:], x[:, heads * dim:])
        gpu_ctx.rope(rope, d_pos, dx, out, tokens, heads, dim, x_stride=xs, out_stride=os_, inverse=True)
        t = turned[:, :heads * dim].reshape(rows.shape)
        want, mag = stepref.rope(t, pos, rope._freqs, rope._axes, pairs == "neighbours", 1.25, inverse=True)
        tol = stepref.rope_tolerance(want, mag, pos[:, :tokens] * 1.0, ot == np.float16)
        assert (np.abs(out.numpy()[:, :heads * dim].reshape(rows.shape) - want) <= tol).all()


def test_rope_far_positions_and_every_quarter(gpu_ctx):
    # positions up to the largest, angles at and next to the borders between quarters of a turn, and no angle at all
    _say("rope far")
    pos = np.array([[0, 1, 2, 3, 4, 5, 7, 8, -1, -2, -3, -5, 2 ** 20 + 1, 2 ** 31 - 1, -2 ** 31]], np.int32)
    freqs = np.array([0.0, np.pi / 8, np.pi / 4, np.pi / 2, -np.pi / 2, 1.0, 1e-9, 3.0])
    x = np.random.default_rng(2).standard_normal((pos.size, 1, 16)).astype(np.float32)
    out = gpu_ctx.empty(x.shape, np.float32)
    gpu_ctx.rope(arf_amd.Rope(freqs), gpu_ctx.to_device(pos), gpu_ctx.to_device(x), out, pos.size, 1, 16)
    # (64 bits hold the largest angles to 2^-20; the reference rounds as often)
    want, mag = stepref.rope(x, pos, freqs, np.zeros(8, int), False)
    tol = stepref.rope_tolerance(want, mag, np.zeros(1), False) + mag * np.abs(pos[0].astype(np.float64))[:, None, None] * 3 * 2.0 ** -51
    assert (np.abs(out.numpy() - want) <= tol).all()
    assert np.array_equal(out.numpy()[:, 0, 0], x[:, 0, 0])


def test_rope_keeps_to_its_rows(gpu_ctx):
    # values that are not finite stay in their pair; the gradient is the rotation back, and differences say the same
    _say("rope rows")
    rng = np.random.default_rng(3)
    rope = arf_amd.Rope.sections([8], 100.0)
    pos = gpu_ctx.to_device(np.arange(6, dtype=np.int32))
    x = rng.standard_normal((6, 2, 24)).astype(np.float32)
    x[2, 1, 3], x[4, 0, 12] = np.nan, np.inf
    out = gpu_ctx.empty(x.shape, np.float32)
    gpu_ctx.rope(rope, pos, gpu_ctx.to_device(x), out, 6, 2, 24)
    bad = np.argwhere(~np.isfinite(out.numpy()))
    assert {tuple(i) for i in bad} <= {(2, 1, 3), (2, 1, 11), (4, 0, 4), (4, 0, 12)} and np.isnan(out.numpy()[2, 1, 3])
    x = np.where(np.isfinite(x), x, 0).astype(np.float32)
    w, step = rng.standard_normal(x.shape).astype(np.float32), rng.standard_normal(x.shape).astype(np.float32)
    run = lambda v, inverse=False: (gpu_ctx.rope(rope, pos, gpu_ctx.to_device(v.astype(np.float32)), out, 6, 2, 24, inverse=inverse),
                                    out.numpy().astype(np.float64))[1]
    grad = run(w, inverse=True)
    # (linear: a step of any length; each value is off by 8 * 2^-24 of its pair)
    rise = (w * (run(x + step) - run(x - step))).sum() / 2
    size = (np.abs(w).max() * np.abs(step).max() + np.abs(w).max() * np.abs(x).max()) * x.size
    assert abs(rise - (grad * step).sum()) <= size * 40 * 2.0 ** -24


def test_rope_more_blocks_than_a_row_of_the_grid(gpu_ctx):
    # 2^23 + 5 rows of one head: the grid's second row
    _say("rope long")
    tokens = (1 << 23) + 5
    rope = arf_amd.Rope.sections([4], 10.0)
    x = np.ones((tokens, 8), np.float16)
    d = gpu_ctx.to_device(x)
    gpu_ctx.rope(rope, gpu_ctx.to_device(np.arange(tokens, dtype=np.int32) % 1000), d, d, tokens, 1, 8)
    got = d.numpy()
    want, mag = stepref.rope(np.ones((1000, 1, 8)), np.arange(1000)[None], rope._freqs, rope._axes, False)
    tol = stepref.rope_tolerance(want, mag, np.array([1000.0]), True)
    for at in (0, 1000000, (1 << 23) - 500):
        rows = np.arange(at, min(at + 1000, tokens))
        assert (np.abs(got[rows][:, None] - want[rows % 1000]) <= tol[rows % 1000]).all()


# ---- adapters ----

def _lora_case(ctx, rng, rows, k, n, rank, adapters, ids, xt, scaled=True, based=True, strides=(0, 0)):
    a = (rng.standard_normal((adapters, rank, k)) / np.sqrt(k)).astype(np.float16)
    b = rng.standard_normal((adapters, n, rank)).astype(np.float16)
    x = rng.standard_normal((rows, k)).astype(xt)
    scale = (rng.random(adapters) + 0.5).astype(np.float32) if scaled else None
    base = rng.standard_normal((rows, n + strides[0])).astype(np.float32) if based else None
    lora = arf_amd.Lora(ctx.to_device(a), ctx.to_device(b), None if scale is None else ctx.to_device(scale))
    d_ids, dx = ctx.to_device(np.asarray(ids, np.int32)), ctx.to_device(x)
    out = ctx.to_device(np.full((rows, n + strides[1]), 7, np.float32))
    d_base = None if base is None else ctx.to_device(base)
    ctx.lora_add(lora, d_ids, dx, rows, out, base=d_base, out_stride=n + strides[1], base_stride=n + strides[0])
    got = out.numpy()
    assert (got[:, n:] == 7).all()
    own = None if base is None else base[:, :n]
    want, mags = stepref.lora(x, ids, a, b, scale, own)
    tol = stepref.lora_tolerance(want, mags, own, k, rank)
    off = np.abs(got[:, :n] - want)
    print("largest share of the tolerance", float((off / tol).max()), flush=True)
    assert (off <= tol).all()
    if base is not None:  # in place, to the bit
        ctx.lora_add(lora, d_ids, dx, rows, d_base, base=d_base, out_stride=n + strides[0], base_stride=n + strides[0])
        assert np.array_equal(d_base.numpy()[:, :n], got[:, :n]) and np.array_equal(d_base.numpy()[:, n:], base[:, n:])
    return lora, d_ids, dx, got


@pytest.mark.parametrize("xt", [np.float32, np.float16])
@pytest.mark.parametrize("rank", [8, 16, 24, 40, 64, 72, 128, 256])
@pytest.mark.parametrize("rows,k,n", [(1, 8, 1), (3, 520, 255), (17, 512, 256), (65, 1032, 100), (97, 136, 321), (150, 2600, 258)])
def test_lora(gpu_ctx, xt, rank, rows, k, n):
    _say("lora", np.dtype(xt).name, rank, rows, k, n)
    rng = np.random.default_rng(rank + rows + k)
    adapters = 5
    ids = rng.integers(-1, adapters, rows)  # some rows with none, tiles with several
    _lora_case(gpu_ctx, rng, rows, k, n, rank, adapters, ids, xt)


def _runs(rng, rows, adapters):
    """Adapters in runs of any length, from one row on; some rows with none."""
    ids = np.concatenate([np.full(n, rng.integers(-1, adapters)) for n in rng.choice([1, 2, 15, 16, 33, 200], rows)])
    return ids[:rows]


# (products of so many rows that they are taken in tiles)
@pytest.mark.parametrize("xt", [np.float32, np.float16])
@pytest.mark.parametrize("rank", [8, 16, 24, 40, 64, 72, 136, 256])
@pytest.mark.parametrize("k,n", [(2056, 2050), (5120, 321), (264, 7172)])
def test_lora_many_rows(gpu_ctx, xt, rank, k, n):
    rows = (4 << 20) // (k + n) + 19
    _say("lora many", np.dtype(xt).name, rank, rows, k, n)
    rng = np.random.default_rng(rank + rows + k)
    _lora_case(gpu_ctx, rng, rows, k, n, rank, 4, _runs(rng, rows, 4), xt)


# (base and out of more bytes than the caches are used for)
@pytest.mark.parametrize("rank,based,strides", [(8, True, (0, 0)), (40, True, (4, 12)), (72, False, (0, 4)), (136, True, (0, 0)),
                                                 (24, True, (1, 2))])
def test_lora_large_outputs(gpu_ctx, rank, based, strides):
    _say("lora large", rank, based, strides)
    rng = np.random.default_rng(rank)
    rows, k, n = 2051, 64, (8196 if based else 16388) + strides[0] % 2
    _lora_case(gpu_ctx, rng, rows, k, n, rank, 4, _runs(rng, rows, 4), np.float16, True, based, strides)


@pytest.mark.parametrize("xt", [np.float32, np.float16])
@pytest.mark.parametrize("scaled,based,strides", [(False, True, (0, 0)), (True, False, (0, 3)), (False, False, (0, 4)), (True, True, (8, 3)),
                                                  (True, True, (4, 8))])
def test_lora_many_rows_without_scale_or_base_and_with_strides(gpu_ctx, xt, scaled, based, strides):
    _say("lora many forms", np.dtype(xt).name, scaled, based, strides)
    rng = np.random.default_rng(5)
    rows = (4 << 20) // (1032 + 1024) + 70
    _lora_case(gpu_ctx, rng, rows, 1032, 1024, 16, 40, rng.integers(-2, 42, rows), xt, scaled, based, strides)


@pytest.mark.parametrize("xt", [np.float32, np.float16])
def test_lora_many_rows_not_finite_and_of_every_size(gpu_ctx, xt):
    _say("lora many not finite", np.dtype(xt).name)
    rng = np.random.default_rng(6)
    k, n, rank, adapters = 520, 640, 16, 3
    rows = (4 << 20) // (k + n) + 5
    a = rng.standard_normal((adapters, rank, k)).astype(np.float16)
    b = rng.standard_normal((adapters, n, rank)).astype(np.float16)
    x = (rng.standard_normal((rows, k)) * 10.0 ** rng.integers(-4, 4, (rows, 1))).astype(xt)
    ids = np.arange(rows) // 5 % adapters
    lora = arf_amd.Lora(gpu_ctx.to_device(a), gpu_ctx.to_device(b))
    out, d_ids = gpu_ctx.empty((rows, n), np.float32), gpu_ctx.to_device(ids.astype(np.int32))
    gpu_ctx.lora_add(lora, d_ids, gpu_ctx.to_device(x), rows, out)
    want, mags = stepref.lora(x, ids, a, b, None, None)
    assert (np.abs(out.numpy() - want) <= stepref.lora_tolerance(want, mags, None, k, rank)).all()
    a[1, 3, 5], b[2, 7, 1], x[3, 9] = np.nan, np.inf, np.inf  # (row 3 has adapter 0)
    lora = arf_amd.Lora(gpu_ctx.to_device(a), gpu_ctx.to_device(b))
    gpu_ctx.lora_add(lora, d_ids, gpu_ctx.to_device(x), rows, out)
    got = out.numpy()
    assert np.isfinite(got[(ids == 0) & (np.arange(rows) != 3)]).all() and np.isnan(got[ids == 1]).all() and not np.isfinite(got[3]).any()
    rest = np.arange(n) != 7
    assert np.isfinite(got[ids == 2][:, rest]).all() and not np.isfinite(got[ids == 2][:, 7]).any()


@pytest.mark.parametrize("xt", [np.float32, np.float16])
@pytest.mark.parametrize("rows,scaled,based,strides", [(4, False, True, (0, 0)), (4, True, False, (0, 3)), (200, False, False, (0, 4)),
                                                       (200, True, True, (8, 3)), (200, False, True, (1, 0)), (64, True, True, (5, 7))])
def test_lora_without_scale_or_base_and_with_strides(gpu_ctx, xt, rows, scaled, based, strides):
    _say("lora forms", np.dtype(xt).name, rows, scaled, based, strides)
    rng = np.random.default_rng(rows)
    ids = np.sort(rng.integers(0, 3, rows))
    _lora_case(gpu_ctx, rng, rows, 264, 132, 16, 3, ids, xt, scaled, based, strides)


@pytest.mark.parametrize("rows", [9, 300])
def test_lora_rows_with_none_and_strange_ids(gpu_ctx, rows):
    # ids outside [0, adapters): base, to the bit; the largest adapter number
    _say("lora ids", rows)
    rng = np.random.default_rng(rows)
    ids = rng.choice([-1, 0, 6, 7, 8, 2 ** 31 - 1, -2 ** 31], rows)
    _lora_case(gpu_ctx, rng, rows, 64, 96, 8, 7, ids, np.float32)
    base = rng.standard_normal((rows, 96)).astype(np.float32)
    d_base, out = gpu_ctx.to_device(base), gpu_ctx.to_device(np.full((rows, 96), 7, np.float32))
    one = np.zeros((1, 96, 8), np.float16)
    lora = arf_amd.Lora(gpu_ctx.to_device(one.reshape(1, 8, 96)), gpu_ctx.to_device(one))
    gpu_ctx.lora_add(lora, gpu_ctx.to_device(np.full(rows, -1, np.int32)), gpu_ctx.to_device(base), rows, out, base=d_base)
    assert np.array_equal(out.numpy(), base)
    gpu_ctx.lora_add(lora, gpu_ctx.to_device(np.full(rows, 1, np.int32)), gpu_ctx.to_device(base), rows, out)
    assert (out.numpy() == 0).all()


@pytest.mark.parametrize("xt", [np.float32, np.float16])
@pytest.mark.parametrize("rows", [6, 100])
def test_lora_what_is_not_finite_stays_with_its_rows(gpu_ctx, rows, xt):
    _say("lora not finite", rows, np.dtype(xt).name)
    rng = np.random.default_rng(rows)
    k, n, rank, adapters = 96, 80, 16, 3
    a = rng.standard_normal((adapters, rank, k)).astype(np.float16)
    b = rng.standard_normal((adapters, n, rank)).astype(np.float16)
    x = rng.standard_normal((rows, k)).astype(xt)
    ids = np.arange(rows) % adapters
    a[1, 3, 5], b[2, 7, 1], x[3, 9] = np.nan, np.inf, np.inf  # (row 3 has adapter 0)
    lora = arf_amd.Lora(gpu_ctx.to_device(a), gpu_ctx.to_device(b))
    out = gpu_ctx.empty((rows, n), np.float32)
    gpu_ctx.lora_add(lora, gpu_ctx.to_device(ids.astype(np.int32)), gpu_ctx.to_device(x), rows, out)
    got = out.numpy()
    clean = (ids == 0) & (np.arange(rows) != 3)
    assert np.isfinite(got[clean]).all() and np.isnan(got[ids == 1]).all() and not np.isfinite(got[3]).any()
    rest = np.arange(n) != 7
    assert np.isfinite(got[ids == 2][:, rest]).all() and not np.isfinite(got[ids == 2][:, 7]).any()


@pytest.mark.parametrize("rows", [5, 130])
def test_lora_small_and_large_values(gpu_ctx, rows):
    # rows of every size: h's parts go by the row's largest
    _say("lora sizes", rows)
    rng = np.random.default_rng(rows)
    k, n, rank = 128, 64, 32
    a, b = rng.standard_normal((2, rank, k)).astype(np.float16), rng.standard_normal((2, n, rank)).astype(np.float16)
    x = (rng.standard_normal((rows, k)) * 10.0 ** rng.integers(-30, 30, (rows, 1))).astype(np.float32)
    x[2] = 0
    ids = np.arange(rows) % 2
    out = gpu_ctx.empty((rows, n), np.float32)
    gpu_ctx.lora_add(arf_amd.Lora(gpu_ctx.to_device(a), gpu_ctx.to_device(b)), gpu_ctx.to_device(ids.astype(np.int32)),
                     gpu_ctx.to_device(x), rows, out)
    want, mags = stepref.lora(x, ids, a, b, None, None)
    assert (np.abs(out.numpy() - want) <= stepref.lora_tolerance(want, mags, None, k, rank)).all()


# ---- attention over chosen blocks ----

def _bounds(ctx, kv, batch):
    d = ctx.to_device(np.full((kv.n_pages, kv.heads, 2, kv.head_dim), 9, np.float16))
    ctx.kv_bounds(kv, batch.whole, d)
    return d


def _attend(ctx, kv, batch, d_bounds, q, out_dtype, scale, count, stride=None, **kw):
    tokens, hq, dim = q.shape
    out = ctx.to_device(np.full((tokens, hq, dim), 7, out_dtype))
    chosen = ctx.to_device(np.full((tokens, kv.heads, count), 55, np.int32))
    if stride:
        wide = np.full((tokens, stride), 3, q.dtype)
        wide[:, :hq * dim] = q.reshape(tokens, -1)
        q = wide
    ctx.kv_attention_blocks(kv, batch.seqs, d_bounds, ctx.to_device(q), out, hq, scale, count, chosen=chosen, q_stride=stride, **kw)
    return out.numpy(), chosen.numpy()


def _check(batch, got, chosen, q, hk, hv, scale, count, first=0, last=1, softcap=0.0, absent=None, rows=None):
    """rows: of each sequence, those that are looked at (all)."""
    f16 = got.dtype == np.float16 and q.dtype == np.float16
    worst = 0.0
    for b, (ln, n) in enumerate(zip(batch.lens, batch.news)):
        r, c = batch.start[b], batch.cached(b)
        if ln <= 0:
            assert (got[r:r + n] == 0).all() and (chosen[r:r + n] == -1).all(), b
            continue
        pick = range(n) if rows is None else [t for t in rows if t < n]
        bnd = stepref.bounds(hk[c], batch.page)
        for t in pick:
            part = slice(c.start, c.start + ln - n + t + 1)
            want, mag, eps, floor, keys, blocks = stepref.attend_blocks(
                q[r + t:r + t + 1], hk[part], hv[part], batch.page, scale, count, first, last, softcap,
                None if absent is None else absent[b], bnd)
            assert np.array_equal(chosen[r + t], blocks[0]), (b, ln, n, t)
            g, want = got[r + t].astype(np.float64), want[0]
            assert np.array_equal(np.isnan(g), np.isnan(want)), (b, t)
            ok = ~np.isnan(want)
            tol = kvref.tolerance(want, mag[0], eps[0], floor[0], keys, f16)
            if got.dtype == np.float16 and not f16:
                tol = tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
            off = np.abs(g - want)
            worst = max(worst, float((off / tol)[ok].max()) if ok.any() else 0.0)
            assert (off[ok] <= tol[ok]).all(), (b, ln, n, t, float((off / tol)[ok].max()))
    print("largest share of the tolerance", worst, flush=True)


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,page", [(1, 16), (3, 48), (2, 256)])
def test_bounds(gpu_ctx, dim, heads, page):
    _say("bounds", dim, heads, page)
    rng = np.random.default_rng(dim + page)
    batch = Batch(gpu_ctx, [1, 700, 0, 17, page, page + 1], [1, 650, 1, 1, page, 2], page, rng, spare=3)
    kv = gpu_ctx.kv_cache(heads, dim, page, batch.n_pages)
    k = _rows(rng, int(batch.whole_start[-1]), heads, dim, np.float32)
    k[5, 0, 3] = np.nan
    k[40] = 0
    gpu_ctx.kv_write(kv, batch.whole, gpu_ctx.to_device(k), gpu_ctx.to_device(k))
    hk, _ = kvref.held_pair(k, k)
    want = np.full((batch.n_pages, heads, 2, dim), 9.0)
    for b, ln in enumerate(batch.lens):
        if ln:
            want[batch.table[b, :-(-ln // page)]] = stepref.bounds(hk[batch.cached(b)], page)
    got = _bounds(gpu_ctx, kv, batch).numpy().astype(np.float64)
    assert np.array_equal(got, want, equal_nan=True)
    # the step's rows: the pages that they lie in, no others
    d = gpu_ctx.to_device(np.full(want.shape, 9, np.float16))
    gpu_ctx.kv_bounds(kv, batch.seqs, d)
    part = np.full(want.shape, 9.0)
    for b, (ln, n) in enumerate(zip(batch.lens, batch.news)):
        if ln:
            ids = batch.table[b, max(ln - n, 0) // page:-(-ln // page)]
            part[ids] = want[ids]
    assert np.array_equal(d.numpy().astype(np.float64), part, equal_nan=True)


@pytest.mark.parametrize("qt,ot", [(np.float32, np.float32), (np.float16, np.float16), (np.float32, np.float16), (np.float16, np.float32)])
@pytest.mark.parametrize("dim,heads,group,page", [(64, 2, 1, 16), (96, 1, 3, 48), (128, 3, 8, 64), (256, 2, 16, 16), (64, 1, 20, 32),
                                                  (128, 1, 33, 16)])
def test_chosen_blocks(gpu_ctx, qt, ot, dim, heads, group, page):
    _say("blocks", np.dtype(qt).name, np.dtype(ot).name, dim, heads, group, page)
    rng = np.random.default_rng(dim + group + page)
    # prompts, drafts, single tokens, an idle slot, one that all blocks of are chosen, ends inside a block and on its border
    batch = Batch(gpu_ctx, [page * 9 + 5, 1, 0, page * 12, page * 7 + 1, 20, 37], [3, 1, 1, 1, 17, 2, 37], page, rng, spare=2)
    kv = gpu_ctx.kv_cache(heads, dim, page, batch.n_pages)
    hk, hv = _filled(gpu_ctx, kv, batch, rng)
    d_bounds = _bounds(gpu_ctx, kv, batch)
    q = _rows(rng, batch.tokens, heads * group, dim, qt, False)
    for kw in (dict(count=4), dict(count=5, first=2, last=2, softcap=20.0), dict(count=1), dict(count=3, first=1, last=2), dict(count=40)):
        for scale in (dim ** -0.5, -0.02):
            got, chosen = _attend(gpu_ctx, kv, batch, d_bounds, q, ot, scale, **kw)
            _check(batch, got, chosen, q, hk, hv, scale, **kw)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("lens,count,page,heads,group,dim", [([40000], 64, 16, 1, 4, 64), ([9000, 33], 100, 16, 2, 5, 96),
                                                             ([6001, 4100], 9, 256, 2, 8, 128), ([20000, 3], 40, 64, 1, 2, 256)])
def test_long_sequences(gpu_ctx, dtype, lens, count, page, heads, group, dim):
    # more blocks than a thread keeps (2048), keys in several pieces, waves with several runs of blocks
    _say("blocks long", np.dtype(dtype).name, lens, count, page, heads, group, dim)
    rng = np.random.default_rng(count)
    batch = Batch(gpu_ctx, lens, [1] * len(lens), page, rng, use_start=False)
    kv = gpu_ctx.kv_cache(heads, dim, page, batch.n_pages)
    hk, hv = _filled(gpu_ctx, kv, batch, rng)
    q = _rows(rng, batch.tokens, heads * group, dim, dtype, False)
    kw = dict(count=count, first=1, last=2)
    got, chosen = _attend(gpu_ctx, kv, batch, _bounds(gpu_ctx, kv, batch), q, dtype, dim ** -0.5, stride=heads * group * dim + 32, **kw)
    _check(batch, got, chosen, q, hk, hv, dim ** -0.5, **kw)


@pytest.mark.parametrize("heads,group,dim,lens,news", [(8, 4, 64, [1700, 900], [300, 250]), (16, 3, 96, [700, 2100], [130, 131]),
                                                       (40, 2, 128, [1337], [70])])
def test_prompts_of_more_tiles_than_compute_units(gpu_ctx, heads, group, dim, lens, news):
    # (waves' shares of the blocks that do not come out even; a tile with rows of two sequences)
    _say("blocks of prompts", heads, group, dim, lens, news)
    rng = np.random.default_rng(heads)
    batch = Batch(gpu_ctx, lens, news, 16, rng)
    kv = gpu_ctx.kv_cache(heads, dim, 16, batch.n_pages)
    hk, hv = _filled(gpu_ctx, kv, batch, rng)
    q = _rows(rng, batch.tokens, heads * group, dim, np.float16, False)
    kw = dict(count=10, first=1, last=2)
    got, chosen = _attend(gpu_ctx, kv, batch, _bounds(gpu_ctx, kv, batch), q, np.float16, dim ** -0.5, **kw)
    _check(batch, got, chosen, q, hk, hv, dim ** -0.5, rows=[0, 1, 2, 3, 66, 127, 129, 130, 249, 298, 299], **kw)


def test_alike_blocks_the_earlier_first(gpu_ctx):
    # keys alike everywhere; alike in runs; scores of zero, +0 and -0
    _say("blocks alike")
    rng = np.random.default_rng(1)
    page, dim = 16, 64
    batch = Batch(gpu_ctx, [page * 300 + 3], [2], page, rng)
    kv = gpu_ctx.kv_cache(1, dim, page, batch.n_pages)
    rows = int(batch.whole_start[-1])
    q = _rows(rng, 2, 2, dim, np.float32, False)
    for k in (np.ones((rows, 1, dim)), np.zeros((rows, 1, dim)), np.sign(rng.standard_normal((1, 1, dim))) * (np.arange(rows) // (page * 7) % 3)[:, None, None]):
        k = k.astype(np.float32)
        v = _rows(rng, rows, 1, dim, np.float32, False)
        gpu_ctx.kv_write(kv, batch.whole, gpu_ctx.to_device(k), gpu_ctx.to_device(v))
        hk, hv = kvref.held_pair(k, v)
        kw = dict(count=50, first=1, last=3)
        for x in (q, np.zeros_like(q), -np.zeros_like(q)):
            got, chosen = _attend(gpu_ctx, kv, batch, _bounds(gpu_ctx, kv, batch), x, np.float32, 0.125, **kw)
            _check(batch, got, chosen, x, hk, hv, 0.125, **kw)


def test_scores_of_every_size(gpu_ctx):
    # keys over 2^40, so that the counted ranges are cut again and again; scores that differ in their last bits
    _say("blocks sizes")
    rng = np.random.default_rng(8)
    page, dim, n = 16, 64, 400
    batch = Batch(gpu_ctx, [page * n], [1], page, rng, use_start=False)
    kv = gpu_ctx.kv_cache(1, dim, page, batch.n_pages)
    size = np.exp2(rng.integers(-20, 13, n)).repeat(page)
    k = (rng.choice([-1, 1], (page * n, 1, dim)) * size[:, None, None]).astype(np.float32)
    v = _rows(rng, page * n, 1, dim, np.float32, False)
    gpu_ctx.kv_write(kv, batch.whole, gpu_ctx.to_device(k), gpu_ctx.to_device(v))
    hk, hv = kvref.held_pair(k, v)
    q = np.exp2(rng.integers(-30, 3, (1, 1, dim))).astype(np.float32) * 1e-3
    for count in (2, 60, 200, 399):
        got, chosen = _attend(gpu_ctx, kv, batch, _bounds(gpu_ctx, kv, batch), q, np.float32, 1.0, count=count)
        _check(batch, got, chosen, q, hk, hv, 1.0, count=count)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_not_finite_and_pages_that_are_not_the_caches(gpu_ctx, dtype):
    _say("blocks bad", np.dtype(dtype).name)
    rng = np.random.default_rng(4)
    page, heads, dim, group = 16, 2, 128, 4
    batch = Batch(gpu_ctx, [page * 30 + 4, page * 10], [1, 1], page, rng)
    rows = int(batch.whole_start[-1])
    kv = gpu_ctx.kv_cache(heads, dim, page, batch.n_pages)
    k, v = (_rows(rng, rows, heads, dim, np.float32) for _ in "kv")
    k[7 * page + 3, 1, 9] = np.inf  # that key of head 1 is NaN: its block comes first, and the row's head is NaN
    v[page * 30 + 4 + 20, 0, 70] = np.nan  # key NaN, too, of the second sequence's head 0
    gpu_ctx.kv_write(kv, batch.whole, gpu_ctx.to_device(k), gpu_ctx.to_device(v))
    hk, hv = kvref.held_pair(k, v)
    d_bounds = _bounds(gpu_ctx, kv, batch)
    # blocks 3 (by rule), 12 and 20 of the first sequence are nowhere
    table, absent = batch.table.copy(), [np.zeros(31, bool), np.zeros(10, bool)]
    table[0, [0, 12, 20]] = [-1, batch.n_pages, 2 ** 31 - 1]
    absent[0][[0, 12, 20]] = True
    batch.d_table.upload(table)
    q = _rows(rng, 2, heads * group, dim, dtype, False)
    for kw in (dict(count=6, first=1, last=1), dict(count=30), dict(count=31)):
        got, chosen = _attend(gpu_ctx, kv, batch, d_bounds, q, dtype, dim ** -0.5, **kw)
        _check(batch, got, chosen, q, hk, hv, dim ** -0.5, absent=absent, **kw)
    q[0, 1, 5] = np.nan  # a head's q: all its group's scores are NaN, the earliest blocks come; the other head's stay
    q[1, 7, 6] = np.inf
    got, chosen = _attend(gpu_ctx, kv, batch, d_bounds, q, dtype, dim ** -0.5, count=6)
    assert np.array_equal(chosen[0, 0], [0, 1, 2, 3, 4, 30]) or np.array_equal(chosen[0, 0], [1, 2, 3, 4, 5, 30])
    assert np.isnan(got[0, 1]).all() and np.isfinite(got[0, 0]).all()


def test_rows_of_no_sequence(gpu_ctx):
    # left as they were, out and chosen; none from where start decreases on
    _say("blocks nobody")
    rng = np.random.default_rng(6)
    page, heads, dim = 16, 1, 64
    batch = Batch(gpu_ctx, [100, 200, 60], [2, 3, 2], page, rng)
    kv = gpu_ctx.kv_cache(heads, dim, page, batch.n_pages)
    hk, hv = _filled(gpu_ctx, kv, batch, rng)
    d_bounds = _bounds(gpu_ctx, kv, batch)
    q = _rows(rng, 12, 2, dim, np.float32, False)
    for start, owned in (([0, 2, 5, 7], range(7)), ([1, 3, 6, 8], range(1, 8)), ([0, 2, 5, 4], range(5)), ([0, 2, 1, 3], range(2)),
                         ([0, 2, 5, 13], range(5)), ([-1, 2, 5, 7], range(2, 7))):
        seqs = arf_amd.KVSeqs(batch.d_table, batch.d_len, gpu_ctx.to_device(np.array(start, np.int32)), 12)
        out, chosen = gpu_ctx.to_device(np.full(q.shape, 7, np.float32)), gpu_ctx.to_device(np.full((12, 1, 3), 55, np.int32))
        gpu_ctx.kv_attention_blocks(kv, seqs, d_bounds, gpu_ctx.to_device(q), out, 2, 0.125, 3, chosen=chosen)
        rest = np.setdiff1d(np.arange(12), list(owned))
        assert (out.numpy()[rest] == 7).all() and (chosen.numpy()[rest] == 55).all()
        assert (chosen.numpy()[list(owned), 0, 0] >= 0).all() and (out.numpy()[list(owned)] != 7).all()


def test_rows_in_several_chunks(gpu_ctx):
    # a table so wide that the scores of all rows at once pass the workspace's bound; chosen may be left out
    _say("blocks chunks")
    rng = np.random.default_rng(7)
    page, heads, dim, group, n = 16, 8, 64, 2, 1500
    batch = Batch(gpu_ctx, [2000, 1300], [n, 700], page, rng)
    wide = np.full((2, 6000), -1, np.int32)
    wide[:, :batch.table.shape[1]] = batch.table
    batch.d_table = gpu_ctx.to_device(wide)
    batch.seqs = arf_amd.KVSeqs(batch.d_table, batch.d_len, batch.d_start, batch.tokens)
    batch.whole = arf_amd.KVSeqs(batch.d_table, batch.d_len, batch.d_whole, int(batch.whole_start[-1]))
    kv = gpu_ctx.kv_cache(heads, dim, page, batch.n_pages)
    hk, hv = _filled(gpu_ctx, kv, batch, rng)
    q = _rows(rng, batch.tokens, heads * group, dim, np.float32, False)
    kw = dict(count=12, first=1, last=2)
    d_bounds = _bounds(gpu_ctx, kv, batch)
    assert gpu_ctx.kv_attention_blocks_workspace(kv, batch.seqs, heads * group, 12) < 300 << 20
    got, chosen = _attend(gpu_ctx, kv, batch, d_bounds, q, np.float32, 0.125, **kw)
    chunk = (256 << 20) // (heads * (6000 * 8 + 12 * 4))
    _check(batch, got, chosen, q, hk, hv, 0.125, rows=[0, 1, 300, chunk - 1, chunk, chunk + 1, 699, n - 1], **kw)
    out = gpu_ctx.empty(q.shape, np.float32)
    gpu_ctx.kv_attention_blocks(kv, batch.seqs, d_bounds, gpu_ctx.to_device(q), out, heads * group, 0.125, 12, first=1, last=2)
    assert np.array_equal(out.numpy(), got)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("lens,count,width", [([40005, 100], 2100, 0), ([9000, 2000, 400], 20, 17000), ([40005], 2300, 17000)])
def test_choices_in_a_launch_of_their_own(gpu_ctx, dtype, lens, count, width):
    # more chosen blocks than the attention's workgroups keep, and tables wider than they look through
    _say("blocks wide", np.dtype(dtype).name, lens, count, width)
    rng = np.random.default_rng(count + width)
    page, heads, dim, group = 16, 2, 64, 3
    batch = Batch(gpu_ctx, lens, [2] * len(lens), page, rng)
    if width:
        wide = np.full((len(lens), width), -1, np.int32)
        wide[:, :batch.table.shape[1]] = batch.table
        batch.d_table = gpu_ctx.to_device(wide)
        batch.seqs = arf_amd.KVSeqs(batch.d_table, batch.d_len, batch.d_start, batch.tokens)
        batch.whole = arf_amd.KVSeqs(batch.d_table, batch.d_len, batch.d_whole, int(batch.whole_start[-1]))
    kv = gpu_ctx.kv_cache(heads, dim, page, batch.n_pages)
    hk, hv = _filled(gpu_ctx, kv, batch, rng)
    q = _rows(rng, batch.tokens, heads * group, dim, dtype, False)
    kw = dict(count=count, first=2, last=3)
    got, chosen = _attend(gpu_ctx, kv, batch, _bounds(gpu_ctx, kv, batch), q, dtype, 0.125, **kw)
    _check(batch, got, chosen, q, hk, hv, 0.125, **kw)


def test_all_blocks_are_what_attention_takes(gpu_ctx):
    # count from the table's width on: kv_attention's rows
    _say("blocks all")
    rng = np.random.default_rng(9)
    batch = Batch(gpu_ctx, [500, 31, 0, 1000], [4, 1, 1, 1], 32, rng)
    kv = gpu_ctx.kv_cache(2, 128, 32, batch.n_pages)
    hk, hv = _filled(gpu_ctx, kv, batch, rng)
    q = _rows(rng, batch.tokens, 8, 128, np.float32, False)
    got, chosen = _attend(gpu_ctx, kv, batch, _bounds(gpu_ctx, kv, batch), q, np.float32, 0.1, count=64)
    _check(batch, got, chosen, q, hk, hv, 0.1, count=64)


def test_bounds_and_pages_beyond_32_bits_of_bytes(gpu_ctx):
    _say("blocks far")
    rng = np.random.default_rng(10)
    page, heads, dim, far = 16, 32, 256, 140000  # 1 KB of bounds and 4.5 KB of codes a page and head: 4.6 GB, 20 GB
    kv = gpu_ctx.kv_cache(heads, dim, page, far)
    batch = Batch(gpu_ctx, [page * 6 + 2, 40], [1, 1], page, rng)
    batch.table = np.where(batch.table >= 0, far - 1 - batch.table, -1).astype(np.int32)
    batch.d_table.upload(batch.table)
    hk, hv = _filled(gpu_ctx, kv, batch, rng)
    d_bounds = gpu_ctx.empty((far, heads, 2, dim), np.float16)
    gpu_ctx.kv_bounds(kv, batch.whole, d_bounds)
    q = _rows(rng, 2, heads, dim, np.float16, False)
    got, chosen = _attend(gpu_ctx, kv, batch, d_bounds, q, np.float16, 0.0625, count=3)
    _check(batch, got, chosen, q, hk, hv, 0.0625, count=3)
    kv.free()


# ---- refusals ----

def test_refusals(gpu_ctx):
    _say("refusals")
    up = gpu_ctx.to_device
    i32 = lambda *s: up(np.zeros(s, np.int32))
    # plan
    def step(**kw):
        a = dict(page_size=16, add=i32(2), held=i32(2), held_next=i32(2), pages=i32(2, 4), free=i32(8), n_free=i32(1), n_free_next=i32(1),
                 start=i32(3), lens=i32(2), taken=i32(3), freed=i32(3), positions=i32(5), slots=up(np.zeros(5, np.int64)))
        a.update(kw)
        return arf_amd.KVStep(**a)
    gpu_ctx.kv_plan(step())
    for kw in (dict(page_size=0), dict(page_size=65537), dict(start=i32(2)), dict(slots=i32(5)), dict(lens=i32(3)), dict(pages=i32(8)),
               dict(positions=up(np.zeros(5, np.float32)))):
        with pytest.raises(ValueError):
            gpu_ctx.kv_plan(step(**kw))
    same, wider, one = i32(2), i32(3), i32(1)
    for kw in (dict(held=same, held_next=same), dict(add=same, lens=same), dict(lens=same, held_next=same), dict(start=wider, freed=wider),
               dict(taken=wider, freed=wider), dict(n_free=one, n_free_next=one)):
        with pytest.raises(arf_amd.ArfqError, match="places of their own"):
            gpu_ctx.kv_plan(step(**kw))
    bad = step()
    for field, value, status in (("tokens", -1, arfq.ARFQ_E_SHAPE), ("tokens", (1 << 30) + 1, arfq.ARFQ_E_SHAPE), ("batch", 16385, arfq.ARFQ_E_SHAPE),
                                 ("max_pages", 1 << 30, arfq.ARFQ_E_SHAPE), ("n_pages", 1 << 31, arfq.ARFQ_E_SHAPE), ("add", None, arfq.ARFQ_E_INVALID),
                                 ("slots", None, arfq.ARFQ_E_INVALID), ("freed", None, arfq.ARFQ_E_INVALID)):
        bad = step()
        setattr(bad.struct, field, value)
        assert arfq._lib.arfq_kv_plan(gpu_ctx.handle, bad.ref) == status, field
    assert arfq._lib.arfq_kv_plan(gpu_ctx.handle, None) == arfq.ARFQ_E_INVALID
    # rope
    x, pos = up(np.zeros((4, 64), np.float32)), i32(4)
    rope = arf_amd.Rope.sections([16])
    for kw in (dict(head_dim=63), dict(head_dim=2048), dict(tokens=5), dict(head_dim=24), dict(x_stride=65)):
        a = dict(tokens=1, heads=1, head_dim=64)
        a.update(kw)
        with pytest.raises((ValueError, arf_amd.ArfqError)):
            gpu_ctx.rope(rope, pos, x, x, **a)
    with pytest.raises(ValueError, match="axes"):
        gpu_ctx.rope(arf_amd.Rope.sections([8, 8]), pos, x, x, 1, 1, 64)
    with pytest.raises(ValueError, match="position_stride|hold"):
        gpu_ctx.rope(rope, i32(1, 3), x, x, 4, 1, 64)
    with pytest.raises(arf_amd.ArfqError, match="finite"):
        gpu_ctx.rope(arf_amd.Rope([np.inf] * 16), pos, x, x, 4, 1, 64)
    with pytest.raises(arf_amd.ArfqError, match="in place"):
        gpu_ctx.rope(rope, pos, x, x, 2, 1, 32, x_stride=64)
    with pytest.raises(ValueError, match="rot_dim"):
        gpu_ctx.rope(arf_amd.Rope.sections([7]), pos, x, x, 4, 1, 64)
    with pytest.raises(ValueError):
        gpu_ctx.rope(arf_amd.Rope.sections([2, 2, 2, 2, 8]), i32(5, 4), x, x, 4, 1, 64)
    with pytest.raises(ValueError):
        gpu_ctx.rope(rope, up(np.zeros(4, np.int64)), x, x, 4, 1, 64)
    # adapters
    a, b = up(np.zeros((2, 8, 16), np.float16)), up(np.zeros((2, 5, 8), np.float16))
    y = up(np.zeros((3, 5), np.float32))
    lx = up(np.zeros((3, 16), np.float32))
    gpu_ctx.lora_add(arf_amd.Lora(a, b), i32(3), lx, 3, y)
    for la, lb in (((2, 4, 16), (2, 5, 4)), ((2, 264, 16), (2, 5, 264)), ((2, 8, 12), (2, 5, 8))):
        with pytest.raises(arf_amd.ArfqError) as e:
            gpu_ctx.lora_add(arf_amd.Lora(up(np.zeros(la, np.float16)), up(np.zeros(lb, np.float16))), i32(3), lx, 3, y)
        assert e.value.status == arfq.ARFQ_E_UNSUPPORTED
    lora = arf_amd.Lora(a, b)
    big = arf_amd.Lora(up(np.zeros((1, 8, 16392), np.float16)), up(np.zeros((1, 5, 8), np.float16)))  # (in two launches)
    for bad in (lambda: arf_amd.Lora(a, a), lambda: arf_amd.Lora(lx, b), lambda: arf_amd.Lora(a, b, i32(2)),
                lambda: gpu_ctx.lora_add(lora, i32(2), lx, 3, y), lambda: gpu_ctx.lora_add(lora, i32(4), lx, 4, y),
                lambda: gpu_ctx.lora_add(lora, i32(3), lx, 3, y, out_stride=6), lambda: gpu_ctx.lora_add(lora, i32(3), lx, 3, lx, base_stride=4, base=y),
                lambda: gpu_ctx.lora_add(big, i32(1), up(np.zeros((1, 16392), np.float32)), 1, y, workspace=up(np.zeros(4, np.uint8)))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(arf_amd.ArfqError, match="in place"):
        gpu_ctx.lora_add(lora, i32(2), lx, 2, y, base=y, base_stride=6)
    # bounds and blocks
    kv = gpu_ctx.kv_cache(2, 64, 16, 8)
    seqs = arf_amd.KVSeqs(i32(1, 4), i32(1))
    bounds, q = up(np.zeros((8, 2, 2, 64), np.float16)), up(np.zeros((1, 4, 64), np.float32))
    gpu_ctx.kv_attention_blocks(kv, seqs, bounds, q, q, 4, 0.1, 2)
    for kw in (dict(count=0), dict(count=(1 << 20) + 1), dict(first=-1), dict(last=0), dict(first=2, last=1), dict(q_heads=3),
               dict(chosen=i32(1)), dict(bounds=up(np.zeros((7, 2, 2, 64), np.float16))), dict(scale=float("nan")),
               dict(softcap=-1.0), dict(workspace=up(np.zeros(16, np.uint8)))):
        a = dict(bounds=bounds, q=q, out=q, q_heads=4, scale=0.1, count=2)
        a.update(kw)
        with pytest.raises((ValueError, arf_amd.ArfqError)):
            gpu_ctx.kv_attention_blocks(kv, seqs, **a)
    with pytest.raises(ValueError):
        gpu_ctx.kv_bounds(kv, seqs, up(np.zeros((8, 2, 2, 64), np.float32)))
    kv.free()
