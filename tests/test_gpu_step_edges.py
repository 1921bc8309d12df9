"""Where a serving step's operators could be off without the other tests' notice: adapters' bits by the norm of the errors, in every
form of the tiles and one by one, and on both sides of the borders between kernels."""
import numpy as np
import pytest

import arf_amd
import kvref
import stepref
from test_gpu_kv import Batch, _filled, _rows, _say
from test_gpu_step import _attend, _bounds, _check, _lora_case
from test_step_edges_cpu import RANKS, SHAPES

pytestmark = pytest.mark.gpu


def _sample(rng, rows):
    """Rows that are looked at: the first, the last, others in between."""
    return np.unique(np.concatenate([np.arange(min(rows, 40)), np.arange(max(rows - 40, 0), rows), rng.integers(0, rows, 150)]))


def _adapters(ctx, rng, rows, k, n, rank, ids, xt, based=True, skip=0):
    """out = base + adapters' products, `skip` elements of x into an allocation; against the oracle by value and by norm."""
    adapters = 4
    a = (rng.standard_normal((adapters, rank, k)) / np.sqrt(k)).astype(np.float16)
    b = rng.standard_normal((adapters, n, rank)).astype(np.float16)
    x = rng.standard_normal((rows, k), dtype=np.float32).astype(xt)
    scale = (rng.random(adapters) + 0.5).astype(np.float32)
    base = rng.standard_normal((rows, n), dtype=np.float32) if based else None
    dx = ctx.to_device(np.concatenate([np.zeros(skip, xt), x.reshape(-1)]))
    lora = arf_amd.Lora(ctx.to_device(a), ctx.to_device(b), ctx.to_device(scale))
    out = ctx.empty((rows, n), np.float32)
    ctx.lora_add(lora, ctx.to_device(np.asarray(ids, np.int32)), dx.columns(skip) if skip else dx, rows, out,
                 base=ctx.to_device(base) if based else None)
    s = _sample(rng, rows)
    own = base[s] if based else None
    want, mags = stepref.lora(x[s], np.asarray(ids)[s], a, b, scale, own)
    off = out.numpy()[s] - want
    assert (np.abs(off) <= stepref.lora_tolerance(want, mags, own, k, rank)).all()
    most = stepref.lora_norm_tolerance(want, own, k, rank)
    print("share of the norm's tolerance", float(np.linalg.norm(off) / most), flush=True)
    assert np.linalg.norm(off) <= most


def _runs(rng, rows):
    return np.repeat(rng.integers(0, 4, rows), rng.choice([1, 2, 15, 16, 33, 200], rows))[:rows]


# rows * (k + n) * (rank + 8) from which on every shape and type is taken in tiles
IN_TILES = 1.3e9


@pytest.mark.parametrize("xt", [np.float32, np.float16])
@pytest.mark.parametrize("rank", RANKS)
@pytest.mark.parametrize("k,n", SHAPES)
def test_adapters_in_tiles_keep_their_bits(gpu_ctx, xt, rank, k, n):
    rows = int(IN_TILES / ((k + n) * (rank + 8))) + 19
    _say("adapters' bits", np.dtype(xt).name, rank, rows, k, n)
    rng = np.random.default_rng(rank + k)
    _adapters(gpu_ctx, rng, rows, k, n, rank, _runs(rng, rows), xt, based=rank % 16 == 8 or rank == 64)


@pytest.mark.parametrize("xt", [np.float32, np.float16])
@pytest.mark.parametrize("rank", [8, 64, 136])
@pytest.mark.parametrize("rows,k,n", [(1, 5120, 700), (33, 2056, 2050), (70, 264, 1172)])
def test_adapters_one_by_one_keep_their_bits(gpu_ctx, xt, rank, rows, k, n):
    _say("adapters' bits, few rows", np.dtype(xt).name, rank, rows, k, n)
    rng = np.random.default_rng(rank + k)
    _adapters(gpu_ctx, rng, rows, k, n, rank, rng.integers(0, 4, rows), xt)


@pytest.mark.parametrize("xt", [np.float32, np.float16])
@pytest.mark.parametrize("rank", [8, 32, 64])
@pytest.mark.parametrize("rows", [0, 3, 70])  # 0: in tiles
def test_adapters_of_x_at_any_16_bytes(gpu_ctx, xt, rank, rows):
    _say("adapters, x 16 bytes on", np.dtype(xt).name, rank, rows)
    rng = np.random.default_rng(rank + rows)
    k, n = 520, 648
    rows = rows or int(IN_TILES / ((k + n) * (rank + 8))) + 19
    _adapters(gpu_ctx, rng, rows, k, n, rank, _runs(rng, rows), xt, skip=16 // np.dtype(xt).itemsize)


def test_refusals_name_their_call(gpu_ctx):
    _say("refusals' names")
    up = lambda shape, t=np.float32: gpu_ctx.to_device(np.zeros(shape, t))
    kv, seqs = gpu_ctx.kv_cache(2, 64, 16, 8), arf_amd.KVSeqs(up((1, 4), np.int32), up(1, np.int32))
    bounds, q = up((8, 2, 2, 64), np.float16), up((1, 4, 64))
    wide = arf_amd.Lora(up((1, 12, 16), np.float16), up((1, 5, 12), np.float16))
    few = arf_amd.KVSeqs(up((1, 4), np.int32), up(1, np.int32), None, 2)
    for call, name, why in (
            (lambda: gpu_ctx.kv_attention_blocks(kv, seqs, bounds, q, q, 3, 0.1, 2), "kv_attention_blocks", "multiple of the cache's heads"),
            (lambda: gpu_ctx.kv_attention_blocks_workspace(kv, seqs, 3, 2), "kv_attention_blocks_workspace", "multiple of the cache's heads"),
            (lambda: gpu_ctx.kv_attention_blocks(kv, seqs, bounds, q, q, 4, 0.1, 2, workspace=up(16, np.uint8)), "kv_attention_blocks",
             "workspace of 16 bytes, [0-9]+ \\(16-byte aligned\\) are wanted"),
            (lambda: gpu_ctx.kv_attention(kv, seqs, q, q, 3, 0.1), "kv_attention", "multiple of the cache's heads"),
            (lambda: gpu_ctx.kv_bounds(kv, few, bounds), "kv_bounds", "more rows than sequences, and no start"),
            (lambda: gpu_ctx.rope(arf_amd.Rope.sections([16]), up(1, np.int32), q, q, 1, 2, 64, x_stride=130), "rope: x", "multiples of 16 bytes"),
            (lambda: gpu_ctx.lora_add(wide, up(1, np.int32), up((1, 16)), 1, up((1, 5))), "lora_add", "rank must be a multiple of 8 up to 256"),
            (lambda: gpu_ctx.lora_workspace(wide, 1), "lora_workspace", "rank must be a multiple of 8 up to 256")):
        with pytest.raises((ValueError, arf_amd.ArfqError), match=f"{name}: .*{why}"):
            call()
    kv.free()


def test_adapters_mixed_rows_stay_one_by_one(gpu_ctx):
    # 512 rows of rank 16 whose adapters may change from row to row: the parts of k are those of rows one by one (11 of 512)
    _say("adapters' border")
    rng = np.random.default_rng(1)
    k, n, rank = 5128, 7160, 16
    lora = arf_amd.Lora(gpu_ctx.empty((4, rank, k), np.float16), gpu_ctx.empty((4, n, rank), np.float16))
    assert gpu_ctx.lora_workspace(lora, 512) == 11 * 512 * rank * 4
    # a workspace of the bytes that are asked for does for both types, on either side of either's border
    k, n, rank = 1032, 1040, 64
    a, b = ((rng.standard_normal(s) / 8).astype(np.float16) for s in ((4, rank, k), (4, n, rank)))
    lora = arf_amd.Lora(gpu_ctx.to_device(a), gpu_ctx.to_device(b))
    for rows in (2000, 2100, 4000, 4100):
        ids, x = rng.integers(0, 4, rows), rng.standard_normal((rows, k), dtype=np.float32)
        need = gpu_ctx.lora_workspace(lora, rows)
        ws, d_ids, out = gpu_ctx.to_device(np.zeros(need, np.uint8)), gpu_ctx.to_device(ids.astype(np.int32)), gpu_ctx.empty((rows, n), np.float32)
        for xt in (np.float32, np.float16):
            gpu_ctx.lora_add(lora, d_ids, gpu_ctx.to_device(x.astype(xt)), rows, out, workspace=ws)
            s = _sample(rng, rows)
            want, mags = stepref.lora(x.astype(xt)[s], ids[s], a, b, None, None)
            assert (np.abs(out.numpy()[s] - want) <= stepref.lora_tolerance(want, mags, None, k, rank)).all()


@pytest.mark.parametrize("xt", [np.float32, np.float16])
@pytest.mark.parametrize("rank,k,n", [(8, 64, 64), (16, 256, 2049), (64, 264, 700)])
def test_adapters_of_many_small_rows_take_two_launches(gpu_ctx, xt, rank, k, n):
    # one launch while two workgroups (of 1024 outputs) a compute unit do, one above rank 32
    most = (256 if rank > 32 else 512) // -(-n // 1024)
    for rows in (most, most + 1, 3 * most):
        _say("adapters, small rows", np.dtype(xt).name, rank, rows, k, n)
        rng = np.random.default_rng(rank + rows)
        _adapters(gpu_ctx, rng, rows, k, n, rank, rng.integers(0, 4, rows), xt)
        lora = arf_amd.Lora(gpu_ctx.empty((4, rank, k), np.float16), gpu_ctx.empty((4, n, rank), np.float16))
        assert (gpu_ctx.lora_workspace(lora, rows) == 0) == (rows == most)


def _rows_in_tiles(k, n, rank, xt):
    return int((6.1e8 if xt == np.float32 else 3.1e8) / ((k + n) * (rank + 8))) + 19


@pytest.mark.parametrize("xt", [np.float32, np.float16])
@pytest.mark.parametrize("rank,scaled,based,strides", [(16, False, True, (0, 0)), (16, True, False, (0, 3)), (40, False, False, (0, 4)),
                                                       (16, True, True, (8, 3)), (136, True, True, (4, 8)), (72, True, True, (1, 0))])
def test_adapters_in_tiles_without_scale_or_base_and_with_strides(gpu_ctx, xt, rank, scaled, based, strides):
    _say("adapters in tiles, forms", np.dtype(xt).name, rank, scaled, based, strides)
    rng = np.random.default_rng(rank)
    rows = _rows_in_tiles(1032, 1024, rank, xt)
    _lora_case(gpu_ctx, rng, rows, 1032, 1024, rank, 40, rng.integers(-2, 42, rows), xt, scaled, based, strides)


def test_adapters_in_tiles_of_the_smallest_rank_past_the_caches(gpu_ctx):
    _say("adapters in tiles, large")
    rng = np.random.default_rng(8)
    rows = _rows_in_tiles(64, 8196, 8, np.float16)
    _lora_case(gpu_ctx, rng, rows, 64, 8196, 8, 4, _runs(rng, rows), np.float16)


@pytest.mark.parametrize("xt", [np.float32, np.float16])
@pytest.mark.parametrize("rank", [16, 72])
def test_adapters_in_tiles_what_is_not_finite_stays_with_its_rows(gpu_ctx, xt, rank):
    # and rows of every size: h's parts go by the row's largest
    _say("adapters in tiles, not finite", np.dtype(xt).name, rank)
    rng = np.random.default_rng(rank)
    k, n, adapters = 520, 640, 3
    rows = _rows_in_tiles(k, n, rank, xt)
    a = rng.standard_normal((adapters, rank, k)).astype(np.float16)
    b = rng.standard_normal((adapters, n, rank)).astype(np.float16)
    x = (rng.standard_normal((rows, k)) * 10.0 ** rng.integers(-4, 4, (rows, 1))).astype(xt)
    ids = np.arange(rows) // 5 % adapters
    out, d_ids = gpu_ctx.empty((rows, n), np.float32), gpu_ctx.to_device(ids.astype(np.int32))
    gpu_ctx.lora_add(arf_amd.Lora(gpu_ctx.to_device(a), gpu_ctx.to_device(b)), d_ids, gpu_ctx.to_device(x), rows, out)
    want, mags = stepref.lora(x, ids, a, b, None, None)
    assert (np.abs(out.numpy() - want) <= stepref.lora_tolerance(want, mags, None, k, rank)).all()
    a[1, 3, 5], b[2, 7, 1], x[3, 9] = np.nan, np.inf, np.inf  # (row 3 has adapter 0)
    gpu_ctx.lora_add(arf_amd.Lora(gpu_ctx.to_device(a), gpu_ctx.to_device(b)), d_ids, gpu_ctx.to_device(x), rows, out)
    got, rest = out.numpy(), np.arange(n) != 7
    assert np.isfinite(got[(ids == 0) & (np.arange(rows) != 3)]).all() and np.isnan(got[ids == 1]).all() and not np.isfinite(got[3]).any()
    assert np.isfinite(got[ids == 2][:, rest]).all() and not np.isfinite(got[ids == 2][:, 7]).any()


# ---- attention over chosen blocks ----

@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("width", [2047, 2048, 2049, 2300])
def test_choices_where_a_launch_of_their_own_begins(gpu_ctx, dtype, width):
    _say("blocks' border", np.dtype(dtype).name, width)
    rng = np.random.default_rng(width)
    page, heads, dim, group = 16, 2, 64, 2
    batch = Batch(gpu_ctx, [width * page - 3, 1000], [1, 2], page, rng)
    kv = gpu_ctx.kv_cache(heads, dim, page, batch.n_pages)
    hk, hv = _filled(gpu_ctx, kv, batch, rng)
    q, d_bounds = _rows(rng, batch.tokens, heads * group, dim, dtype, False), _bounds(gpu_ctx, kv, batch)
    for kw in (dict(count=64, first=1, last=2), dict(count=1500), dict(count=width - 1, last=3)):
        got, chosen = _attend(gpu_ctx, kv, batch, d_bounds, q, dtype, 0.125, **kw)
        _check(batch, got, chosen, q, hk, hv, 0.125, **kw)
    # the workspace: scores, a place for the choices where wide tables' rows are cut into pieces, and the pieces' parts
    def need(tokens):
        seqs = arf_amd.KVSeqs(gpu_ctx.to_device(np.zeros((1, width), np.int32)), gpu_ctx.to_device(np.zeros(1, np.int32)),
                              gpu_ctx.to_device(np.zeros(2, np.int32)), tokens)
        return gpu_ctx.kv_attention_blocks_workspace(kv, seqs, heads * group, 64)
    assert need(4096) == 4096 * heads * width * 8
    assert need(16) == 16 * heads * (width * 8 + (64 * 4 if width > 2048 else 0) + 4 * 16 * (dim + 4) * 4)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("dim,heads,group", [(64, 1, 4), (128, 2, 4), (256, 2, 20)])
def test_all_blocks_are_attentions_own_result(gpu_ctx, dtype, dim, heads, group):
    # count from the table's width on: kv_attention itself, within what either's roundings allow
    _say("all blocks", np.dtype(dtype).name, dim, heads, group)
    rng = np.random.default_rng(dim)
    batch = Batch(gpu_ctx, [500, 31, 0, 1000, 130], [4, 1, 1, 1, 130], 32, rng)
    kv = gpu_ctx.kv_cache(heads, dim, 32, batch.n_pages)
    hk, hv = _filled(gpu_ctx, kv, batch, rng)
    q = _rows(rng, batch.tokens, heads * group, dim, dtype, False)
    out = gpu_ctx.empty(q.shape, dtype)
    for count, softcap in ((32, 0.0), (100, 20.0)):
        got, chosen = _attend(gpu_ctx, kv, batch, _bounds(gpu_ctx, kv, batch), q, dtype, 0.1, count, softcap=softcap)
        gpu_ctx.kv_attention(kv, batch.seqs, gpu_ctx.to_device(q), out, heads * group, 0.1, softcap=softcap)
        full = out.numpy().astype(np.float64)
        for b, (ln, n) in enumerate(zip(batch.lens, batch.news)):
            r, c = batch.start[b], batch.cached(b)
            if ln == 0:
                assert (got[r:r + n] == 0).all() and (full[r:r + n] == 0).all() and (chosen[r:r + n] == -1).all()
                continue
            want, mag, eps, floor = kvref.attention(q[r:r + n], hk[c], hv[c], 0.1, softcap=softcap)
            tol = kvref.tolerance(want, mag, eps, floor, ln, dtype == np.float16)
            assert (np.abs(got[r:r + n] - full[r:r + n]) <= 2 * tol).all(), b
            seen = (ln - n + np.arange(n)) // 32 + 1
            assert np.array_equal(chosen[r:r + n], np.where(np.arange(count) < seen[:, None], np.arange(count), -1)[:, None].repeat(heads, 1))


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_scores_that_are_nan_or_infinite_beside_pages_that_are_not_the_caches(gpu_ctx, dtype):
    _say("blocks' scores not finite", np.dtype(dtype).name)
    rng = np.random.default_rng(4)
    page, heads, dim, group, count = 16, 2, 128, 4, 6
    batch = Batch(gpu_ctx, [page * 30 + 4, page * 10], [1, 1], page, rng)
    kv = gpu_ctx.kv_cache(heads, dim, page, batch.n_pages)
    rows = int(batch.whole_start[-1])
    k, v = (_rows(rng, rows, heads, dim, np.float32) for _ in "kv")
    k[7 * page + 3, 1, 9] = np.nan  # block 7 of the first sequence's head 1
    gpu_ctx.kv_write(kv, batch.whole, gpu_ctx.to_device(k), gpu_ctx.to_device(v))
    hk, hv = kvref.held_pair(k, v)
    d_bounds = _bounds(gpu_ctx, kv, batch)
    table, absent = batch.table.copy(), [np.zeros(31, bool), np.zeros(10, bool)]
    table[0, [0, 12, 20]] = [-1, batch.n_pages, 2 ** 31 - 1]
    table[1, 2] = -5
    absent[0][[0, 12, 20]] = absent[1][2] = True
    batch.d_table.upload(table)
    q = _rows(rng, 2, heads * group, dim, dtype, False)
    q[0, 1, 5], q[1, 6, 6] = np.nan, np.inf  # of head 0 in the first row, of head 1 in the second
    got, chosen = _attend(gpu_ctx, kv, batch, d_bounds, q, dtype, dim ** -0.5, count=count)
    # NaN scores before all others, the earliest of them; what is not the cache's after them; then the row's own
    assert np.array_equal(chosen[0, 0], [1, 2, 3, 4, 5, 30])
    with np.errstate(invalid="ignore"):
        for t in (0, 1):
            bnd = stepref.bounds(hk[batch.cached(t)], page)
            for h in range(heads):
                mine = slice(h * group, (h + 1) * group)
                blocks = stepref.choose(q[t, mine], bnd[:, h], [31, 10][t], count, 0, 1, absent=absent[t])
                assert np.array_equal(chosen[t, h], blocks), (t, h)
    assert 7 in chosen[0, 1] and np.isnan(got[0, 4:]).all()  # (a key that is NaN: its block comes first, its rows are NaN)
    assert np.isnan(got[0, 1]).all() and np.isfinite(got[0, [0, 2, 3]]).all() and np.isfinite(got[1, :4]).all()
    # the rows without such values, against the oracle
    for t, heads_of in ((0, [0, 2, 3]), (1, [0, 1, 2, 3])):
        c = batch.cached(t)
        keys = (chosen[t, 0][:, None] * page + np.arange(page)).ravel()
        keys = keys[keys < batch.lens[t]]
        want, mag, eps, floor = kvref.attention(q[t:t + 1, heads_of], hk[c][keys, :1], hv[c][keys, :1], dim ** -0.5, absent=absent[t][keys // page])
        tol = kvref.tolerance(want, mag, eps, floor, keys.size, dtype == np.float16)
        assert (np.abs(got[t:t + 1, heads_of] - want) <= tol).all()


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("lens,news,width", [([30000], [1], 0), ([700, 2500], [60, 1], 0), ([193], [1], 0), ([9000], [2], 3000)])
def test_the_same_call_gives_the_same_bits(gpu_ctx, dtype, lens, news, width):
    # whatever the workspace and the outputs held before: keys in pieces, rows of prompts, choices of either kind
    _say("blocks again", np.dtype(dtype).name, lens, news, width)
    rng = np.random.default_rng(lens[0])
    page, heads, dim, group = 16, 2, 128, 4
    batch = Batch(gpu_ctx, lens, news, page, rng)
    if width:
        wide = np.full((len(lens), width), -1, np.int32)
        wide[:, :batch.table.shape[1]] = batch.table
        batch.d_table = gpu_ctx.to_device(wide)
        batch.seqs = arf_amd.KVSeqs(batch.d_table, batch.d_len, batch.d_start, batch.tokens)
        batch.whole = arf_amd.KVSeqs(batch.d_table, batch.d_len, batch.d_whole, int(batch.whole_start[-1]))
    kv = gpu_ctx.kv_cache(heads, dim, page, batch.n_pages)
    _filled(gpu_ctx, kv, batch, rng)
    d_bounds = _bounds(gpu_ctx, kv, batch)
    q = _rows(rng, batch.tokens, heads * group, dim, dtype, False)
    need = gpu_ctx.kv_attention_blocks_workspace(kv, batch.seqs, heads * group, 40)
    dq, shape = gpu_ctx.to_device(q), (batch.tokens, heads, 40)
    first = None
    for fill in (0, 255, 127, 1, 60):
        ws = gpu_ctx.to_device(np.full(need + 16, fill, np.uint8))
        out, chosen = gpu_ctx.to_device(np.full(q.shape, fill, dtype)), gpu_ctx.to_device(np.full(shape, fill, np.int32))
        gpu_ctx.kv_attention_blocks(kv, batch.seqs, d_bounds, dq, out, heads * group, 0.1, 40, first=1, last=2, chosen=chosen, workspace=ws)
        got = out.numpy(), chosen.numpy()
        first = first or got
        assert np.array_equal(got[0], first[0]) and np.array_equal(got[1], first[1])
