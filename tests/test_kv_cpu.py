"""The 4-bit K/V cache without a GPU: the block definition, the kernels' integer arithmetic, and the
refusals that are made before the library or the device is reached."""
import ctypes

import numpy as np
import pytest

import arf_amd
import kvref
from arf_amd import arfq


def test_null_handles_are_rejected():
    L = arf_amd.load_library()
    bad = arfq.ARFQ_E_INVALID
    assert L.arfq_kv_create(None, 8, 128, 64, 4, None) == bad
    assert L.arfq_kv_free(None) == bad
    assert L.arfq_kv_info(None, None, None, None, None, None) == bad
    assert L.arfq_kv_write(None, None, None, None, 0, None, 0, 0) == bad
    assert L.arfq_kv_read(None, None, None, None, 0, None, 0, 0) == bad
    assert L.arfq_kv_attention(None, None, None, 8, None, 0, 0, None, 0, 0, 1.0, 0.0, 0, 1, None, 0) == bad
    assert L.arfq_kv_attention_workspace(None, None, 1, 1, 1, 8, None) == bad


class _Array:
    """A device array's description, without a device."""

    def __init__(self, shape, dtype):
        self.shape, self.dtype, self.ptr = shape, np.dtype(dtype), 4096
        self.nbytes = int(np.prod(shape)) * self.dtype.itemsize


def test_batches_are_checked():
    pages, lens = _Array((3, 5), np.int32), _Array((3,), np.int32)
    assert arf_amd.KVSeqs(pages, lens).tokens == 3
    s = arf_amd.KVSeqs(pages, lens, _Array((4,), np.int32), 7).struct
    assert (s.batch, s.tokens, s.max_pages) == (3, 7, 5)
    for args in [(_Array((3, 5), np.int64), lens), (pages, _Array((4,), np.int32)), (_Array((15,), np.int32), lens),
                 (pages, lens, _Array((3,), np.int32), 7), (pages, lens, _Array((4,), np.int32))]:
        with pytest.raises(ValueError):
            arf_amd.KVSeqs(*args)


def test_struct_matches_the_header():
    # int64, int64, three pointers, int64
    assert ctypes.sizeof(arfq._KVSeqsStruct) == 48
    assert [f[0] for f in arfq._KVSeqsStruct._fields_] == ["batch", "tokens", "start", "len", "pages", "max_pages"]


def test_row_arrays_are_checked():
    a = _Array((4, 8, 128), np.float16)
    assert arfq._row_stride(a, 4, 1024, None, "x") == 1024
    assert arfq._row_stride(a, 2, 1024, 3000, "x") == 3000
    for tokens, stride in [(5, None), (4, 1040), (4, 1000)]:
        with pytest.raises(ValueError):
            arfq._row_stride(a, tokens, 1024, stride, "x")
    with pytest.raises(ValueError):
        arfq._float_type(_Array((4,), np.float64), "x")


@pytest.mark.parametrize("tiles", range(2, 17))
def test_page_of_a_tile_by_reciprocal(tiles):
    # floor(t / tiles) as the high word of t * ceil(2^32 / tiles), for 16-key tiles of 2^29 keys
    magic = ((1 << 32) + tiles - 1) // tiles
    t = np.concatenate([np.arange(1 << 16), np.arange((1 << 25) - 4096, 1 << 25),
                        (np.arange(1, (1 << 25) // tiles, 997) * tiles)[:, None].repeat(2, 1).ravel()
                        - np.tile([0, 1], (((1 << 25) // tiles - 1) + 996) // 997)]).astype(np.uint64)
    assert np.array_equal((t * np.uint64(magic)) >> np.uint64(32), t // np.uint64(tiles))


def test_held_values_are_f16():
    # a scale of 8 significant bits times a code: an f16 exactly, subnormals and the largest among them
    d = np.arange(1, 1 << 15, dtype=np.uint16).view(np.float16).astype(np.float64)
    d = d[np.isfinite(d) & (d <= 8160)]
    m, _ = np.frexp(d)
    normal = np.rint(m * 256) == m * 256
    v = d[normal][:, None] * np.arange(-8, 8)
    assert np.array_equal(v.astype(np.float16).astype(np.float64), v)


@pytest.mark.parametrize("seed", range(4))
def test_held_definition(seed):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((200, 64)) * np.exp2(rng.integers(-30, 16, (200, 1)))).astype(np.float32)
    x[5] = 0
    h, d = kvref.held(x), np.abs(kvref.scales(x))
    # (65280 = 8 * 8160 is the largest value: what lies beyond is held as that)
    off = np.abs(h - np.clip(x.astype(np.float64), -65280, 65280)).reshape(200, 2, 32)
    # half a step, or up to a whole one for values opposite to the largest (codes end at +7),
    # plus the scale's own rounding: 8 codes of 2^-9, or of f16's 2^-25 (and all of x where d is 0)
    assert (off <= 1.0 * d[..., None] + np.abs(d[..., None]) * 8 * 2.0 ** -8 + 8 * 2.0 ** -25).all()
    assert np.array_equal(h[5], np.zeros(64))
    # held again, the values stay, where d is normal: 8 significant bits round s / -8 by less than 2^-8 of it, so s / d
    # is above -8.04 and below -7.96, its code -8, and the held extreme -8 d has the scale d.  (A
    # subnormal d is rounded by up to half of itself, and the extreme's code may be -5.)
    normal = (d >= 2.0 ** -14).repeat(32, -1)
    assert normal.any() and np.array_equal(kvref.held(h)[normal], h[normal])
