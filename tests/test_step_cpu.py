"""What of a serving step's operators needs no GPU: null handles, the binding's checks, and stepref against cases worked out
by hand."""
import numpy as np
import pytest

import arf_amd
import stepref
from arf_amd import arfq


class Fake:
    """A device array as far as the binding's checks look."""

    def __init__(self, shape, dtype):
        self.shape, self.dtype, self.ptr = tuple(shape), np.dtype(dtype), 4096
        self.nbytes = int(np.prod(self.shape)) * self.dtype.itemsize


def test_null_handles_are_rejected():
    L = arf_amd.load_library()
    bad = arfq.ARFQ_E_INVALID
    assert L.arfq_kv_plan(None, None) == bad
    assert L.arfq_rope(None, None, None, 0, 0, 1, 64, None, 64, 0, None, 64, 0, 0) == bad
    assert L.arfq_kv_bounds(None, None, None, None) == bad
    assert L.arfq_kv_attention_blocks(None, None, None, None, 1, None, 64, 0, None, 64, 0, 1.0, 0.0, 1, 0, 1, None, None, 0) == bad
    assert L.arfq_kv_attention_blocks_workspace(None, None, 1, 1, 1, 1, 1, None) == bad
    assert L.arfq_lora_add(None, None, None, 0, None, 0, None, 0, None, 0, None, 0) == bad
    assert L.arfq_lora_workspace(None, None, 0, None) == bad


def _step(**kw):
    i32 = lambda *s: Fake(s, np.int32)
    a = dict(page_size=16, add=i32(2), held=i32(2), held_next=i32(2), pages=i32(2, 4), free=i32(8), n_free=i32(1), n_free_next=i32(1),
             start=i32(3), lens=i32(2), taken=i32(3), freed=i32(3), positions=i32(5), slots=Fake((5,), np.int64))
    a.update(kw)
    return arf_amd.KVStep(**a)


@pytest.mark.parametrize("name,shape,dtype", [("add", (3,), np.int32), ("held", (2,), np.int64), ("pages", (8,), np.int32), ("free", (2, 4), np.int32),
                                              ("start", (2,), np.int32), ("slots", (5,), np.int32), ("slots", (4,), np.int64), ("n_free", (2,), np.int32)])
def test_a_steps_arrays(name, shape, dtype):
    assert _step().seqs.tokens == 5
    with pytest.raises(ValueError):
        _step(**{name: Fake(shape, dtype)})


def test_rope_sections():
    r = arf_amd.Rope.sections([3, 2, 1], 10.0, "cycle")
    assert r._axes.tolist() == [0, 1, 2, 0, 1, 0] and r.rot_dim == 12 and r.axes == 3
    assert np.allclose(r._freqs, 10.0 ** (-np.arange(6) / 6))
    r = arf_amd.Rope.sections([2, 4], 10.0, "own", "neighbours")
    assert r._axes.tolist() == [0, 0, 1, 1, 1, 1] and np.allclose(r._freqs, 10.0 ** -np.array([0, 0.5, 0, 0.25, 0.5, 0.75]))
    assert arf_amd.Rope.sections([4, 4])._axes.tolist() == [0] * 4 + [1] * 4 and arf_amd.Rope([1.0] * 4).axes == 1
    for bad in (lambda: arf_amd.Rope.sections([]), lambda: arf_amd.Rope.sections([-1, 5]), lambda: arf_amd.Rope.sections([4], layout="x"),
                lambda: arf_amd.Rope([1.0], pairs="x"), lambda: arf_amd.Rope([1.0, 2.0], [0])):
        with pytest.raises(ValueError):
            bad()


def test_adapters_shapes():
    a, b = Fake((2, 8, 16), np.float16), Fake((2, 5, 8), np.float16)
    l = arf_amd.Lora(a, b)
    assert (l.adapters, l.rank, l.k, l.n) == (2, 8, 16, 5)
    for bad in ((a, a), (Fake((2, 8, 16), np.float32), b), (a, Fake((3, 5, 8), np.float16)), (a, b, Fake((3,), np.float32)), (a, b, Fake((2,), np.float16))):
        with pytest.raises(ValueError):
            arf_amd.Lora(*bad)


def test_the_reference_of_a_plan():
    # pages of 4; the first gives two back (12, 13), the second takes them and one from the stack, the third finds none,
    # the fourth wants none, the fifth gets nothing either (not overtaken)
    pages = np.array([[11, 12, 13], [21, -1, -1], [31, -1, -1], [41, -1, -1], [-1, -1, -1]], np.int32)
    got = stepref.plan(4, [-6, 7, 5, 1, 1], [10, 4, 4, 2, 0], pages, np.array([7, 8, 9, 0, 0, 0], np.int32), 1, 14)
    assert got["pages"].tolist() == [[11, 12, 13], [21, 12, 13], [31, -1, -1], [41, -1, -1], [-1, -1, -1]]
    assert got["held_next"] == [4, 11, 4, 3, 0] and got["lens"] == [4, 11, 0, 3, 0]
    assert got["taken"] == [0, 0, 2, 2, 2, 2] and got["freed"] == [0, 2, 2, 2, 2, 2] and got["n_free_next"] == [1]
    assert got["start"].tolist() == [0, 0, 7, 12, 13, 14]
    assert got["positions"].tolist() == [4, 5, 6, 7, 8, 9, 10] + [-1] * 5 + [2, -1]
    assert got["slots"].tolist() == [48, 49, 50, 51, 52, 53, 54] + [-1] * 5 + [166, -1]


def test_the_reference_of_chosen_blocks():
    # one channel: bounds [hi, lo] of five blocks; q = 2 goes by hi, q = -1 by lo
    bnd = np.array([[5, 1], [3, -4], [9, 9], [3, -9], [0, 0]], float)[:, :, None]
    q = lambda *v: np.array(v, float)[:, None]
    assert stepref.choose(q(2), bnd, 5, 2, 0, 1).tolist() == [2, 4]
    assert stepref.choose(q(-1), bnd, 5, 3, 0, 1).tolist() == [1, 3, 4]
    assert stepref.choose(q(2, -1), bnd, 5, 3, 1, 1).tolist() == [0, 2, 4]
    assert stepref.choose(q(2), bnd, 5, 3, 0, 1, negative=True).tolist() == [1, 3, 4]
    assert stepref.choose(q(0), bnd, 5, 3, 0, 1).tolist() == [0, 1, 4]
    assert stepref.choose(q(2), bnd, 3, 3, 0, 1).tolist() == [0, 1, 2]
