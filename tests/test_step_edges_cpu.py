"""What the tests of a serving step's operators would let pass, found on the CPU: the oracle with a mistake planted."""
import numpy as np
import pytest

import stepref

# of test_gpu_step_edges.py: the shapes of adapters in tiles
SHAPES = [(64, 2500), (2056, 2050), (5120, 321), (264, 1172)]
RANKS = [8, 16, 24, 40, 64, 72, 128, 136, 256]


@pytest.mark.parametrize("k,n", SHAPES)
@pytest.mark.parametrize("rank", RANKS)
def test_adapters_in_fewer_bits_are_noticed(rank, k, n):
    # x in one f16, and h in one f16 part, pass the bound on the norm of the errors; sums in 32 bits do not
    rng = np.random.default_rng(rank + k)
    rows = 40
    a = (rng.standard_normal((1, rank, k)) / np.sqrt(k)).astype(np.float16)
    b = rng.standard_normal((1, n, rank)).astype(np.float16)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    base = rng.standard_normal((rows, n)).astype(np.float32)
    want, _ = stepref.lora(x, np.zeros(rows, int), a, b, None, base)
    most = stepref.lora_norm_tolerance(want, base, k, rank)
    off = lambda got: np.linalg.norm(got - want)
    a32, b32 = a[0].astype(np.float32), b[0].astype(np.float32)
    assert off(base + (x @ a32.T) @ b32.T) <= most
    wide = lambda x: x.astype(np.float64)
    fewer = wide(x.astype(np.float16)) @ wide(a[0]).T @ wide(b[0]).T + base
    assert off(fewer) > 3 * most
    h = wide(x) @ wide(a[0]).T
    assert off(wide(h.astype(np.float16)) @ wide(b[0]).T + base) > 3 * most
