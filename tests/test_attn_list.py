"""The attention's work list on the CPU: tests/attn_list_driver.cpp compiles the kernels' own search
(arf_amd/csrc/arfq_attn_list.h) over a wave of coroutines (tests/host_wave) and takes every workgroup's item of
a call.  Whatever the batch holds, every (row, piece) of a sequence that has rows is some workgroup's, no row is
two sequences', and every entry that the join reads was written and names rows of the call."""
import os
import shutil
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CXX = shutil.which("clang++") or shutil.which("amdclang++") or "/opt/rocm/llvm/bin/clang++"


@pytest.fixture(scope="module")
def driver(tmp_path_factory):
    if not os.path.exists(CXX):
        pytest.skip("no clang++")
    exe = str(tmp_path_factory.mktemp("list") / "attn_list_drv")
    cmd = [CXX, "-std=c++17", "-O2", "-Wno-unused-function", "-I", os.path.join(HERE, "host_wave"),
           "-I", os.path.join(ROOT, "arf_amd", "csrc"), "-I", os.path.join(ROOT, "include"),
           os.path.join(HERE, "attn_list_driver.cpp"), "-o", exe]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]

    def run(calls):
        text = "\n".join(" ".join(map(str, c)) for c in calls) + "\n"
        r = subprocess.run([exe], input=text, capture_output=True, text=True, timeout=600)
        assert r.returncode == 0, r.stderr[-2000:]
        lines = r.stdout.splitlines()
        assert len(lines) == 3 * len(calls)
        return [([int(x) for x in lines[3 * i].split()], [int(x) for x in lines[3 * i + 1].split()],
                 int(lines[3 * i + 2].split(":")[1])) for i in range(len(calls))]

    return run


def _call(start, lens, tokens, heads=8, q_heads=32, dim=128, page=64, max_pages=2048, window=0, causal=1, cus=256):
    return [cus, heads, dim, q_heads, page, max_pages, window, causal, tokens, len(lens), int(start is not None),
            *(start or []), *lens]


def _check(got):
    for i, (few, many, left) in enumerate(got):
        for tr, slots, cut, items, joins, bad in (few, many):
            assert bad == 0, (i, tr, bad)
            assert items <= slots and joins <= cut, (i, tr)
        assert left == 0, (i, left)


def test_starts_that_decrease(driver):
    # sequences whose rows would overlap are more items than the call has workgroups: from the first decrease on
    # no sequence has rows
    for n in (65, 399):
        got = driver([_call(([0, 16] * n)[:n + 1], [100] * (n - 1) + [131072], 16)])
        _check(got)
        assert got[0][0][3] == 4  # the first sequence's 64 rows
    lens = [5000, 131072, 300] + [100] * 150
    for start in ([0, 3, 16] + [0, 16] * 76, [16] + [0, 16] * 77, [0] * 70 + [16, 0] * 42, [-4, 16] * 77,
                  [0, 2 ** 31 - 1, -2 ** 31] + [0, 16] * 76, list(range(154, 0, -1)), [0, 8] * 32 + [8, 16] * 45):
        _check(driver([_call(start[:154], lens, 16), _call(start[:154], lens, 16, heads=1, q_heads=7),
                       _call(start[:154], lens[::-1], 16, window=1000)]))


def test_prompts_whose_starts_decrease(driver):
    # 128-row tiles, among them those of a long sequence, and short rows behind
    for start in ([0, 400] * 40, [0, 300, 400] + [0, 400] * 39, [0, 100, 99] + [0, 390, 400] * 26):
        lens = [9000, 400, 131072] + [500] * (len(start) - 4)
        _check(driver([_call(start, lens, 400, heads=2, q_heads=8, causal=c) for c in (0, 1)]))


@pytest.mark.parametrize("seed", range(3))
def test_any_batch(driver, seed):
    # sequences of any lengths, as the contract has them; and the same with a few entries of start spoilt
    rng = np.random.default_rng(seed)
    calls = []
    for _ in range(8):
        batch = int(np.exp(rng.uniform(0, np.log(300))))
        heads = int(rng.choice([1, 2, 8, 64]))
        q_heads = heads * int(rng.choice([1, 3, 4, 17, 70]))
        news = rng.integers(0, int(rng.choice([2, 6, 90, 700])), batch)
        news[rng.random(batch) < 0.3] = 1
        if news.sum() * q_heads > 40000:
            news = np.minimum(news, 1)
        lens = np.exp(rng.uniform(0, np.log(rng.choice([50, 600, 10000, 131072])), batch)).astype(int)
        lens[rng.random(batch) < 0.1] = rng.choice([0, -1, 2 ** 31 - 1, 131072])
        start = np.concatenate([[0], np.cumsum(news)])
        tokens = max(1, int(start[-1]))
        kw = dict(heads=heads, q_heads=q_heads, dim=int(rng.choice([64, 96, 128, 256])), max_pages=int(rng.choice([1, 5, 2048])),
                  window=int(rng.choice([0, 0, 1, 3000])), causal=int(rng.integers(0, 2)))
        calls.append(_call(start.tolist(), lens.tolist(), tokens, **kw))
        calls.append(_call(None, lens.tolist(), batch - int(rng.integers(0, batch)), **kw))
        start[rng.integers(0, batch + 1, 3)] = rng.integers(-2, tokens + 2, 3)
        calls.append(_call(start.tolist(), lens.tolist(), tokens, **kw))
    _check(driver(calls))
