"""perf/operators.py with the framework's kernels: its results are ordered on torch's current stream, and
are the definition's.  In a process of its own, where torch comes first (it finds no GPU where another
HIP runtime than its own is in use)."""
import importlib.util
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)

pytestmark = pytest.mark.gpu


def test_results_follow_on_torchs_stream():
    r = subprocess.run([sys.executable, "-u", os.path.abspath(__file__)], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]


def main():
    import torch
    torch.cuda.init()
    sys.path.insert(0, ROOT)
    import arf_amd
    spec = importlib.util.spec_from_file_location("perf_operators", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.own = True
    cases = {c["name"]: c for c in m.listed()}
    for name in ("decode batch", "write decode"):
        print("case:", name, flush=True)
        s = m.prepare(cases[name], 3)
        assert arf_amd.load_library().arfq_ctx_stream(m.context().handle) == torch.cuda.current_stream().cuda_stream
        want = m.exact(cases[name], 3)
        got = m.run(s)
        if isinstance(got, dict):
            got = {k: v.clone() for k, v in got.items()}  # (nothing waits in between)
            assert all(torch.equal(got[k].double(), want[k]) for k in got)
        else:
            got = got.clone()
            # a score's terms are 10 in all (128 products of about 0.8, over 128 ** 0.5), rounded (128 / 32 + 16) times
            # by 2^-24: 1.2e-5; its p is off by as much, and the divisor
            off = float((got.double() - want).norm() / want.norm())
            assert off < 2.4e-5, off
    torch.cuda.synchronize()


if __name__ == "__main__":
    main()
