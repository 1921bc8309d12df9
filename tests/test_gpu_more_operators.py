"""perf/more_operators.py with the framework's kernels: its results are ordered on torch's current stream, and are
the definition's.  In a process of its own, where torch comes first (it finds no GPU where another HIP runtime than
its own is in use)."""
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
    spec = importlib.util.spec_from_file_location("perf_more_operators", os.path.join(ROOT, "perf", "more_operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.own = True
    for case in m.listed():
        if case["name"] not in ("plan decode", "adapt decode", "rotate image", "blocks batch"):
            continue
        print("case:", case["name"], flush=True)
        s = m.prepare(case, 3)
        want, got = m.exact(case, 3), m.run(s)
        if not isinstance(got, dict):
            got, want = {"out": got}, {"out": want}
        got = {k: v.clone() for k, v in got.items()}  # (nothing waits in between)
        for name, v in got.items():
            if v.dtype in (torch.int32, torch.int64) or name == "bounds":
                assert torch.equal(v.double(), want[name].double()), name
                continue
            # norms over values of both signs: f16 roundings of 2^-11 at most, and f32's of sums of a few thousand terms
            off = float((v.double() - want[name]).norm() / want[name].norm())
            assert off < (2.0 ** -11 if v.dtype == torch.float16 else 2.4e-5), (name, off)
    torch.cuda.synchronize()


if __name__ == "__main__":
    main()
