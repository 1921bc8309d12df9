"""perf/operators.py with the framework's kernels: its results are ordered on torch's current stream, and
are the definition's."""
import importlib.util
import os

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))

pytestmark = pytest.mark.gpu


@pytest.fixture()
def operators():
    torch = pytest.importorskip("torch")
    before = torch.cuda.current_stream()
    spec = importlib.util.spec_from_file_location("perf_operators", os.path.join(HERE, "..", "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.own = True
    yield m
    torch.cuda.synchronize()
    m.context().close()
    torch.cuda.set_stream(before)


def test_results_follow_on_torchs_stream(operators):
    import torch

    import arf_amd
    cases = {c["name"]: c for c in operators.listed()}
    for name in ("decode batch", "write decode"):
        s = operators.prepare(cases[name], 3)
        assert arf_amd.load_library().arfq_ctx_stream(operators.context().handle) == torch.cuda.current_stream().cuda_stream
        want = operators.exact(cases[name], 3)
        got = operators.run(s)
        if isinstance(got, dict):
            got = {k: v.clone() for k, v in got.items()}  # (nothing waits in between)
            assert all(torch.equal(got[k].double(), want[k]) for k in got)
        else:
            got = got.clone()
            # f32 sums of the operators' listed cases, 1e-6 of the values' size and below
            assert float((got.double() - want).norm() / want.norm()) < 2e-6
