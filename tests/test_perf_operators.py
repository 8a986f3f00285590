"""The library's calls as perf/operators.py makes them."""
import importlib.util
import os

import pytest

from conftest import REPO

gpu = pytest.mark.gpu


def load():
    spec = importlib.util.spec_from_file_location("perf_operators", os.path.join(REPO, "perf", "operators.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.own = True
    return module


def tensors(out):
    return [t.clone() for t in (out.values() if isinstance(out, dict) else [out])]


@gpu
@pytest.mark.parametrize("kind", ["shared", "tables", "qk_norm", "logits"])
def test_a_state_runs_on_the_current_stream(torch_mod, dev, kind):
    """Run once on the default stream, then on another and captured there: the graph holds the call."""
    torch = torch_mod
    ops = load()
    case = next(c for c in ops.listed() if c["kind"] == kind)
    state = ops.prepare(case, 3)
    first = tensors(ops.run(state))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for t in ops.run(state).values() if kind != "shared" else [ops.run(state)]:
            t.record_stream(stream)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = ops.run(state)
    written = [out] if kind == "shared" else [out["q"]] if kind == "qk_norm" else [out["out"], out["next"]] if kind == "logits" else [out["pos"], out["slot"]]
    for _ in range(3):
        for t in written:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, tensors(out)))
