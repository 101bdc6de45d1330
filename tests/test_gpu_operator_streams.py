"""perf/operators.py calls the library on the caller's current stream: a replayed capture of one pass does all its work,
and a pass is ordered behind what stands on the stream before it."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CASES = {
    "select": dict(dtype="bf16", groups=2, beams=3, out=4, vocab=5000, pad=0, softcap=30.0, temperature=1.0, alpha=0.6,
                   masked=0.0, done=0),
    "reorder": dict(dtype="bf16", groups=2, beams=3, layers=2, heads=2, max_len=40, live=33, dim=16),
    "fork": dict(dtype="bf16", groups=2, beams=3, pools=2, segs=1, page_tokens=8, width=30, pages=200, prompt_lo=40,
                 prompt_hi=90, grown=21, new=1),
    "compact": dict(dtype="bf16", seqs=3, pools=2, page_tokens=8, width=30, pages=128, length=60, used=0.5),
}


@pytest.fixture(scope="module")
def ops(g4, torch_cuda):
    spec = importlib.util.spec_from_file_location("perf_operators", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    at = os.getcwd()
    os.chdir(ROOT)
    m.own = True
    yield m
    os.chdir(at)


def outputs(torch, ops, state):
    return {k: v.clone() for k, v in ops.run(state).items() if k != "moves"}


@pytest.mark.parametrize("op", CASES)
def test_a_pass_belongs_to_the_current_stream(ops, torch_cuda, op):
    torch = torch_cuda
    case = {"op": op, "name": op, **CASES[op]}
    state = ops.prepare(case, 1)
    torch.cuda.synchronize()
    ops.run(state)  # (the context and its buffers)
    torch.cuda.synchronize()

    # each pass from fresh inputs; `clear` stands for what a program did on the stream before
    def fresh():
        s = ops.prepare(case, 2)
        for v in s["out"].values():
            v.zero_()
        torch.cuda.synchronize()
        return s

    s = fresh()
    want = outputs(torch, ops, s)
    torch.cuda.synchronize()

    s = fresh()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ops.run(s)
    torch.cuda.synchronize()
    assert all(not v.any() for v in s["out"].values())  # a capture runs nothing
    graph.replay()
    torch.cuda.synchronize()
    got = {k: v for k, v in {**s["out"], **({"pools": s["pools"]} if "pools" in s else {})}.items() if k != "moves"}
    assert all(torch.equal(got[k], want[k]) for k in want)

    # behind work of the current stream that takes longer than the call
    for on in (None, torch.cuda.Stream()):
        s = fresh()
        with torch.cuda.stream(on):
            torch.cuda._sleep(20_000_000)
            for v in s["out"].values():
                v.fill_(7)
            got = outputs(torch, ops, s)
        torch.cuda.synchronize()
        for k in want:
            keep = want[k] != 0 if k in ("table", "kv", "hist") else torch.ones_like(want[k], dtype=torch.bool)
            assert torch.equal(got[k][keep], want[k][keep]), (op, k)
