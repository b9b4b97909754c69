"""perf/operators.py: its passes run on the stream that is current, on every pass anew."""
import importlib.util
import os

import pytest

import nemotron_hip as NH

torch = pytest.importorskip("torch")

PATH = os.path.join(os.path.dirname(__file__), "..", "perf", "operators.py")
SMALL = [{"op": "quant", "rows": 3, "cols": 70, "x": "bf16"},
         {"op": "linear", "m": 20, "k": 100, "n": 40, "x": "f32", "out": "bf16", "bias": True},
         {"op": "moe", "tokens": 5, "hidden": 64, "inter": 40, "experts": 4, "top_k": 2, "x": "f32"},
         {"op": "balance", "tokens": 9, "experts": 8, "top_k": 2, "sequences": 2, "pad": 1, "softmax": True}]


@pytest.fixture
def operators():
    spec = importlib.util.spec_from_file_location("operators_under_test", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.own = True
    return module


class Library:
    """Notes the stream of each call in place of making it; sizes are the library's."""

    def __init__(self):
        self.streams = []

    def __getattr__(self, name):
        real = getattr(NH.lib(), name)
        if name.endswith("_size"):
            return real

        def note(*args):
            assert len(args) == len(real.argtypes)
            self.streams.append(args[-2].value if isinstance(args[-2], NH.C.c_void_p) else args[-2])
            return NH.OK
        note.argtypes = real.argtypes
        return note


@pytest.mark.parametrize("case", SMALL, ids=lambda c: c["op"])
def test_a_pass_goes_to_the_current_stream(operators, monkeypatch, case):
    class Binding:
        F32, BF16, NhError, check = NH.F32, NH.BF16, NH.NhError, staticmethod(NH.check)
        library = Library()

        @classmethod
        def lib(cls):
            return cls.library

    class Program:
        handle, stream = NH.P(), 0

    empty = torch.empty
    monkeypatch.setattr(operators, "_library", (Binding, Program))
    monkeypatch.setattr(torch, "empty", lambda shape, dtype, device=None: empty(shape, dtype=dtype))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: Program.stream, raising=False)
    t = torch.zeros(8)
    state = {"case": case, **{v: t for v in ("x", "logits", "indices", "offsets", "dloss", "bias", "tiled", "tiled_up",
                                             "tiled_down", "codes", "scales")}}
    state["indices"] = torch.zeros((case.get("tokens", 1), 2), dtype=torch.int32)
    calls = 0
    for handle in (0x1000, 0x2000, 0x1000):
        Program.stream = handle
        operators.run(state)
        seen = Binding.library.streams[calls:]
        assert seen and all(s == handle for s in seen)
        calls += len(seen)


@pytest.mark.gpu
@pytest.mark.parametrize("case", SMALL, ids=lambda c: c["op"])
def test_a_state_that_has_run_is_captured_and_replayed(operators, case):
    """First eagerly, then under a capture: replays over other inputs give what an eager pass gives on them."""
    print(f"[gpu-case] pass in a graph: {case}", flush=True)
    states = [operators.prepare(case, seed) for seed in range(3)]
    flat = lambda out: [v.clone() for v in (out.values() if isinstance(out, dict) else [out])]  # noqa: E731
    want = [flat(operators.run(s)) for s in states]
    state = states[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = operators.run(state)
    inputs = [v for v in ("x", "logits", "indices", "offsets", "dloss", "bias", "tiled", "tiled_up", "tiled_down")
              if isinstance(state.get(v), torch.Tensor)]
    for turn in (1, 2, 1):
        for v in inputs:
            state[v].copy_(states[turn][v])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(flat(out), want[turn])), turn
        states[1]["again"] = operators.run(states[1])  # the program's own work between the replays
