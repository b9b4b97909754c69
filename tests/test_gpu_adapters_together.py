"""The rows by expert, the experts' low-rank adapters and the projection beside them, as a training step and a server run
them: in a chain, captured, on two streams, and on the stream that is current."""
import importlib.util
import os

import numpy as np
import pytest

import adapters_reference as A
import nemotron_hip as NH
from test_gpu_mxfp4 import Guarded, note
from test_operator_passes import Library

DT = {"f32": NH.F32, "bf16": NH.BF16}
NP = {"f32": np.float32, "bf16": np.uint16}


@pytest.fixture(scope="module")
def ctx():
    c = NH.Context(0)
    yield c
    c.close()


class Experts:
    """out_t = shared_t + sum_j w_tj E_e(x_t), E_e = low-rank products of expert e: routes sorted, rows dispatched, the
    experts' matrices as adapters whose ids are the slots' experts, joined; then every gradient."""

    def __init__(self, ctx, t, k, e, h, n, rank, dtype, stream=None, seed=0):
        self.ctx, self.sizes, self.dtype, self.stream = ctx, (t, k, e, h, n, rank), dtype, stream
        slots = t * k
        up = ctx.upload
        self.x, self.dout, self.shared = ctx.empty((t, h), NP[dtype]), ctx.empty((t, n), NP[dtype]), ctx.empty((t, n), NP[dtype])
        self.ids, self.w = ctx.empty((t, k), np.int32), ctx.empty((t, k), np.float32)
        self.slot_ids = ctx.empty(slots, np.int32)
        self.a, self.b = ctx.empty((e, rank, h), NP[dtype]), ctx.empty((e, n, rank), NP[dtype])
        self.outs = {name: Guarded(ctx, shape, d) for name, shape, d in (
            ("offsets", (e + 1,), np.int32), ("perm", (slots,), np.int32), ("pos", (t, k), np.int32),
            ("rows", (slots, h), NP[dtype]), ("h", (slots, rank), np.float32), ("y", (slots, n), NP[dtype]),
            ("out", (t, n), NP[dtype]), ("dy", (slots, n), NP[dtype]), ("dw", (t, k), np.float32),
            ("drows", (slots, h), NP[dtype]), ("da", (e, rank, h), np.float32), ("db", (e, n, rank), np.float32),
            ("dx", (t, h), NP[dtype]))}
        lib, s = NH.lib(), (slots, n, h, rank, e)
        self.ws = [up(np.full(f(*s), 0xFF, np.uint8)) for f in
                   (lib.nh_linear_lora_workspace_size, lib.nh_linear_lora_backward_workspace_size)]
        self.renew(seed)

    def renew(self, seed):
        t, k, e, h, n, rank = self.sizes
        rng = np.random.default_rng(seed)
        self.v = {}
        for name, shape, std in (("x", (t, h), 1.0), ("dout", (t, n), 1.0), ("shared", (t, n), 1.0), ("a", (e, rank, h), h ** -0.5),
                                 ("b", (e, n, rank), 1.0)):
            stored, self.v[name] = A.held(rng.standard_normal(shape) * std, self.dtype)
            getattr(self, name).copy_from(stored)
        ids = np.argsort(rng.random((t, e)), axis=1)[:, :k].astype(np.int32)
        w = rng.uniform(0.1, 1, (t, k)).astype(np.float32)
        self.ids.copy_from(ids)
        self.w.copy_from(w)
        self.v["ids"], self.v["w"] = ids, w.astype(np.float64)
        self.slot_ids.copy_from(np.sort(ids.reshape(-1), kind="stable"))  # every route is placed: the slots' experts

    def issue(self):
        t, k, e, h, n, rank = self.sizes
        d, slots, hd, s = DT[self.dtype], t * k, self.ctx.handle, self.stream
        o = {name: v.ptr for name, v in self.outs.items()}
        lora = (slots, n, h, rank, e)
        mats = (self.slot_ids.ptr, self.a.ptr, self.b.ptr, d, None)
        NH.call("nh_moe_permute", hd, self.ids.ptr, t, k, e, o["offsets"], o["perm"], o["pos"], s)
        NH.call("nh_moe_dispatch", hd, self.x.ptr, d, o["pos"], None, t, k, h, slots, o["rows"], d, s)
        NH.call("nh_linear_lora", hd, o["rows"], d, *mats, *lora, None, o["y"], d, o["h"], self.ws[0].ptr, self.ws[0].nbytes, s)
        NH.call("nh_moe_combine_rows", hd, o["y"], d, o["pos"], self.w.ptr, self.shared.ptr, t, k, n, slots, o["out"], d, s)
        NH.call("nh_moe_combine_rows_backward", hd, self.dout.ptr, d, o["y"], d, o["pos"], self.w.ptr, t, k, n, slots, o["dy"],
                o["dw"], s)
        NH.call("nh_linear_lora_backward", hd, o["rows"], d, *mats, o["h"], o["dy"], d, *lora, None, o["drows"], o["da"],
                o["db"], 0, self.ws[1].ptr, self.ws[1].nbytes, s)
        NH.call("nh_moe_dispatch_backward", hd, o["drows"], d, None, d, o["pos"], None, t, k, h, slots, o["dx"], None, s)

    def plain(self, v=None, absolute=False):
        """The layer in 64 bits, from its definition; with absolute, of the operands' absolute values, which bounds
        every sum of absolute terms on the way."""
        v = dict(v or self.v)
        if absolute:
            v = {n: a if n == "ids" else np.abs(a) for n, a in v.items()}
        r = {"out": v["shared"].copy(), "dw": np.zeros_like(v["w"]), "dx": np.zeros_like(v["x"]), "da": np.zeros_like(v["a"]),
             "db": np.zeros_like(v["b"])}
        for i in range(len(v["x"])):
            for j, e in enumerate(v["ids"][i]):
                a, b, w = v["a"][e], v["b"][e], v["w"][i, j]
                h = a @ v["x"][i]
                y = b @ h
                r["out"][i] += w * y
                r["dw"][i, j] = y @ v["dout"][i]
                dh = b.T @ (w * v["dout"][i])
                r["dx"][i] += a.T @ dh
                r["da"][e] += np.outer(dh, v["x"][i])
                r["db"][e] += np.outer(w * v["dout"][i], h)
        return r

    def check(self):
        """Along any path at most five values are stored on the way (rows, y, dy, drows, the result), each off by half a
        step, and at most two low-rank values cut to bf16 (2^-15), where the type is bf16; every sum has at most `longest`
        terms of three parts each, at most four sums in a path."""
        t, k, e, h, n, rank = self.sizes
        self.ctx.synchronize(self.stream)
        got = {name: o.numpy() for name, o in self.outs.items()}
        flat = self.v["ids"].reshape(-1)
        order = np.argsort(flat, kind="stable")
        assert np.array_equal(got["perm"], order) and np.array_equal(np.argsort(order), got["pos"].reshape(-1))
        assert np.array_equal(got["offsets"], np.concatenate([[0], np.cumsum(np.bincount(flat, minlength=e))]))
        longest = max(t * k, h, n, rank)
        off = 5 * A.HALF[self.dtype] + (2 * 2.0 ** -15 if self.dtype == "bf16" else 0) + 4 * (3 * longest + 40) * A.U
        want, size = self.plain(), self.plain(absolute=True)
        for name in want:
            assert (np.abs(A.values(got[name]) - want[name]) <= 1.05 * off * size[name] + 1e-40).all(), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("t,k,e,h,n,rank", [(1, 2, 4, 64, 40, 8), (9, 3, 8, 70, 33, 5), (50, 4, 6, 130, 96, 16), (120, 6, 20, 96, 65, 33)])
def test_experts_forward_and_backward(ctx, t, k, e, h, n, rank, dtype):
    note(f"experts together t={t} k={k} e={e} h={h} n={n} rank={rank} {dtype}")
    c = Experts(ctx, t, k, e, h, n, rank, dtype)
    c.issue()
    c.check()


@pytest.mark.parametrize("name", ["x", "a", "b", "w", "shared"])
def test_the_plain_gradients_are_differences(name):
    """Of the loss <out, dout>, which is linear in each operand alone: one difference is exact but for rounding."""
    c = object.__new__(Experts)
    rng = np.random.default_rng(1)
    c.v = {"x": rng.standard_normal((5, 7)), "dout": rng.standard_normal((5, 6)), "shared": rng.standard_normal((5, 6)),
           "a": rng.standard_normal((4, 3, 7)), "b": rng.standard_normal((4, 6, 3)), "w": rng.uniform(0.1, 1, (5, 2)),
           "ids": np.argsort(rng.random((5, 4)), axis=1)[:, :2]}
    g = {"x": "dx", "a": "da", "b": "db", "w": "dw"}
    d = rng.standard_normal(c.v[name].shape)
    want = np.sum(d * (c.plain()[g[name]] if name in g else c.v["dout"]))
    loss = lambda s: np.sum(c.plain({**c.v, name: c.v[name] + s * d})["out"] * c.v["dout"])  # noqa: E731
    size = np.sum(np.abs(c.plain(absolute=True)["out"] * c.v["dout"]))
    assert abs((loss(1) - loss(-1)) / 2 - want) <= 1e-12 * (size + abs(want)) * 10


@pytest.mark.gpu
def test_experts_on_two_streams_and_replayed(ctx):
    """Two layers in flight, each captured; other routes, rows and matrices between the replays, and eager work."""
    note("experts together on two streams, captured")
    graphs, runs = NH.HipGraphs(), []
    for seed in (1, 2):
        stream = NH.P()
        NH.call("nh_stream_create", ctx.handle, NH.C.byref(stream))
        runs.append(Experts(ctx, 60, 4, 12, 96, 80, 16, "bf16", stream, seed))
    for c in runs:
        c.issue()
        c.check()
        c.graph = graphs.capture(c.stream, c.issue)
    for turn in range(4):
        for c in runs:
            c.renew(10 * turn + 100)
        for _ in range(2):
            for c in runs if turn % 2 else runs[::-1]:
                graphs.launch(c.graph[1], c.stream)
        for c in runs:
            c.check()
        runs[turn % 2].issue()  # the program's own work between the replays
        runs[turn % 2].check()
    for c in runs:
        graphs.destroy(*c.graph)
        NH.call("nh_stream_destroy", ctx.handle, c.stream)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 20, 200])
def test_beside_a_quantized_layer(ctx, m):
    """The projection in int8, then its requests' adapters onto its output where it stands; the same result as on a copy
    of it, and in rows without an adapter the projection's bits."""
    note(f"quantized layer with adapters m={m}")
    n, k, rank, adapters = 160, 256, 16, 5
    rng = np.random.default_rng(m)
    xs, x = A.held(rng.standard_normal((m, k)), "bf16")
    codes = rng.integers(-127, 128, (n, k)).astype(np.int8)
    ids = rng.integers(-1, adapters, m).astype(np.int32)
    as_, a = A.held(rng.standard_normal((adapters, rank, k)) / 16, "bf16")
    bs, b = A.held(rng.standard_normal((adapters, n, rank)), "bf16")
    s = rng.uniform(0.5, 2, adapters).astype(np.float32)
    dx, raw, sw, di, da, db, ds = [ctx.upload(v) for v in (xs, codes, np.full(n, 1e-3, np.float32), ids, as_, bs, s)]
    tiled = NH.tile_weights(ctx, raw, n, k)
    out = Guarded(ctx, (m, n), np.uint16)
    lib = NH.lib()
    ws = ctx.empty(max(lib.nh_linear_w8a8_workspace_size(m, k), lib.nh_linear_lora_workspace_size(m, n, k, rank, adapters)), np.uint8)
    NH.call("nh_linear_w8a8", ctx.handle, dx.ptr, NH.BF16, tiled.ptr, sw.ptr, None, m, n, k, out.ptr, NH.BF16, ws.ptr, ws.nbytes,
            None, None, None, None)
    base = out.numpy().copy()
    args = (dx.ptr, NH.BF16, di.ptr, da.ptr, db.ptr, NH.BF16, ds.ptr, m, n, k, rank, adapters)
    NH.call("nh_linear_lora", ctx.handle, *args, out.ptr, out.ptr, NH.BF16, None, ws.ptr, ws.nbytes, None)
    got = out.numpy()
    want, _, parts = A.forward(x, ids, a, b, s, A.values(base))
    assert (np.abs(A.values(got) - want) <= A.forward_tolerance(want, parts, k, rank, "bf16", "bf16")).all()
    assert np.array_equal(got[ids < 0], base[ids < 0])
    copy, other = ctx.upload(base), Guarded(ctx, (m, n), np.uint16)
    NH.call("nh_linear_lora", ctx.handle, *args, copy.ptr, other.ptr, NH.BF16, None, ws.ptr, ws.nbytes, None)
    assert np.array_equal(other.numpy(), got)


# ---- the measured passes ------------------------------------------------------

torch = pytest.importorskip("torch")
PATH = os.path.join(os.path.dirname(__file__), "..", "perf", "more_operators.py")
SMALL = [{"op": "rows", "tokens": 9, "hidden": 70, "experts": 8, "top_k": 2, "x": "bf16"},
         {"op": "rows_train", "tokens": 9, "hidden": 70, "experts": 8, "top_k": 2, "x": "f32"},
         {"op": "lora", "m": 5, "k": 70, "n": 40, "rank": 8, "adapters": 3, "x": "bf16", "w": "bf16", "spread": "rows"},
         {"op": "lora", "m": 130, "k": 70, "n": 40, "rank": 20, "adapters": 3, "x": "bf16", "w": "f32", "spread": "runs"},
         {"op": "lora_train", "m": 130, "k": 70, "n": 40, "rank": 20, "adapters": 3, "x": "bf16", "w": "bf16", "spread": "runs"}]
NAMES = lambda c: f"{c['op']}-{c.get('m', c.get('tokens'))}"  # noqa: E731


@pytest.fixture
def operators():
    spec = importlib.util.spec_from_file_location("more_operators_under_test", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.own = True
    return module


@pytest.mark.parametrize("case", SMALL, ids=NAMES)
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
    state = {"case": case, **{v: t for v in ("indices", "weights", "x", "y", "pos", "dout", "drows", "ids", "base", "a", "b",
                                             "scales", "dx_base")}}
    calls = 0
    for handle in (0x1000, 0x2000, 0x1000):
        Program.stream = handle
        operators.run(state)
        seen = Binding.library.streams[calls:]
        assert seen and all(s == handle for s in seen)
        calls += len(seen)


@pytest.mark.gpu
@pytest.mark.parametrize("case", SMALL, ids=NAMES)
def test_a_state_that_has_run_is_captured_and_replayed(operators, case):
    """First eagerly, then under a capture: replays over other inputs give what an eager pass gives on them."""
    note(f"pass in a graph: {case}")
    states = [operators.prepare(case, seed) for seed in range(3)]
    flat = lambda out: [v.clone() for v in (out.values() if isinstance(out, dict) else [out])]  # noqa: E731
    want = [flat(operators.run(s)) for s in states]
    state = states[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = operators.run(state)
    inputs = [v for v in state if isinstance(state[v], torch.Tensor)]
    for turn in (1, 2, 1):
        for v in inputs:
            state[v].copy_(states[turn][v])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(flat(out), want[turn])), turn
        states[1]["again"] = operators.run(states[1])  # the program's own work between the replays
