"""The sort with pos over its ids, the adapters' workspaces at their ends, rows past the caches, and f32 passes."""
import numpy as np
import pytest

import nemotron_hip as NH
import test_gpu_lora as L
import test_gpu_moe_rows as R
from test_gpu_adapters_together import operators  # noqa: F401
from test_gpu_mxfp4 import Guarded, note

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = NH.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (700, 16, 3), (1500, 128, 8), (9000, 128, 4), (7000, 4096, 3), (33000, 600, 5)])
def test_sort_in_place(ctx, t, e, k):
    note(f"permute in place t={t} e={e} k={k}")
    rng = np.random.default_rng(t)
    ids = rng.integers(0, e, t * k).astype(np.int32)
    if t > 1:
        ids[rng.integers(0, t * k, 9)] = rng.choice([-1, e, 2 ** 31 - 1, -2 ** 31])
    outs = [Guarded(ctx, (n,), np.int32) for n in (e + 1, t * k, t * k)]
    outs[2].buf.copy_from(np.concatenate([np.full(outs[2].at, 0xA5, np.uint8), ids.view(np.uint8), np.full(256, 0xA5, np.uint8)]))
    NH.call("nh_moe_permute", ctx.handle, outs[2].ptr, t, k, e, *[o.ptr for o in outs], None)
    off, perm, pos = [o.numpy() for o in outs]
    valid = (ids >= 0) & (ids < e)
    order = np.flatnonzero(valid)[np.argsort(ids[valid], kind="stable")]
    where = np.full(t * k, -1)
    where[order] = np.arange(order.size)
    assert np.array_equal(off, np.concatenate([[0], np.cumsum(np.bincount(ids[valid], minlength=e))]))
    assert np.array_equal(perm[:order.size], order) and np.array_equal(pos, where)


@pytest.mark.parametrize("m,n,k,rank,adapters,rows", [
    (1, 40, 40, 3, 1, 1), (16, 40, 3000, 16, 64, 1), (64, 2100, 40, 33, 3, 17), (64, 70, 70, 128, 5, 16), (65, 70, 70, 100, 65, 1),
    (300, 130, 2701, 20, 3, 65), (1000, 70, 40, 8, 1024, 1), (2112, 40, 70, 16, 32, 65), (4161, 130, 64, 17, 31, 129),
    (6200, 40, 40, 8, 30, 193), (8385, 64, 130, 64, 40, 193)])
@pytest.mark.parametrize("x,w,out", [("bf16", "bf16", "bf16"), ("f32", "f32", "f32")])
def test_workspaces_end_where_they_say(ctx, monkeypatch, m, n, k, rank, adapters, rows, x, w, out):
    """As many adapters as there are rows for have `rows` each (one more than whole tiles or items of them: the most
    tiles, items and partial sums); nothing is written in front of a workspace or behind it."""
    note(f"lora workspaces m={m} n={n} k={k} rank={rank} adapters={adapters} rows={rows} {x} {w} {out}")
    ids = np.minimum(np.arange(m) // rows, adapters).astype(np.int32)  # the rest have none
    monkeypatch.setattr(L, "make_ids", lambda rng, m, adapters, kind: rng.permutation(ids))
    c = L.Case(ctx, m, n, k, rank, adapters, x, w, out)
    c.ws = [Guarded(ctx, (v.nbytes,), np.uint8) for v in c.ws]
    y, h = Guarded(ctx, (m, n), L.NP[out]), Guarded(ctx, (m, rank), np.float32)
    dx, da, db = [Guarded(ctx, s, d) for s, d in (((m, k), L.NP[x]), ((adapters, rank, k), np.float32), ((adapters, n, rank), np.float32))]
    c.forward(y.ptr, h.ptr)
    c.ws[0].numpy()
    c.check_out(y.numpy())
    for given in (h.ptr, None):
        c.backward(given, dx.ptr, da.ptr, db.ptr)
        c.ws[1].numpy()
        c.check_grads(dx.numpy(), da.numpy(), db.numpy())


@pytest.mark.parametrize("t,k,h", [(1500, 9, 2701), (2100, 6, 2688)])
@pytest.mark.parametrize("token,row", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32")])
def test_rows_past_the_caches(ctx, t, k, h, token, row):
    """64 MiB of rows and more, of several routes a token: the forms whose loads and stores go past the caches."""
    assert t * k * h * (2 if row == "bf16" else 4) >= 64 << 20
    R.test_dispatch_and_its_gradient(ctx, t, k, h, token, row, 1)
    R.test_combine_and_its_gradient(ctx, t, k, h, token, row, 0)


F32 = [{"op": "lora", "m": 5, "k": 70, "n": 40, "rank": 8, "adapters": 3, "x": "f32", "w": "f32", "spread": "rows"},
       {"op": "lora", "m": 2, "k": 70, "n": 41, "rank": 4, "adapters": 3, "x": "f32", "w": "f32", "spread": "rows"},
       {"op": "lora", "m": 130, "k": 70, "n": 40, "rank": 20, "adapters": 3, "x": "f32", "w": "f32", "spread": "runs"},
       {"op": "lora_train", "m": 130, "k": 70, "n": 40, "rank": 20, "adapters": 3, "x": "f32", "w": "f32", "spread": "runs"}]


@pytest.mark.parametrize("case", F32, ids=lambda c: f"{c['op']}-{c['m']}")
def test_f32_passes_eager_and_replayed(operators, case):  # noqa: F811
    """An f32 pass adds onto its base where it stands, so inputs are new before each: eager and replayed passes of the
    same inputs have the same bits, and the library out of place has them too and leaves its inputs alone."""
    torch = pytest.importorskip("torch")
    note(f"f32 pass: {case}")
    flat = lambda out: [v.clone() for v in (out.values() if isinstance(out, dict) else [out])]  # noqa: E731
    inputs = lambda s: {v: s[v].clone() for v in s if isinstance(s[v], torch.Tensor)}  # noqa: E731
    fresh = [inputs(operators.prepare(case, seed)) for seed in range(3)]
    want = [flat(operators.run({"case": case, **{v: t.clone() for v, t in f.items()}})) for f in fresh]
    state = {"case": case, **{v: t.clone() for v, t in fresh[0].items()}}
    operators.run(state)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = operators.run(state)
    for turn in (1, 2, 1, 0):
        for v, t in fresh[turn].items():
            state[v].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(flat(out), want[turn])), turn
        for v, t in fresh[turn].items():  # the same state's eager pass
            state[v].copy_(t)
        assert all(torch.equal(a, b) for a, b in zip(flat(operators.run(state)), want[turn])), turn
    monkey = operators._Bound.onto
    try:
        operators._Bound.onto = lambda self, case, base: self.empty(base.shape, base.dtype)
        apart = {"case": case, **{v: t.clone() for v, t in fresh[0].items()}}
        for _ in range(2):  # a second pass starts from the same base
            assert all(torch.equal(a, b) for a, b in zip(flat(operators.run(apart)), want[0]))
        assert all(torch.equal(apart[v], t) for v, t in fresh[0].items())
    finally:
        operators._Bound.onto = monkey
