"""nh_linear_lora and its gradients on the device against plain 64-bit forms."""
import numpy as np
import pytest

import adapters_reference as A
import nemotron_hip as NH
from test_gpu_mxfp4 import Guarded, note, shifted

pytestmark = pytest.mark.gpu

DT = {"f32": NH.F32, "bf16": NH.BF16}
NP = {"f32": np.float32, "bf16": np.uint16}


@pytest.fixture(scope="module")
def ctx():
    c = NH.Context(0)
    yield c
    c.close()


def make_ids(rng, m, adapters, kind):
    if kind == "each":
        ids = rng.integers(-1, adapters, m)
    elif kind == "runs":
        cuts = np.sort(rng.integers(0, m + 1, min(m, 2 * adapters)))
        ids = (np.searchsorted(cuts, np.arange(m), side="right") % (adapters + 1)) - 1
    elif kind == "one":
        ids = np.full(m, adapters - 1)
    else:
        ids = rng.choice([-1, adapters, 2 ** 31 - 1, -2 ** 31], m)
    ids = ids.astype(np.int32)
    if kind == "each" and m > 3:
        ids[1] = adapters + 7
    return ids


class Case:
    def __init__(self, ctx, m, n, k, rank, adapters, x="bf16", w="bf16", out="bf16", kind="each", shift=0, base=True,
                 scales=True, seed=0):
        rng = np.random.default_rng(seed + m + n + k + rank)
        self.ctx, self.sizes, self.types, self.shift = ctx, (m, n, k, rank, adapters), (x, w, out), shift
        self.ids = make_ids(rng, m, adapters, kind)
        # what no row may see: other adapters' matrices and other rows
        used = np.zeros(adapters, bool)
        valid = (self.ids >= 0) & (self.ids < adapters)
        used[self.ids[valid]] = True
        xs, self.x = A.held(rng.standard_normal((m, k)), x)
        as_, self.a = A.held(rng.standard_normal((adapters, rank, k)) / np.sqrt(k), w)
        bs, self.b = A.held(rng.standard_normal((adapters, n, rank)), w)
        os_, self.base = A.held(rng.standard_normal((m, n)), out)
        ds, self.dout = A.held(rng.standard_normal((m, n)), out)
        gs, self.dx_base = A.held(rng.standard_normal((m, k)), x)
        nan16, nan32 = np.uint16(0x7FC0), np.float32(np.nan)
        for stored in (as_, bs):
            stored[~used] = nan16 if w == "bf16" else nan32
        for stored, d in ((xs, x), (ds, out)):
            stored[~valid] = nan16 if d == "bf16" else nan32
        self.s = rng.uniform(0.25, 2, adapters).astype(np.float32) * rng.choice([-1, 1], adapters) if scales else None
        if scales:
            self.s = self.s.astype(np.float32)
            self.s[~used] = np.nan
        up = lambda v, sh=shift: shifted(ctx, v, sh)  # noqa: E731
        self.keep = {"x": up(xs), "ids": up(self.ids, shift), "a": up(as_), "b": up(bs), "base": up(os_), "dout": up(ds),
                     "dx_base": up(gs), "s": up(self.s if scales else np.zeros(1, np.float32))}
        self.p = {n_: v[1] for n_, v in self.keep.items()}
        if not base:
            self.base, self.dx_base, self.p["base"], self.p["dx_base"] = None, None, None, None
        if not scales:
            self.p["s"] = None
        lib = NH.lib()
        self.ws = [ctx.upload(np.full(f(*self.sizes), 0xFF, np.uint8)) for f in
                   (lib.nh_linear_lora_workspace_size, lib.nh_linear_lora_backward_workspace_size)]
        with np.errstate(invalid="ignore"):
            self.want = A.forward(self.x, self.ids, self.a, self.b, self.s, self.base)
            self.grads = A.backward(self.x, self.ids, self.a, self.b, self.s, self.dout, self.dx_base)

    def forward(self, out, h=None, stream=None, base=None, **over):
        x, w, o = self.types
        p = {**self.p, **over}
        NH.call("nh_linear_lora", self.ctx.handle, p["x"], DT[x], p["ids"], p["a"], p["b"], DT[w], p["s"], *self.sizes,
                p["base"] if base is None else base, out, DT[o], h, self.ws[0].ptr, self.ws[0].nbytes, stream)

    def backward(self, h, dx, da, db, accumulate=0, stream=None, **over):
        x, w, o = self.types
        p = {**self.p, **over}
        NH.call("nh_linear_lora_backward", self.ctx.handle, p["x"], DT[x], p["ids"], p["a"], p["b"], DT[w], p["s"], h,
                p["dout"], DT[o], *self.sizes, p["dx_base"], dx, da, db, accumulate, self.ws[1].ptr, self.ws[1].nbytes,
                stream)

    def check_out(self, got):
        m, n, k, rank, _ = self.sizes
        want, _, parts = self.want
        assert (np.abs(A.values(got) - want) <= A.forward_tolerance(want, parts, k, rank, *self.types[1:])).all()

    def check_grads(self, dx=None, da=None, db=None, da0=0.0, db0=0.0):
        m, n, k, rank, adapters = self.sizes
        x, w, o = self.types
        wdx, wda, wdb, parts = self.grads
        if dx is not None:
            tol = A.forward_tolerance(wdx, parts, n, rank, w, x)
            assert (np.abs(A.values(dx) - wdx) <= tol).all()
        if da is not None:
            assert (np.abs(da - wda - da0) <= A.gradient_tolerance(parts, "da", n, m) + A.U * np.abs(wda + da0)).all()
        if db is not None:
            assert (np.abs(db - wdb - db0) <= A.gradient_tolerance(parts, "db", k, m) + A.U * np.abs(wdb + db0)).all()


SHAPES = [  # m, n, k, rank, adapters, ids
    (1, 1, 1, 1, 1, "one"), (1, 300, 517, 16, 3, "one"), (2, 40, 64, 128, 2, "each"), (16, 96, 130, 8, 1, "one"),
    (17, 33, 31, 5, 1, "one"), (33, 129, 257, 33, 2, "each"), (64, 64, 64, 64, 70, "each"), (64, 100, 96, 20, 1, "one"),
    (5, 50, 60, 7, 4, "none"), (65, 64, 40, 8, 1, "one"), (66, 70, 41, 9, 300, "each"), (130, 48, 300, 33, 4, "runs"),
    (300, 513, 700, 64, 5, "runs"), (500, 40, 96, 100, 3, "runs"), (80, 31, 33, 4, 2, "none"), (1000, 65, 72, 17, 1024, "each"),
    (2200, 130, 70, 12, 2, "runs"), (3, 4200, 5000, 16, 2, "each"), (40, 2700, 9000, 24, 3, "each"),
    (150, 3100, 4500, 16, 2, "runs"), (97, 5000, 2600, 40, 2, "runs"), (70, 2049, 2303, 72, 1, "one"),
    (9000, 33, 40, 5, 1024, "each"), (63, 300, 130, 40, 3, "each"), (64, 1030, 90, 16, 2, "runs"), (8200, 40, 70, 16, 3, "runs"),
    (20011, 24, 16, 3, 7, "each")]
TYPES = [("bf16", "bf16", "bf16"), ("f32", "f32", "f32"), ("bf16", "f32", "bf16"), ("bf16", "bf16", "f32"),
         ("f32", "bf16", "bf16")]


@pytest.mark.parametrize("m,n,k,rank,adapters,kind", SHAPES)
@pytest.mark.parametrize("x,w,out", TYPES)
def test_forward(ctx, m, n, k, rank, adapters, kind, x, w, out):
    for shift, base, scales in ((0, True, True), (1, False, False)):
        note(f"lora m={m} n={n} k={k} rank={rank} adapters={adapters} {kind} {x} {w} {out} shift={shift}")
        c = Case(ctx, m, n, k, rank, adapters, x, w, out, kind, shift, base, scales)
        y, h = Guarded(ctx, (m, n), NP[out], shift), Guarded(ctx, (m, rank), np.float32, shift)
        c.forward(y.ptr, h.ptr)
        c.check_out(y.numpy())
        assert (np.abs(h.numpy() - c.want[1]) <= A.h_tolerance(c.want[2], k)).all()
        bare = (c.ids < 0) | (c.ids >= adapters)
        assert (h.numpy()[bare] == 0).all()
        if base:  # rows without an adapter are their base to the bit; out over base gives the same
            raw = np.frombuffer(c.keep["base"][0].numpy()[c.p["base"] - c.keep["base"][0].ptr:][:y.nbytes], NP[out]).reshape(m, n)
            assert np.array_equal(y.numpy()[bare], raw[bare])
            c.forward(c.p["base"], None)
            ctx.synchronize()
            again = np.frombuffer(c.keep["base"][0].numpy()[c.p["base"] - c.keep["base"][0].ptr:][:y.nbytes], NP[out])
            assert np.array_equal(again.reshape(m, n), y.numpy())
        else:
            assert (A.values(y.numpy())[bare] == 0).all()


@pytest.mark.parametrize("m,n,k,rank,adapters,kind", SHAPES)
@pytest.mark.parametrize("x,w,out", TYPES)
def test_backward(ctx, m, n, k, rank, adapters, kind, x, w, out):
    for shift, base, scales in ((0, True, True), (1, False, False)):
        note(f"lora backward m={m} n={n} k={k} rank={rank} adapters={adapters} {kind} {x} {w} {out} shift={shift}")
        c = Case(ctx, m, n, k, rank, adapters, x, w, out, kind, shift, base, scales, seed=1)
        h = ctx.empty((m, rank), np.float32)
        y = ctx.empty((m, n), NP[out])
        c.forward(y.ptr, h.ptr)
        dx = Guarded(ctx, (m, k), NP[x], shift)
        da, db = Guarded(ctx, (adapters, rank, k), np.float32, shift), Guarded(ctx, (adapters, n, rank), np.float32, shift)
        c.backward(h.ptr, dx.ptr, da.ptr, db.ptr)
        first = [v.numpy().copy() for v in (dx, da, db)]
        c.check_grads(*first)
        # h computed again, and added to what was there
        c.backward(None, dx.ptr, da.ptr, db.ptr, accumulate=1)
        c.check_grads(dx.numpy(), da.numpy(), db.numpy(), first[1].astype(np.float64), first[2].astype(np.float64))
        assert np.array_equal(dx.numpy(), first[0])
        # each alone, without what it does not need
        c.backward(None, dx.ptr, None, None, x=None)
        assert np.array_equal(dx.numpy(), first[0])
        c.backward(None, None, da.ptr, None, a=None)
        assert np.array_equal(da.numpy(), first[1])
        c.backward(h.ptr, None, None, db.ptr, x=None, a=None, b=None)
        assert np.array_equal(db.numpy(), first[2])
        if base:  # over dx_base itself
            c.backward(h.ptr, c.p["dx_base"], None, None)
            ctx.synchronize()
            buf = c.keep["dx_base"][0]
            again = np.frombuffer(buf.numpy()[c.p["dx_base"] - buf.ptr:][:dx.nbytes], NP[x]).reshape(m, k)
            assert np.array_equal(again, first[0])


@pytest.mark.parametrize("m", [40, 200])
def test_gradients_are_differences(ctx, m):
    """<dout, out(p + e v) - out(p - e v)> / 2 e of the 64-bit forward form is <gradient, v>: out is bilinear in (a, b)
    and linear in x, so the difference along one of them has no error of its own beyond 64 bits."""
    note(f"lora differences m={m}")
    c = Case(ctx, m, 70, 50, 6, 3, "f32", "f32", "f32", "runs" if m > 64 else "each")
    dx, da, db = (ctx.empty(s, np.float32) for s in (c.x.shape, c.a.shape, c.b.shape))
    c.backward(None, dx.ptr, da.ptr, db.ptr)
    ctx.synchronize()
    base = np.zeros_like(c.base)
    bare = (c.ids < 0) | (c.ids >= 3)
    rng = np.random.default_rng(5)
    x, dout = np.where(bare[:, None], 0, c.x), np.where(bare[:, None], 0, c.dout)
    g = dx.numpy().astype(np.float64) - c.dx_base
    for got, at, tol in ((g, "x", c.grads[3]["far"]), (da.numpy(), "a", c.grads[3]["da_far"]), (db.numpy(), "b", c.grads[3]["db_far"])):
        v = rng.standard_normal(got.shape)
        e, p = 0.5, {"x": x, "a": c.a, "b": c.b}
        diff = 0.0
        for sign in (1, -1):
            q = {**p, at: p[at] + sign * e * v}
            diff += sign * (dout * A.forward(q["x"], c.ids, q["a"], q["b"], c.s, base)[0]).sum() / (2 * e)
        slack = (3 * m + 200) * A.U * (np.abs(v) * (tol + (np.abs(dx.numpy()) if at == "x" else 0))).sum()
        assert abs((got * v).sum() - diff) <= slack


def test_the_same_bits_on_every_run(ctx):
    note("lora determinism")
    c = Case(ctx, 700, 300, 520, 24, 5, kind="each")
    outs = [Guarded(ctx, s, d) for s, d in (((700, 300), np.uint16), ((700, 520), np.uint16), ((5, 24, 520), np.float32),
                                            ((5, 300, 24), np.float32))]
    seen = []
    for _ in range(3):
        c.forward(outs[0].ptr)
        c.backward(None, *[o.ptr for o in outs[1:]])
        seen.append([o.numpy().copy() for o in outs])
    assert all(np.array_equal(a, b) for s in seen[1:] for a, b in zip(seen[0], s))


def test_infinities_stay_in_their_rows(ctx):
    note("lora non-finite rows")
    for m, adapters in ((30, 3), (150, 3)):
        c = Case(ctx, m, 64, 64, 8, adapters, kind="one")
        buf, at = c.keep["x"]
        raw = buf.numpy()
        x = raw[at - buf.ptr:][:m * 64 * 2].view(np.uint16).reshape(m, 64)
        x[3, 5], x[7, 9] = 0x7F80, 0x7FC0
        buf.copy_from(raw)
        y, dx = Guarded(ctx, (m, 64), np.uint16), Guarded(ctx, (m, 64), np.uint16)
        c.forward(y.ptr)
        got = A.values(y.numpy())
        rows = np.delete(np.arange(m), [3, 7])
        want, _, parts = c.want
        tol = A.forward_tolerance(want, parts, 64, 8, *c.types[1:])
        assert (np.abs(got - want) <= tol)[rows].all() and not np.isfinite(got[3]).any() and np.isnan(got[7]).all()
        c.backward(None, dx.ptr, None, None)  # dx does not depend on x
        c.check_grads(dx=dx.numpy())


@pytest.mark.parametrize("m", [24, 500])
def test_two_streams_and_graphs(ctx, m):
    """Two training steps in flight, eager and replayed, with new ids and rows between the replays."""
    note(f"lora on two streams m={m}")
    graphs = NH.HipGraphs()

    class Run:
        def __init__(self, seed):
            self.stream = NH.P()
            NH.call("nh_stream_create", ctx.handle, NH.C.byref(self.stream))
            self.seed = seed
            self.c = Case(ctx, m, 200, 330, 12, 4, kind="each", seed=seed)
            self.h = ctx.empty((m, 12), np.float32)
            self.outs = [Guarded(ctx, s, d) for s, d in (((m, 200), np.uint16), ((m, 330), np.uint16),
                                                         ((4, 12, 330), np.float32), ((4, 200, 12), np.float32))]
            self.issue()
            self.check()
            self.graph = graphs.capture(self.stream, self.issue)

        def issue(self):
            self.c.forward(self.outs[0].ptr, self.h.ptr, stream=self.stream)
            self.c.backward(self.h.ptr, *[o.ptr for o in self.outs[1:]], stream=self.stream)

        def renew(self):
            self.seed += 10
            new = Case(ctx, m, 200, 330, 12, 4, kind="each", seed=self.seed)
            for name in self.c.keep:
                self.c.keep[name][0].copy_from(new.keep[name][0].numpy())
            self.c.want, self.c.grads, self.c.ids = new.want, new.grads, new.ids

        def check(self):
            ctx.synchronize(self.stream)
            got = [o.numpy() for o in self.outs]
            self.c.check_out(got[0])
            self.c.check_grads(*got[1:])

    runs = [Run(1), Run(2)]
    for turn in range(5):
        order = runs if turn % 2 else runs[::-1]
        for r in order * 2:
            r.issue() if turn < 1 else graphs.launch(r.graph[1], r.stream)
        for r in order:
            r.check()
            r.renew()
    for r in runs:
        graphs.destroy(*r.graph)
        NH.call("nh_stream_destroy", ctx.handle, r.stream)
