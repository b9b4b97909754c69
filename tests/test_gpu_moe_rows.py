"""nh_moe_dispatch, nh_moe_combine_rows and their gradients on the device against plain 64-bit forms."""
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


class Case:
    """Routes with some that are not placed (-1, past the slots) and some slots that no route has."""

    def __init__(self, ctx, t, k, h, token, row, shift=0, weights=True, seed=0, spare=3, lost=True):
        rng = self.rng = np.random.default_rng(seed)
        self.ctx, self.t, self.k, self.h, self.token, self.row, self.shift = ctx, t, k, h, token, row, shift
        self.slots = t * k + spare
        self.pos = rng.permutation(self.slots)[:t * k].reshape(t, k).astype(np.int32)
        if lost and t * k > 4:
            flat = self.pos.reshape(-1)
            flat[rng.integers(0, t * k)] = -1
            flat[rng.integers(0, t * k)] = self.slots
            flat[rng.integers(0, t * k)] = 2 ** 31 - 1
        self.dpos = ctx.upload(self.pos)
        self.w = rng.uniform(-1, 1, (t, k)).astype(np.float32) if weights else None
        self.dw_in = ctx.upload(self.w).ptr if weights else None
        if weights:
            self._keep = ctx.upload(self.w)
            self.dw_in = self._keep.ptr
        self.w64 = None if self.w is None else self.w.astype(np.float64)

    def up(self, shape, dtype, bad_rows=()):
        x = self.rng.standard_normal(shape).astype(np.float32)
        stored, v = A.held(x, dtype)
        stored = stored.copy()
        for r in bad_rows:
            stored[r] = A.held(np.full(shape[1], np.nan), dtype)[0]
        buf, at = shifted(self.ctx, stored, self.shift)
        return buf, at, v

    def out(self, rows, dtype):
        return Guarded(self.ctx, (rows, self.h), NP[dtype], self.shift)

    def sizes(self):
        return self.t, self.k, self.h, self.slots

    def check_dweights(self, got, want, size):
        assert (np.abs(got - want) <= 1.01 * (self.h + 20) * A.U * size + 1e-40).all()
        assert (got[~A.placed(self.pos, self.slots)] == 0).all()

    def check_rows(self, out, want, touched):
        got = A.values(out.numpy())
        assert (np.abs(got - want)[touched] <= 1.01 * (A.HALF[self.row] + A.U) * np.abs(want)[touched] + 1e-40).all()
        raw = out.numpy().view(np.uint8).reshape(self.slots, -1)
        assert (raw[~touched] == 0xA5).all(), "a slot that no route has was written"

    def check_tokens(self, out, want, size):
        got = A.values(out.numpy())
        tol = 1.01 * (A.HALF[self.token] * np.abs(want) + 2 * (self.k + 2) * A.U * size) + 1e-40
        assert (np.abs(got - want) <= tol).all()


SHAPES = [(1, 1, 1), (1, 6, 7), (3, 2, 8), (5, 8, 9), (4, 9, 31), (13, 10, 130), (8, 6, 2688), (2, 3, 4096), (3, 17, 4100),
          (40, 4, 2701)]
TYPES = [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32")]


@pytest.mark.parametrize("t,k,h", SHAPES)
@pytest.mark.parametrize("token,row", TYPES)
@pytest.mark.parametrize("shift", [0, 1])
def test_dispatch_and_its_gradient(ctx, t, k, h, token, row, shift):
    note(f"dispatch t={t} k={k} h={h} {token} {row} shift={shift}")
    for weights in (False, True):
        c = Case(ctx, t, k, h, token, row, shift, weights, seed=t + k + h)
        bx, x, vx = c.up((t, h), token)
        rows, dx = c.out(c.slots, row), c.out(t, token)
        NH.call("nh_moe_dispatch", ctx.handle, x, DT[token], c.dpos.ptr, c.dw_in, *c.sizes(), rows.ptr, DT[row], None)
        want, touched, _, _ = A.scatter(vx, c.pos, c.w64, c.slots)
        c.check_rows(rows, want, touched)
        # rows that no route has may hold anything
        bd, d, vd = c.up((c.slots, h), row, bad_rows=np.flatnonzero(~touched))
        dw = Guarded(ctx, (t, k), np.float32)
        out, size, g, g_abs = A.gather(vd, c.pos, c.w64, dot=vx)
        for with_dw in (True, False):
            NH.call("nh_moe_dispatch_backward", ctx.handle, d, DT[row], x if with_dw else None, DT[token], c.dpos.ptr,
                    c.dw_in, *c.sizes(), dx.ptr, dw.ptr if with_dw else None, None)
            c.check_tokens(dx, out, size)
        c.check_dweights(dw.numpy(), g, g_abs)


@pytest.mark.parametrize("t,k,h", SHAPES)
@pytest.mark.parametrize("token,row", TYPES)
@pytest.mark.parametrize("shift", [0, 1])
def test_combine_and_its_gradient(ctx, t, k, h, token, row, shift):
    note(f"combine t={t} k={k} h={h} {token} {row} shift={shift}")
    for weights in (True, False):
        c = Case(ctx, t, k, h, token, row, shift, weights, seed=2 * t + k + h)
        taken = np.zeros(c.slots, bool)
        taken[c.pos[A.placed(c.pos, c.slots)]] = True
        by, y, vy = c.up((c.slots, h), row, bad_rows=np.flatnonzero(~taken))
        bs, shared, vs = c.up((t, h), token)
        out = c.out(t, token)
        for s, v in ((None, None), (shared, vs)):
            NH.call("nh_moe_combine_rows", ctx.handle, y, DT[row], c.dpos.ptr, c.dw_in, s, *c.sizes(), out.ptr, DT[token],
                    None)
            want, size, _, _ = A.gather(vy, c.pos, c.w64, shared=v)
            c.check_tokens(out, want, size)
        # over shared itself
        NH.call("nh_moe_combine_rows", ctx.handle, y, DT[row], c.dpos.ptr, c.dw_in, shared, *c.sizes(), shared, DT[token],
                None)
        ctx.synchronize()
        again = bs.numpy()[shared - bs.ptr:][:t * h * np.dtype(NP[token]).itemsize]
        assert np.array_equal(again, out.numpy().reshape(-1).view(np.uint8))
        bd, d, vd = c.up((t, h), token)
        drows, dw = c.out(c.slots, row), Guarded(ctx, (t, k), np.float32)
        NH.call("nh_moe_combine_rows_backward", ctx.handle, d, DT[token], y, DT[row], c.dpos.ptr, c.dw_in, *c.sizes(),
                drows.ptr, dw.ptr, None)
        want, touched, g, g_abs = A.scatter(vd, c.pos, c.w64, c.slots, rows=vy)
        c.check_rows(drows, want, touched)
        c.check_dweights(dw.numpy(), g, g_abs)
        first = drows.numpy().copy()
        drows2 = c.out(c.slots, row)
        NH.call("nh_moe_combine_rows_backward", ctx.handle, d, DT[token], None, DT[row], c.dpos.ptr, c.dw_in, *c.sizes(),
                drows2.ptr, None, None)
        assert np.array_equal(drows2.numpy(), first)
        # the gradient over the rows themselves
        dw2 = Guarded(ctx, (t, k), np.float32)
        NH.call("nh_moe_combine_rows_backward", ctx.handle, d, DT[token], y, DT[row], c.dpos.ptr, c.dw_in, *c.sizes(), y,
                dw2.ptr, None)
        ctx.synchronize()
        raw = by.numpy()[y - by.ptr:][:first.nbytes].view(first.dtype).reshape(first.shape)
        assert np.array_equal(raw[touched], first[touched])
        assert np.array_equal(dw2.numpy().view(np.uint32), dw.numpy().view(np.uint32))


def test_routes_that_are_not_placed_hide_what_they_hold(ctx):
    """A route without a slot with a NaN weight, a slot of NaN that no route has: neither reaches anything."""
    note("rows: NaN in places that take no part")
    c = Case(ctx, 6, 3, 40, "bf16", "bf16", lost=False)
    c.pos[2] = -1
    c.pos[4, 1] = c.slots + 5
    c.w[2] = np.nan
    c.w[4, 1] = np.inf
    pos, w = ctx.upload(c.pos), ctx.upload(c.w)
    taken = np.zeros(c.slots, bool)
    taken[c.pos[A.placed(c.pos, c.slots)]] = True
    _, y, vy = c.up((c.slots, 40), "bf16", bad_rows=np.flatnonzero(~taken))
    out, dx, dw = c.out(6, "bf16"), c.out(6, "bf16"), Guarded(ctx, (6, 3), np.float32)
    NH.call("nh_moe_combine_rows", ctx.handle, y, NH.BF16, pos.ptr, w.ptr, None, *c.sizes(), out.ptr, NH.BF16, None)
    want, size, _, _ = A.gather(vy, c.pos, c.w.astype(np.float64))
    c.check_tokens(out, want, size)
    assert (out.numpy()[2] == 0).all()
    _, x, vx = c.up((6, 40), "bf16")
    NH.call("nh_moe_dispatch_backward", ctx.handle, y, NH.BF16, x, NH.BF16, pos.ptr, w.ptr, *c.sizes(), dx.ptr, dw.ptr, None)
    assert np.isfinite(A.values(dx.numpy())).all() and np.isfinite(dw.numpy()).all()


def test_nothing_to_do(ctx):
    for t, s in ((0, 4), (0, 0)):
        NH.call("nh_moe_dispatch", ctx.handle, None, NH.F32, None, None, t, 2, 8, s, None, NH.F32, None)
        NH.call("nh_moe_dispatch_backward", ctx.handle, None, NH.F32, None, NH.F32, None, None, t, 2, 8, s, None, None, None)
        NH.call("nh_moe_combine_rows", ctx.handle, None, NH.F32, None, None, None, t, 2, 8, s, None, NH.F32, None)
        NH.call("nh_moe_combine_rows_backward", ctx.handle, None, NH.F32, None, NH.F32, None, None, t, 2, 8, s, None, None, None)
    # no slots: nothing is joined
    pos, out = ctx.upload(np.zeros((3, 2), np.int32)), Guarded(ctx, (3, 8), np.float32)
    NH.call("nh_moe_combine_rows", ctx.handle, None, NH.F32, pos.ptr, None, None, 3, 2, 8, 0, out.ptr, NH.F32, None)
    assert (out.numpy() == 0).all()


@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (700, 16, 3), (9000, 128, 4), (8192, 128, 6), (40000, 8, 2), (33000, 600, 5),
                                   (5000, 4096, 3), (70001, 130, 7)])
def test_sort_of_many_routes(ctx, t, e, k):
    """A stable sort by expert, ids outside the experts and skewed loads among them."""
    note(f"permute t={t} e={e} k={k}")
    rng = np.random.default_rng(t)
    ids = (rng.integers(0, e, (t, k)) * (rng.random((t, k)) < 0.7)).astype(np.int32)
    ids.reshape(-1)[rng.integers(0, t * k, 1 + t // 50)] = rng.choice([-1, e, 2 ** 31 - 1, -2 ** 31])
    d = ctx.upload(ids)
    outs = [Guarded(ctx, (n,), np.int32) for n in (e + 1, t * k, t * k)]
    flat = ids.reshape(-1)
    valid = (flat >= 0) & (flat < e)
    order = np.flatnonzero(valid)[np.argsort(flat[valid], kind="stable")]
    where = np.full(t * k, -1)
    where[order] = np.arange(order.size)
    want = [np.concatenate([[0], np.cumsum(np.bincount(flat[valid], minlength=e))]), order, where]
    for _ in range(2):
        NH.call("nh_moe_permute", ctx.handle, d.ptr, t, k, e, *[o.ptr for o in outs], None)
        off, perm, pos = [o.numpy() for o in outs]
        assert np.array_equal(off, want[0]) and np.array_equal(perm[:order.size], order) and np.array_equal(pos, where)
        for o in outs:
            o.buf.fill_bytes(0xA5)
