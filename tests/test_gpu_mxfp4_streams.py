"""The MXFP4 MoE layer and the router's balance loss in flight twice: on two streams with a workspace each, eager and as
graphs, both launched before either is waited for."""
import numpy as np
import pytest

import mx_reference as R
import nemotron_hip as NH
from test_gpu_moe_balance import U
from test_gpu_mxfp4 import Guarded, moe_case, note, route, tile_all
from test_gpu_mxfp4_edges import moe_want

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = NH.Context(0)
    yield c
    c.close()


# the routes sorted inside the first launch (t = 20), and in one of their own
@pytest.mark.parametrize("t", [20, 300])
def test_experts_and_balance_on_two_streams(ctx, t):
    h, i, e, k, cuts = 520, 250, 24, 4, [0, t // 3, t // 3, t - 3]
    note(f"moe and balance on two streams t={t}")
    rng, _, _, ups, downs = moe_case(ctx, t, h, i, e, k, t)
    du, dd = tile_all(ctx, ups), tile_all(ctx, downs)
    off, up = ctx.upload(np.array(cuts, np.int32)), ctx.upload(np.array([2.0], np.float32))
    graphs, lib = NH.HipGraphs(), NH.lib()

    class Run:
        """One stream's inputs, outputs and workspaces, its calls and a graph of them."""

        def __init__(self):
            self.stream = NH.P()
            NH.call("nh_stream_create", ctx.handle, NH.C.byref(self.stream))
            self.dx, self.dl = ctx.empty((t, h), np.float32), ctx.empty((t, e), np.float32)
            self.idx, self.wts = ctx.empty((t, k), np.int32), ctx.empty((t, k), np.float32)
            self.outs = [Guarded(ctx, (t, h), np.float32), Guarded(ctx, (len(cuts) - 1, e), np.int32),
                         Guarded(ctx, (1,), np.float32), Guarded(ctx, (t, e), np.float32)]
            self.bws = ctx.upload(np.full(lib.nh_moe_balance_loss_workspace_size(len(cuts) - 1, t, e), 0xFF, np.uint8))
            self.mws = ctx.upload(np.full(lib.nh_moe_forward_mxfp4_workspace_size(t, h, i, e, k), 0xFF, np.uint8))
            self.new_inputs()
            self.issue()  # what a program has run before it captures
            self.results()
            self.graph = graphs.capture(self.stream, self.issue)

        def new_inputs(self):
            self.x = R.grid_matrix(rng, t, h, 0)
            self.logits = rng.standard_normal((t, e)).astype(np.float32)
            self.dx.copy_from(self.x)
            self.dl.copy_from(self.logits)

        def issue(self):
            c, s, (out, counts, loss, grad) = ctx.handle, self.stream, self.outs
            NH.call("nh_moe_route_sigmoid_topk", c, self.dl.ptr, t, e, k, 1, 1.0, self.idx.ptr, self.wts.ptr, s)
            NH.call("nh_moe_balance_loss", c, self.dl.ptr, self.idx.ptr, off.ptr, len(cuts) - 1, t, e, k, 0, 0.01, counts.ptr,
                    loss.ptr, self.bws.ptr, self.bws.nbytes, s)
            NH.call("nh_moe_forward_mxfp4", c, self.dx.ptr, NH.F32, self.dl.ptr, t, h, i, e, k, 1, 1.0, du.ptr, dd.ptr, None,
                    None, out.ptr, NH.F32, self.mws.ptr, self.mws.nbytes, None, s)
            NH.call("nh_moe_balance_loss_backward", c, self.dl.ptr, counts.ptr, off.ptr, len(cuts) - 1, t, e, k, 0, 0.01, up.ptr,
                    grad.ptr, s)

        def results(self):
            ctx.synchronize(self.stream)
            return [v.numpy() for v in self.outs]

        def check(self, got):
            want, size = moe_want(self.x, self.logits, ups, downs, k)
            assert (np.abs(got[0] - want) <= (i + 10 + 2 * k) * U * size).all()
            counts, loss, grad = R.balance(self.logits, route(self.logits, k, 1, 1.0)[0], cuts, 0, 0.01, 2.0)
            assert np.array_equal(got[1], counts) and abs(got[2][0] - loss) <= 200 * U * loss
            assert np.abs(got[3] - grad).max() <= 200 * U * np.abs(grad).max()

    runs = [Run(), Run()]
    for turn in range(6):
        order = runs if turn % 2 else runs[::-1]
        for r in order * 2:  # each call's predecessor on the other stream is in flight
            r.issue() if turn < 2 else graphs.launch(r.graph[1], r.stream)
        got = [r.results() for r in order]
        for r, g in zip(order, got):
            r.check(g)
            r.new_inputs()
    for r in runs:
        graphs.destroy(*r.graph)
        NH.call("nh_stream_destroy", ctx.handle, r.stream)
