"""The router's balance loss, its counts and its gradient on the device, against the plain 64-bit form; and a training
step's run of router, balance loss and MXFP4 experts, captured and replayed."""
import numpy as np
import pytest

import mx_reference as R
import nemotron_hip as NH
from test_gpu_mxfp4 import Guarded, moe_case, note, tile_all

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    c = NH.Context(0)
    yield c
    c.close()


def run(ctx, z, idx, seq, softmax, coefficient=0.5, dloss=1.5, stream=None):
    t, e = z.shape
    k = idx.shape[1]
    off = None if seq is None else ctx.upload(np.array(seq, np.int32))
    s = 1 if seq is None else len(seq) - 1
    dz, di, up = ctx.upload(z), ctx.upload(idx), ctx.upload(np.array([dloss], np.float32))
    need = NH.lib().nh_moe_balance_loss_workspace_size(s, t, e)
    ws = ctx.upload(np.full(need, 0xFF, np.uint8))
    counts, loss = Guarded(ctx, (s, e), np.int32), Guarded(ctx, (1,), np.float32)
    grad = Guarded(ctx, (t, e), np.float32)
    NH.call("nh_moe_balance_loss", ctx.handle, dz.ptr, di.ptr, NH.ptr(off), s, t, e, k, softmax, coefficient, counts.ptr,
            loss.ptr, ws.ptr, need, stream)
    NH.call("nh_moe_balance_loss_backward", ctx.handle, dz.ptr, counts.ptr, NH.ptr(off), s, t, e, k, softmax, coefficient,
            up.ptr, grad.ptr, stream)
    ctx.synchronize(stream)
    return counts.numpy(), loss.numpy()[0], grad.numpy()


def routes(rng, t, e, k):
    return np.argsort(rng.random((t, e)), axis=1)[:, :k].astype(np.int32)


def check(got, want, z, seq, softmax, dloss):
    counts, loss, grad = got
    rc, rl, rg = want
    assert np.array_equal(counts, rc)
    t, e = z.shape
    # p: exp's argument (|z| up to A, rounded to 2^-24 A) and its own 2^-22, the row's sum of e terms, a quotient
    a = np.abs(np.where(np.isfinite(z), z, 0)).max() if z.size else 0
    p_err = (2 * a + 16 + np.log2(max(e, 2)) + 4) * U
    # the loss: sums over up to t / 256 + 64 tokens in a lane, the rest in a tree
    assert abs(loss - rl) <= (p_err + (t / 256 + 80) * U) * abs(rl) + 1e-30
    # the gradient: p (f - sum f p) d, the difference's error is of the size of its larger part
    k_err = 4 * p_err + (e + 8) * U
    for s, (lo, hi) in enumerate(R.offsets_of(seq, t)):
        if hi <= lo:
            continue
        top = 2 * counts[s].max() * e / max(1, counts[s].sum())
        for row in range(lo, hi):
            p, slope = R.probabilities(z[row].astype(np.float64), softmax)
            part = 0.5 / (len(R.offsets_of(seq, t)) * (hi - lo)) * dloss
            assert (np.abs(grad[row] - rg[row]) <= k_err * part * p * slope * max(top, 1) + 1e-37).all(), row


# lanes per token from one to 64, experts ragged against four; rows at the ends of chunks, empty and one-token sequences,
# padding before, between (an offset repeated) and behind
SHAPES = [(1, 1, 1, None), (1, 128, 6, None), (3, 4, 2, None), (7, 5, 2, [0, 3, 7]), (65, 8, 2, None), (64, 60, 4, [0, 64]),
          (100, 128, 6, [0, 0, 1, 1, 50, 97]), (129, 128, 8, [5, 60, 129]), (300, 256, 2, None), (70, 257, 3, [0, 30, 70]),
          (40, 512, 8, None), (33, 1000, 4, [1, 2, 33]), (20, 1024, 1, None), (20000, 16, 2, None), (17000, 7, 1, [0, 16000, 16999]),
          (500, 6, 3, list(range(0, 401, 2)))]


@pytest.mark.parametrize("t,e,k,seq", SHAPES)
@pytest.mark.parametrize("softmax", [0, 1])
def test_balance(ctx, t, e, k, seq, softmax):
    note(f"balance t={t} e={e} k={k} sequences={1 if seq is None else len(seq) - 1} softmax={softmax}")
    rng = np.random.default_rng(t + e + softmax)
    z = (rng.standard_normal((t, e)) * 2).astype(np.float32)
    idx = routes(rng, t, e, k)
    got = run(ctx, z, idx, seq, softmax)
    check(got, R.balance(z, idx, seq, softmax, 0.5, 1.5), z, seq, softmax, 1.5)
    inside = np.zeros(t, bool)
    for lo, hi in R.offsets_of(seq, t):
        inside[lo:hi] = True
    assert (got[2][~inside] == 0).all()  # every row is written, padding with zeros


@pytest.mark.parametrize("count", [65, 300, 1500])
def test_balance_of_many_sequences(ctx, count):
    """More sequences than one step over the offsets takes, some of them empty, with rows before and behind."""
    t, e, k = 2000, 24, 3
    note(f"balance of {count} sequences")
    rng = np.random.default_rng(count)
    seq = np.sort(rng.integers(5, t - 7, count + 1)).astype(np.int32)
    z = (rng.standard_normal((t, e)) * 2).astype(np.float32)
    idx = routes(rng, t, e, k)
    got, want = run(ctx, z, idx, seq.tolist(), 0), R.balance(z, idx, seq.tolist(), 0, 0.5, 1.5)
    check(got, want, z, seq.tolist(), 0, 1.5)


@pytest.mark.parametrize("softmax", [0, 1])
def test_balance_of_extreme_rows(ctx, softmax):
    note(f"balance extremes softmax={softmax}")
    rng = np.random.default_rng(0)
    t, e, k = 12, 20, 3
    z = rng.standard_normal((t, e)).astype(np.float32)
    idx = routes(rng, t, e, k)
    z[0] -= 200  # every sigmoid below the smallest f32
    z[1] += 200
    z[2, 5:] = -np.inf  # masked experts
    z[3] = -np.inf      # nothing left
    z[4, 1:] = np.finfo(np.float32).min
    z[5] = np.finfo(np.float32).min
    idx[6, 0], idx[7, 1] = -1, e  # routes that were dropped
    counts, loss, grad = run(ctx, z, idx, None, softmax)
    rc, rl, rg = R.balance(z, idx, None, softmax, 0.5, 1.5)
    assert np.array_equal(counts, rc) and np.isfinite(loss) and np.isfinite(grad).all()
    assert abs(loss - rl) <= 600 * U * abs(rl)  # arguments of exp up to 200: 2^-24 * 2 * 200, twice
    assert (grad[3] == 0).all()
    # row 1's 1 - sigmoid is e^-200 = 1e-87, which f32 does not hold: what lies below its normal range counts as 0.
    # row 4 has one expert alone, so f - f p is f - f: exactly 0, but p = u * (1 / u) is off by the roundings of the
    # reciprocal (2 U) and the product (U), and f p by one more, so the difference by 4 U of f
    part = 0.5 * 1.5 / t * (np.arange(t) == 4)[:, None] * rc.max() * e / (k * t)
    assert (np.abs(grad - rg) <= 2000 * U * np.abs(rg).max(axis=1, keepdims=True) + 4 * U * part + 2.0 ** -126).all()


@pytest.mark.parametrize("softmax", [0, 1])
def test_balance_nan_and_infinity(ctx, softmax):
    rng = np.random.default_rng(1)
    z, idx = rng.standard_normal((10, 9)).astype(np.float32), routes(rng, 10, 9, 2)
    z[4, 8] = np.nan
    _, loss, grad = run(ctx, z, idx, None, softmax)
    assert np.isnan(loss) and np.isnan(grad[4]).all() and np.isfinite(np.delete(grad, 4, 0)).all()
    if not softmax:  # a sigmoid of infinity is 1
        z[4, 8] = np.inf
        got = run(ctx, z, idx, None, softmax)
        z[4, 8] = 100.0
        want = R.balance(z, idx, None, softmax, 0.5, 1.5)
        assert abs(got[1] - want[1]) <= 100 * U * want[1] and np.abs(got[2] - want[2]).max() <= 200 * U * np.abs(want[2]).max()


def test_balance_of_no_tokens(ctx):
    z, idx = np.zeros((0, 8), np.float32), np.zeros((0, 2), np.int32)
    counts, loss, _ = run(ctx, z, idx, None, 1)
    assert (counts == 0).all() and loss == 0
    counts, loss, _ = run(ctx, z, idx, [0, 0, 0], 0)
    assert (counts == 0).all() and loss == 0


@pytest.mark.parametrize("seq", [[0, 50, 0, 50], [-7, 20, 1000], [40, 3, 60], [9, 9, 2, 2000000000, -1]])
def test_balance_bad_offsets_stay_in_bounds(ctx, seq):
    note(f"balance bad offsets {seq}")
    rng = np.random.default_rng(2)
    z, idx = rng.standard_normal((60, 12)).astype(np.float32), routes(rng, 60, 12, 2)
    counts, _, grad = run(ctx, z, idx, seq, 0)  # the guards around the outputs are checked
    assert (counts >= 0).all() and np.isfinite(grad).all()


def test_balance_is_repeatable(ctx):
    rng = np.random.default_rng(4)
    z, idx = rng.standard_normal((5000, 64)).astype(np.float32), routes(rng, 5000, 64, 4)
    first = run(ctx, z, idx, [0, 700, 4999], 0)
    for _ in range(3):
        again = run(ctx, z, idx, [0, 700, 4999], 0)
        assert all(np.array_equal(a, b) for a, b in zip(first, again))


def test_balance_gradient_against_differences(ctx):
    """The device's gradient against central differences of the 64-bit loss."""
    rng = np.random.default_rng(5)
    z, idx, seq = rng.standard_normal((8, 10)).astype(np.float32), routes(rng, 8, 10, 3), [0, 5, 8]
    for softmax in (0, 1):
        grad = run(ctx, z, idx, seq, softmax, dloss=1.0)[2]
        for row, col in np.ndindex(z.shape):
            hi, lo = z.astype(np.float64), z.astype(np.float64)
            hi[row, col] += 1e-5
            lo[row, col] -= 1e-5
            slope = (R.balance(hi, idx, seq, softmax, 0.5)[1] - R.balance(lo, idx, seq, softmax, 0.5)[1]) / 2e-5
            assert abs(slope - grad[row, col]) <= 200 * U * np.abs(grad).max() + 1e-9


def test_router_balance_and_experts_captured_and_replayed(ctx):
    """As a training step uses them: routes, balance loss and its gradient, the MXFP4 experts and a quantized copy of the
    output, on a stream, eager and as a graph replayed on other inputs; twice the same graph's calls on two workspaces."""
    t, h, i, e, k = 37, 200, 96, 16, 3
    note("router + balance + experts in a graph")
    rng, x, logits, ups, downs = moe_case(ctx, t, h, i, e, k, 3)
    du, dd = tile_all(ctx, ups), tile_all(ctx, downs)
    dx, dl, off = ctx.upload(x), ctx.upload(logits), ctx.upload(np.array([0, 20, 35], np.int32))
    up = ctx.upload(np.array([2.0], np.float32))
    stream = NH.P()
    NH.call("nh_stream_create", ctx.handle, NH.C.byref(stream))

    class Set:
        def __init__(self):
            lib = NH.lib()
            self.idx, self.wts = ctx.empty((t, k), np.int32), ctx.empty((t, k), np.float32)
            self.counts, self.loss = ctx.empty((2, e), np.int32), ctx.empty(1, np.float32)
            self.grad, self.out = ctx.empty((t, e), np.float32), ctx.empty((t, h), np.uint16)
            self.codes, self.scales = ctx.empty((t, h // 2), np.uint8), ctx.empty((t, -(-h // 32)), np.uint8)
            self.bws = ctx.empty(lib.nh_moe_balance_loss_workspace_size(2, t, e), np.uint8)
            self.mws = ctx.empty(lib.nh_moe_forward_mxfp4_workspace_size(t, h, i, e, k), np.uint8)

        def issue(self):
            c, s = ctx.handle, stream
            NH.call("nh_moe_route_sigmoid_topk", c, dl.ptr, t, e, k, 1, 1.0, self.idx.ptr, self.wts.ptr, s)
            NH.call("nh_moe_balance_loss", c, dl.ptr, self.idx.ptr, off.ptr, 2, t, e, k, 0, 0.01, self.counts.ptr,
                    self.loss.ptr, self.bws.ptr, self.bws.nbytes, s)
            NH.call("nh_moe_balance_loss_backward", c, dl.ptr, self.counts.ptr, off.ptr, 2, t, e, k, 0, 0.01, up.ptr,
                    self.grad.ptr, s)
            NH.call("nh_moe_forward_mxfp4", c, dx.ptr, NH.F32, dl.ptr, t, h, i, e, k, 1, 1.0, du.ptr, dd.ptr, None, None,
                    self.out.ptr, NH.BF16, self.mws.ptr, self.mws.nbytes, None, s)
            NH.call("nh_quantize_rows_mxfp4", c, self.out.ptr, NH.BF16, t, h, self.codes.ptr, self.scales.ptr, None, s)

        def results(self):
            ctx.synchronize(stream)
            return [v.numpy() for v in (self.idx, self.counts, self.loss, self.grad, self.out, self.codes, self.scales)]

    eager, one, two = Set(), Set(), Set()
    graphs = NH.HipGraphs()
    captured = [graphs.capture(stream, s.issue) for s in (one, two)]
    for turn in range(4):
        logits = rng.standard_normal((t, e)).astype(np.float32)
        dl.copy_from(logits)
        dx.copy_from(R.grid_matrix(rng, t, h, 0))
        eager.issue()
        want = eager.results()
        for _, ex in captured:  # both in flight, each on its own workspace
            graphs.launch(ex, stream)
        for got in (one.results(), two.results()):
            assert all(np.array_equal(a, b) for a, b in zip(got, want)), turn
        rc, rl, _ = R.balance(logits, want[0], [0, 20, 35], 0, 0.01)
        assert np.array_equal(want[1], rc) and abs(want[2][0] - rl) <= 200 * U * rl
        assert (want[3][35:] == 0).all()
        codes, scales, _ = R.quantize(R.from_bf16_bits(want[4]))
        assert np.array_equal(want[5], codes) and np.array_equal(want[6], scales)
    for g, ex in captured:
        graphs.destroy(g, ex)
    NH.call("nh_stream_destroy", ctx.handle, stream)
