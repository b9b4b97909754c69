"""MXFP4 products and experts at the edges of their launch: runs of units that the waves' groups do not share evenly."""
import ctypes as C

import numpy as np
import pytest

import mx_reference as R
import nemotron_hip as NH
from test_gpu_mxfp4 import Guarded, U, moe_case, note, route, run_linear, tile_all, weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = NH.Context(0)
    yield c
    c.close()


# K of up to 512 leaves four or eight groups of waves, and a run of one or two units of 16 columns: the groups behind
# the run's last unit have no outputs and no bias to read.  128 bytes of bias lie in LDS where four groups would have read
# 256, eight 512.
@pytest.mark.parametrize("m,n,k", [(1, 4112, 512), (16, 4112, 100), (3, 16, 128), (2, 8209, 500), (40, 4112, 512)])
def test_bias_of_groups_without_a_unit(ctx, m, n, k):
    note(f"bias, idle groups m={m} n={n} k={k}")
    rng = np.random.default_rng(n + k)
    x, w, bias = R.grid_matrix(rng, m, k, 0), R.grid_matrix(rng, n, k, 0), R.grid_matrix(rng, 1, n, 0)[0]
    tiled, _ = weights(ctx, w)
    assert np.array_equal(run_linear(ctx, x, tiled, n, bias), x @ w.T + bias)  # sums of quarters, exact in f32


def moe(ctx, x, logits, du, dd, h, i, k, biases=None, out_dtype=NH.F32):
    """The layer on f32 rows, renormalised routes: (output, non-finite status)."""
    t, e = logits.shape
    dx, dl = ctx.upload(x), ctx.upload(logits)
    need = NH.lib().nh_moe_forward_mxfp4_workspace_size(t, h, i, e, k)
    ws = ctx.upload(np.full(need, 0xFF, np.uint8))
    out, word = Guarded(ctx, (t, h), np.float32), ctx.upload(np.zeros(1, np.uint64))
    NH.call("nh_moe_forward_mxfp4", ctx.handle, dx.ptr, NH.F32, dl.ptr, t, h, i, e, k, 1, 1.0, du.ptr, dd.ptr, biases, None,
            out.ptr, out_dtype, ws.ptr, need, word.ptr, None)
    ctx.synchronize()
    return out.numpy(), NH.call_status("nh_take_nonfinite", ctx.handle, word.ptr, None)[0]


def moe_want(x, logits, ups, downs, k, bu=None, bd=None):
    """The layer in 64 bits, and the size of its sums.  The sums before h are exact in f32, so h is the kernel's."""
    idx, wts = route(logits, k, 1, 1.0)
    t, h = x.shape
    want, size = np.zeros((t, h)), np.zeros((t, h))
    for n in range(logits.shape[1]):
        tok, j = np.nonzero(idx == n)
        if tok.size == 0:
            continue
        y = (x[tok].astype(np.float32) @ ups[n].T + (0 if bu is None else bu[n])).astype(np.float32)
        hv = R.quantize((np.maximum(y, 0) ** 2).astype(np.float32))[2]
        d, s = hv @ downs[n].T.astype(np.float64), np.abs(hv) @ np.abs(downs[n]).T.astype(np.float64)
        if bd is not None:
            d, s = d + bd[n], s + np.abs(bd[n])
        w = wts[tok, j].astype(np.float64)[:, None]
        want[tok] += w * d
        size[tok] += w * s
    return want, size


def check_moe(ctx, t, h, i, e, k, logits, bias, seed):
    rng, x, _, ups, downs = moe_case(ctx, t, h, i, e, k, seed)
    bu, bd = (R.grid_matrix(rng, e, i, 0), R.grid_matrix(rng, e, h, 0)) if bias else (None, None)
    du, dd = tile_all(ctx, ups), tile_all(ctx, downs)
    dbu, dbd = (ctx.upload(bu), ctx.upload(bd)) if bias else (None, None)
    biases = C.byref(NH.MoeBiases(dbu.ptr, dbd.ptr, None, None)) if bias else None
    got, st = moe(ctx, x, logits, du, dd, h, i, k, biases)
    want, size = moe_want(x, logits, ups, downs, k, bu, bd)
    assert st == NH.OK
    # i products, eight parts, a bias; the weight's product and the sum over the routes
    assert (np.abs(got - want) <= (i + 10 + 2 * k) * U * size).all()


# Two units of h (its one K tile has four) and three of the output in an expert's run, eight groups on them.
@pytest.mark.parametrize("t,h,i,e,k", [(2, 40, 50, 4, 2), (20, 48, 130, 200, 1)])
def test_expert_bias_of_groups_without_a_unit(ctx, t, h, i, e, k):
    note(f"moe bias, idle groups t={t} h={h} i={i}")
    logits = np.random.default_rng(t).standard_normal((t, e)).astype(np.float32)
    check_moe(ctx, t, h, i, e, k, logits, True, t + 1)


# More tokens than a grid's 16 bits; the mean expert has 32 parts of its rows to give out, and each takes many passes.
def test_experts_of_many_tokens(ctx):
    t, h, i, e, k = 70001, 40, 36, 2, 1
    note(f"moe t={t}")
    logits = np.random.default_rng(8).standard_normal((t, e)).astype(np.float32)
    check_moe(ctx, t, h, i, e, k, logits, False, 8)


@pytest.mark.parametrize("hidden,bf16", [(40, False), (40, True), (9, True), (9, False)])
@pytest.mark.parametrize("with_shared", [False, True])
def test_combine_of_many_tokens(ctx, hidden, bf16, with_shared):
    note(f"combine of 140001 tokens hidden={hidden} bf16={bf16} shared={with_shared}")
    t, k = 140001, 2
    rng = np.random.default_rng(hidden)
    d, w = rng.standard_normal((t * k, hidden), dtype=np.float32), rng.standard_normal((t, k), dtype=np.float32)
    shared = rng.standard_normal((t, hidden), dtype=np.float32)
    pos = rng.permutation(t * k).astype(np.int32).reshape(t, k)
    pos[[5, 65535, 139999], 1] = -1  # dropped routes
    dev = [ctx.upload(v) for v in (d, pos, w, shared)]
    out = Guarded(ctx, (t, hidden), np.uint16 if bf16 else np.float32)
    NH.call("nh_moe_combine_shared", ctx.handle, dev[0].ptr, dev[1].ptr, dev[2].ptr, dev[3].ptr if with_shared else None, t, k,
            hidden, out.ptr, NH.BF16 if bf16 else NH.F32, None)
    ctx.synchronize()
    want = shared.copy() if with_shared else np.zeros((t, hidden), np.float32)
    for j in range(k):
        want = np.where(pos[:, j:j + 1] < 0, want, want + w[:, j:j + 1] * d[pos[:, j]])
    assert np.array_equal(out.numpy(), R.to_bf16_bits(want) if bf16 else want)


# The launches are dealt for evenly spread routes; here every token agrees on the same experts, the mean expert has
# several passes of rows (t = 300), or none is compacted away (128 experts, six of them with routes).
@pytest.mark.parametrize("t,h,i,e,k,liked", [(300, 136, 70, 8, 2, (3, 5)), (300, 136, 70, 8, 2, (0, 7)),
                                             (100, 128, 64, 128, 6, (1, 2, 64, 65, 126, 127)), (700, 160, 96, 4, 1, (3,)),
                                             (20, 64, 40, 16, 3, (0, 1, 15)), (33, 4200, 36, 6, 1, (2,))])
def test_experts_of_routes_that_agree(ctx, t, h, i, e, k, liked):
    note(f"moe skew t={t} e={e} k={k} liked={liked}")
    logits = np.random.default_rng(t + e).standard_normal((t, e)).astype(np.float32)
    logits[:, list(liked)] += 20
    check_moe(ctx, t, h, i, e, k, logits, True, t)
