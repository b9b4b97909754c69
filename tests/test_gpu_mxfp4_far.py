"""MXFP4 and balance calls whose arrays pass 2^31 elements or 4 GiB, and the longest K: all zeros but for the far end."""
import numpy as np
import pytest

import mx_reference as R
import nemotron_hip as NH
from test_gpu_mxfp4 import U, note, route, run_linear, weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = NH.Context(0)
    yield c
    c.close()


def zeros(ctx, shape, dtype, free):
    b = ctx.empty(shape, dtype)
    free.append(b)
    b.fill_bytes(0)
    return b


def put(ctx, buf, at, array):
    array = np.ascontiguousarray(array)
    assert at >= 0 and at + array.nbytes <= buf.nbytes
    NH.call("nh_memcpy_htod", ctx.handle, buf.ptr + at, array.ctypes.data, array.nbytes)


def get(ctx, buf, at, shape, dtype):
    out = np.empty(shape, dtype)
    assert at >= 0 and at + out.nbytes <= buf.nbytes
    NH.call("nh_memcpy_dtoh", ctx.handle, out.ctypes.data, buf.ptr + at, out.nbytes)
    return out


@pytest.fixture
def free():
    buffers = []
    yield buffers
    for b in buffers:
        b.free()


@pytest.mark.parametrize("rows,cols", [(1100, 1 << 21), (33_000_000, 65), ((1 << 30) + 5, 1)])
def test_conversions(ctx, free, rows, cols):
    note(f"far conversions {rows} x {cols}")
    rng = np.random.default_rng(0)
    last = R.to_bf16_bits(rng.standard_normal((3, cols)))
    x = zeros(ctx, (rows, cols), np.uint16, free)
    codes, scales = zeros(ctx, (rows, -(-cols // 2)), np.uint8, free), zeros(ctx, (rows, -(-cols // 32)), np.uint8, free)
    put(ctx, x, x.nbytes - last.nbytes, last)
    NH.call("nh_quantize_rows_mxfp4", ctx.handle, x.ptr, NH.BF16, rows, cols, codes.ptr, scales.ptr, None, None)
    ctx.synchronize()
    rc, rs, rv = R.quantize(R.from_bf16_bits(last))
    assert np.array_equal(get(ctx, codes, codes.nbytes - rc.nbytes, rc.shape, np.uint8), rc)
    assert np.array_equal(get(ctx, scales, scales.nbytes - rs.nbytes, rs.shape, np.uint8), rs)
    assert (get(ctx, scales, scales.nbytes - rs.nbytes - 64, 64, np.uint8) == 0).all()
    x.fill_bytes(0xFF)
    NH.call("nh_dequantize_mxfp4", ctx.handle, codes.ptr, scales.ptr, rows, cols, x.ptr, NH.BF16, None)
    ctx.synchronize()
    assert np.array_equal(R.from_bf16_bits(get(ctx, x, x.nbytes - last.nbytes, last.shape, np.uint16)), rv.astype(np.float32))
    assert (get(ctx, x, x.nbytes - last.nbytes - 256, 128, np.uint16) == 0).all()


@pytest.mark.parametrize("m", [2, 40])
def test_linear_of_far_weights(ctx, free, m):
    n, k = 600_000, 16384  # 5.2 GB of weights
    note(f"far weights m={m}")
    rng = np.random.default_rng(m)
    x, w = R.grid_matrix(rng, m, k, 0).astype(np.float32), R.grid_matrix(rng, 16, k, 0)
    codes, scales, _ = R.quantize(w)
    piece = R.tile(codes, scales, 16, k)
    tiled = zeros(ctx, NH.lib().nh_tiled_mxfp4_weights_bytes(n, k), np.uint8, free)
    mid = (1 << 32) // piece.size + 1  # the first row tile past 4 GiB
    put(ctx, tiled, mid * piece.size, piece)
    put(ctx, tiled, tiled.nbytes - piece.size, piece)
    out = zeros(ctx, (m, n), np.float32, free)
    out.fill_bytes(0xFF)
    need = NH.lib().nh_linear_mxfp4_workspace_size(m, n, k)
    ws, dx = zeros(ctx, max(need, 16), np.uint8, free), ctx.upload(x)
    NH.call("nh_linear_mxfp4", ctx.handle, dx.ptr, NH.F32, tiled.ptr, None, m, n, k, out.ptr, NH.F32, ws.ptr, need, None, None)
    ctx.synchronize()
    want = np.zeros((m, n), np.float32)
    want[:, mid * 16:mid * 16 + 16] = want[:, n - 16:] = x @ w.T  # sums of quarters below 2^22
    assert np.array_equal(out.numpy(), want)


@pytest.mark.parametrize("m,n,k", [(140_001, 16, 16384), (70_001, 32768, 128)])
def test_linear_of_far_rows(ctx, free, m, n, k):
    """Rows, or outputs, of more than 2^31 elements."""
    note(f"far rows m={m} n={n} k={k}")
    rng = np.random.default_rng(n)
    last, w = R.grid_matrix(rng, 5, k, 0), R.grid_matrix(rng, n, k, 0)
    tiled, _ = weights(ctx, w)
    free.append(tiled)
    x, out = zeros(ctx, (m, k), np.uint16, free), zeros(ctx, (m, n), np.uint16, free)
    out.fill_bytes(0xFF)
    put(ctx, x, x.nbytes - 5 * k * 2, R.to_bf16_bits(last))
    need = NH.lib().nh_linear_mxfp4_workspace_size(m, n, k)
    ws = zeros(ctx, need, np.uint8, free)
    NH.call("nh_linear_mxfp4", ctx.handle, x.ptr, NH.BF16, tiled.ptr, None, m, n, k, out.ptr, NH.BF16, ws.ptr, need, None, None)
    ctx.synchronize()
    got = get(ctx, out, out.nbytes - 8 * n * 2, (8, n), np.uint16)
    assert (got[:3] == 0).all() and np.array_equal(got[3:], R.to_bf16_bits(last.astype(np.float32) @ w.T.astype(np.float32)))


@pytest.mark.parametrize("m,n,k", [(3, 40, 131072), (40, 33, 131071), (70, 130, 100_000)])
def test_linear_of_the_longest_rows(ctx, m, n, k):
    """Sums of quarters far below 2^22 (131072 products of random sign): exact."""
    note(f"long K m={m} n={n} k={k}")
    rng = np.random.default_rng(k)
    x, w = R.grid_matrix(rng, m, k, 0), R.grid_matrix(rng, n, k, 0)
    tiled, _ = weights(ctx, w)
    assert np.array_equal(run_linear(ctx, x, tiled, n), (x.astype(np.float64) @ w.T.astype(np.float64)).astype(np.float32))


def test_far_experts(ctx, free):
    """1024 experts of 4096 x 2048: 4.8 GB up and down each; the routes go to the last two."""
    t, h, i, e, k = 9, 4096, 2048, 1024, 2
    note("far experts")
    rng = np.random.default_rng(3)
    x, logits = R.grid_matrix(rng, t, h, 0).astype(np.float32), rng.standard_normal((t, e)).astype(np.float32)
    logits[:, -2:] += 9
    idx, wts = route(logits, k, 0, 1.0)
    ups, downs = [R.grid_matrix(rng, i, h, 0) for _ in range(2)], [R.grid_matrix(rng, h, i, 0) for _ in range(2)]
    bufs = []
    for ws, (n, c) in ((ups, (i, h)), (downs, (h, i))):
        size = NH.lib().nh_tiled_mxfp4_weights_bytes(n, c)
        buf = zeros(ctx, e * size, np.uint8, free)
        assert buf.nbytes > 1 << 32
        for j, w in enumerate(ws):
            put(ctx, buf, (e - 2 + j) * size, R.tile(*R.quantize(w)[:2], n, c))
        bufs.append(buf)
    need = NH.lib().nh_moe_forward_mxfp4_workspace_size(t, h, i, e, k)
    ws, dx, dl, out = zeros(ctx, need, np.uint8, free), ctx.upload(x), ctx.upload(logits), ctx.empty((t, h), np.float32)
    NH.call("nh_moe_forward_mxfp4", ctx.handle, dx.ptr, NH.F32, dl.ptr, t, h, i, e, k, 0, 1.0, bufs[0].ptr, bufs[1].ptr, None,
            None, out.ptr, NH.F32, ws.ptr, need, None, None)
    ctx.synchronize()
    want, size = np.zeros((t, h)), np.zeros((t, h))
    for a in range(t):
        for j in range(k):
            n = idx[a, j] - (e - 2)
            assert n >= 0
            hv = R.quantize((np.maximum(x[a] @ ups[n].T, 0) ** 2).astype(np.float32).reshape(1, -1))[2][0]
            want[a] += wts[a, j].astype(np.float64) * (downs[n] @ hv)
            size[a] += wts[a, j].astype(np.float64) * (np.abs(downs[n]) @ np.abs(hv))
    assert (np.abs(out.numpy() - want) <= (i + 10 + 2 * k) * U * size).all()


def test_far_balance(ctx, free):
    """2^31 + 2^21 logits: uniform rows of 1024 experts (p = 2^-10, exactly), the last one with expert 5 alone."""
    t, e = (1 << 21) + (1 << 11), 1024
    note("far balance")
    z, grad = zeros(ctx, (t, e), np.float32, free), zeros(ctx, (t, e), np.float32, free)
    idx = zeros(ctx, (t, 1), np.int32, free)
    last = np.full(e, -np.inf, np.float32)
    last[5] = 0
    put(ctx, z, z.nbytes - last.nbytes, last)
    put(ctx, idx, idx.nbytes - 4, np.array([5], np.int32))
    counts, loss, up = ctx.empty((1, e), np.int32), ctx.empty(1, np.float32), ctx.upload(np.array([float(t)], np.float32))
    need = NH.lib().nh_moe_balance_loss_workspace_size(1, t, e)
    ws = zeros(ctx, need, np.uint8, free)
    NH.call("nh_moe_balance_loss", ctx.handle, z.ptr, idx.ptr, None, 1, t, e, 1, 1, 1.0, counts.ptr, loss.ptr, ws.ptr, need, None)
    grad.fill_bytes(0xFF)
    NH.call("nh_moe_balance_loss_backward", ctx.handle, z.ptr, counts.ptr, None, 1, t, e, 1, 1, 1.0, up.ptr, grad.ptr, None)
    ctx.synchronize()
    got = counts.numpy()[0]
    assert got[0] == t - 1 and got[5] == 1 and got.sum() == t
    f = got * (e / t)
    rows = get(ctx, grad, grad.nbytes - 2 * last.nbytes, (2, e), np.float32)
    p = np.full(e, 1 / e)
    # f has a rounding of its factor and one of the product, f p two more and the sum of two terms, the gradient three
    assert (np.abs(rows[0] - p * (f - f @ p)) <= 8 * U * p * f.max()).all()
    assert np.abs(rows[1]).max() <= 4 * U * f.max()  # p_5 (f_5 - f_5), and 0 elsewhere
    sums = np.full(e, (t - 1) / e)
    sums[5] += 1
    want = e / t / t * float(got.astype(np.float64) @ sums)
    # whole multiples of 2^-10 in a lane's sum of up to 8200 / 16 rows: exact; the loss is rounded once
    assert abs(float(loss.numpy()[0]) - want) <= 2 * U * want
