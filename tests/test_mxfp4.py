"""MXFP4 and the router's balance loss without a GPU: the host twins against plain 64-bit forms, the refusals of the
device entry points, and which kernels a call launches."""
import ctypes as C
import os
import re

import numpy as np
import pytest

import mx_reference as R
import nemotron_hip as NH
import test_gpu_mxfp4 as G
from dispatch import BIAS, OUT, S, W, W2, WS, X, Recorder


@pytest.fixture(scope="module")
def rec():
    r = Recorder()
    yield r
    r.close()


def quantize_host(x, dtype=NH.F32):
    rows, cols = x.shape
    codes = np.zeros((rows, -(-cols // 2)), np.uint8)
    scales = np.zeros((rows, -(-cols // 32)), np.uint8)
    NH.call("nh_quantize_rows_mxfp4_host", x.ctypes.data, dtype, rows, cols, codes.ctypes.data, scales.ctypes.data)
    return codes, scales


def tile_host(codes, scales, n, k):
    out = np.empty(NH.lib().nh_tiled_mxfp4_weights_bytes(n, k), np.uint8)
    NH.call("nh_tile_weights_mxfp4_host", codes.ctypes.data, scales.ctypes.data, n, k, out.ctypes.data, out.size)
    return out


def edge_rows(rng, cols):
    """Rows of every magnitude: zeros, subnormals, the largest values, ties of every grid step."""
    rows = [np.zeros(cols), -np.zeros(cols), rng.standard_normal(cols), rng.standard_normal(cols) * 1e-38,
            rng.integers(-8, 9, cols) * 2.0 ** -149, rng.choice([3.4028234663852886e38, -1e38, 1.0], cols)]
    for e in (-149, -130, -127, -126, -125, -20, 0, 100, 125):
        tie = rng.choice(R.MIDDLE, cols) * 2.0 ** e * rng.choice([-1, 1], cols)
        tie[::32] = 4 * 2.0 ** e
        rows += [tie, np.nextafter(tie.astype(np.float32), np.float32(0)), np.nextafter(tie.astype(np.float32), np.float32(np.inf))]
    return np.array(rows).astype(np.float32)


@pytest.mark.parametrize("cols", [1, 2, 31, 32, 33, 64, 97, 128, 130, 640])
def test_quantize_host_is_the_definition(cols):
    x = edge_rows(np.random.default_rng(cols), cols)
    codes, scales = quantize_host(x)
    rc, rs, rv = R.quantize(x)
    assert np.array_equal(scales, rs) and np.array_equal(codes, rc)
    for dtype, np_dtype in ((NH.F32, np.uint32), (NH.BF16, np.uint16)):
        out = np.empty(x.shape, np_dtype)
        NH.call("nh_dequantize_mxfp4_host", codes.ctypes.data, scales.ctypes.data, *x.shape, out.ctypes.data, dtype)
        want = rv.astype(np.float32).view(np.uint32)
        assert np.array_equal(out, want if dtype == NH.F32 else (want >> 16).astype(np.uint16))  # two bits: exact in bf16


def test_quantize_host_of_bf16_rows_and_bad_values():
    rng = np.random.default_rng(0)
    b = R.to_bf16_bits(rng.standard_normal((5, 77)) * 100)
    codes, scales = quantize_host(b, NH.BF16)
    rc, rs, _ = R.quantize(R.from_bf16_bits(b))
    assert np.array_equal(codes, rc) and np.array_equal(scales, rs)
    for bad in (np.nan, np.inf, -np.inf):
        x = rng.standard_normal((3, 40)).astype(np.float32)
        x[1, 33] = x[2, 0] = bad
        codes = np.full((3, 20), 7, np.uint8)
        st, err = NH.call_status("nh_quantize_rows_mxfp4_host", x.ctypes.data, NH.F32, 3, 40, codes.ctypes.data,
                                 codes.ctypes.data)
        assert st == NH.NON_FINITE_INPUT and err.index == 73 and (codes == 7).all()


def test_dequantize_host_of_every_code_and_scale():
    codes = np.tile(np.arange(256, dtype=np.uint8), (16, 1)).reshape(256, 16)
    codes = np.tile(codes, (16, 1))  # 4096 blocks: 16 code rows x 256 scales
    scales = np.repeat(np.arange(256, dtype=np.uint8), 16).reshape(-1, 1)
    out = np.empty((4096, 32), np.float32)
    NH.call("nh_dequantize_mxfp4_host", codes.ctypes.data, scales.ctypes.data, 4096, 32, out.ctypes.data, NH.F32)
    with np.errstate(over="ignore"):
        want = R.decode(codes, scales, 32).astype(np.float32)
    assert np.array_equal(out, want, equal_nan=True)


@pytest.mark.parametrize("n,k", [(1, 1), (16, 128), (17, 129), (5, 500), (33, 512), (40, 513), (16, 1023)])
def test_tile_host_is_the_documented_layout(n, k):
    rng = np.random.default_rng(n * 1000 + k)
    codes, scales, _ = R.quantize(rng.standard_normal((n, k)))
    assert np.array_equal(tile_host(codes, scales, n, k), R.tile(codes, scales, n, k))
    assert NH.lib().nh_tiled_mxfp4_weights_bytes(n, k) == R.tile(codes, scales, n, k).size


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (3, 18, 33), (2, 33, 300), (5, 16, 128)])
def test_linear_host(m, n, k):
    rng = np.random.default_rng(k)
    x, w = rng.standard_normal((m, k)).astype(np.float32), rng.standard_normal((n, k))
    bias = rng.standard_normal(n).astype(np.float32)
    codes, scales, wv = R.quantize(w)
    tiled = tile_host(codes, scales, n, k)
    out = np.empty((m, n), np.float32)
    NH.call("nh_linear_mxfp4_host", x.ctypes.data, NH.F32, tiled.ctypes.data, bias.ctypes.data, m, n, k, out.ctypes.data,
            NH.F32)
    xv = R.quantize(x)[2]
    # a sum in 64 bits, rounded to 32, and the bias added in 32: two half steps
    y = xv @ wv.T
    assert (np.abs(out - (y + bias)) <= 2.0 ** -24 * (np.abs(y) + np.abs(y + bias)) * (1 + 1e-6)).all()
    x[0, k - 1] = np.inf
    st, err = NH.call_status("nh_linear_mxfp4_host", x.ctypes.data, NH.F32, tiled.ctypes.data, None, m, n, k,
                             out.ctypes.data, NH.F32)
    assert st == NH.NON_FINITE_INPUT and err.argument == b"input" and err.index == k - 1


def test_moe_host_is_its_stages():
    """Routing, the experts as host linears, ReLU^2 in f32, and the combine, put together by hand."""
    t, h, i, e, k = 5, 96, 70, 6, 2
    rng = np.random.default_rng(1)
    x, logits = rng.standard_normal((t, h)).astype(np.float32), rng.standard_normal((t, e)).astype(np.float32)
    wu, wd = [R.quantize(rng.standard_normal((i, h))) for _ in range(e)], [R.quantize(rng.standard_normal((h, i))) for _ in range(e)]
    tu, td = [tile_host(*w[:2], i, h) for w in wu], [tile_host(*w[:2], h, i) for w in wd]
    bu, bd = rng.standard_normal((e, i)).astype(np.float32), rng.standard_normal((e, h)).astype(np.float32)
    shared = rng.standard_normal((t, h)).astype(np.float32)
    idx, wts = np.empty((t, k), np.int32), np.empty((t, k), np.float32)
    NH.call("nh_moe_route_sigmoid_topk_host", logits.ctypes.data, t * e, t, e, k, 1, 2.5, idx.ctypes.data, t * k,
            wts.ctypes.data, t * k)
    want = shared.copy()
    for a in range(t):
        for j in range(k):
            n = idx[a, j]
            y, d = np.empty((1, i), np.float32), np.empty((1, h), np.float32)
            NH.call("nh_linear_mxfp4_host", x[a:a + 1].ctypes.data, NH.F32, tu[n].ctypes.data, bu[n].ctypes.data, 1, i, h,
                    y.ctypes.data, NH.F32)
            y = np.maximum(y, 0) ** 2
            NH.call("nh_linear_mxfp4_host", y.ctypes.data, NH.F32, td[n].ctypes.data, bd[n].ctypes.data, 1, h, i,
                    d.ctypes.data, NH.F32)
            want[a] = want[a] + wts[a, j] * d[0]
    up, down = np.concatenate(tu), np.concatenate(td)
    out = np.empty((t, h), np.float32)
    biases = NH.MoeBiases(bu.ctypes.data, bd.ctypes.data, None, None)
    NH.call("nh_moe_forward_mxfp4_host", x.ctypes.data, NH.F32, logits.ctypes.data, t, h, i, e, k, 1, 2.5, up.ctypes.data,
            down.ctypes.data, C.byref(biases), shared.ctypes.data, out.ctypes.data, NH.F32)
    assert np.array_equal(out, want)


BALANCE = [(1, 1, 1, None), (7, 8, 2, None), (40, 16, 3, [0, 10, 10, 33, 40]), (40, 60, 6, [0, 1, 30]), (9, 5, 1, [3, 9])]


@pytest.mark.parametrize("t,e,k,seq", BALANCE)
@pytest.mark.parametrize("softmax", [0, 1])
def test_balance_host(t, e, k, seq, softmax):
    rng = np.random.default_rng(t * e + softmax)
    z = (rng.standard_normal((t, e)) * 3).astype(np.float32)
    z[0] -= 300.0  # sigmoids that all vanish
    if t > 4:
        z[2], z[3, 1:] = -np.inf, -np.inf
    idx = np.array([rng.permutation(e)[:k] for _ in range(t)], np.int32)
    if t > 4:
        idx[1, 0], idx[4, 0] = -1, e
    counts, loss, grad = balance_host(z, idx, seq, softmax, 0.5, 1.5)
    rc, rl, rg = R.balance(z, idx, seq, softmax, 0.5, 1.5)
    assert np.array_equal(counts, rc)
    assert abs(loss - rl) <= 2.0 ** -23 * abs(rl)  # 64-bit sums, one rounding (and the reference's own order)
    assert (np.abs(grad - rg) <= 2.0 ** -22 * np.abs(rg) + 1e-12 * np.abs(rg).max()).all()


def balance_host(z, idx, seq, softmax, coefficient, dloss):
    t, e = z.shape
    off = None if seq is None else np.array(seq, np.int32)
    s = 1 if seq is None else len(seq) - 1
    po = None if off is None else off.ctypes.data
    counts, loss, grad = np.empty((s, e), np.int32), np.empty(1, np.float32), np.empty((t, e), np.float32)
    up = np.array([dloss], np.float32)
    NH.call("nh_moe_balance_loss_host", z.ctypes.data, idx.ctypes.data, po, s, t, e, idx.shape[1], softmax, coefficient,
            counts.ctypes.data, loss.ctypes.data)
    NH.call("nh_moe_balance_loss_backward_host", z.ctypes.data, counts.ctypes.data, po, s, t, e, idx.shape[1], softmax,
            coefficient, up.ctypes.data, grad.ctypes.data)
    return counts, loss[0], grad


@pytest.mark.parametrize("softmax", [0, 1])
def test_balance_reference_gradient_against_differences(softmax):
    rng = np.random.default_rng(3)
    z, seq = rng.standard_normal((9, 6)) * 2, [0, 4, 9]
    idx = np.array([rng.permutation(6)[:2] for _ in range(9)], np.int32)
    _, _, grad = R.balance(z, idx, seq, softmax, 0.7)
    step = 1e-5
    for row, col in np.ndindex(z.shape):
        up, down = z.copy(), z.copy()
        up[row, col] += step
        down[row, col] -= step
        slope = (R.balance(up, idx, seq, softmax, 0.7)[1] - R.balance(down, idx, seq, softmax, 0.7)[1]) / (2 * step)
        # central differences: third derivative (below 1 here) * step^2 / 6, and rounding 2^-52 / step
        assert abs(slope - grad[row, col]) < 1e-9


# ---- refusals, before any device is touched ------------------------------------

def test_refusals():
    q = lambda **a: NH.call_status("nh_quantize_rows_mxfp4", None, X, a.get("d", NH.F32), a.get("r", 4), a.get("c", 64), OUT,  # noqa: E731
                                   S, None, None)[0]
    assert q(d=5) == NH.INVALID_PARAMS and q(r=1 << 31) == NH.UNSUPPORTED and q(c=1 << 31) == NH.UNSUPPORTED
    assert q(r=1 << 40, c=1 << 40) == NH.INVALID_SHAPE and q() == NH.INVALID_PARAMS  # no context
    t = lambda n, k, size, at=OUT: NH.call_status("nh_tile_weights_mxfp4", None, X, S, n, k, at, size, None)  # noqa: E731
    assert t(0, 4, 0)[0] == t(4, 0, 0)[0] == NH.INVALID_SHAPE
    st, err = t(16, 128, 1024)
    assert st == NH.LENGTH_MISMATCH and (err.argument, err.expected) == (b"tiled", 1280)
    assert t(16, 128, 1280, OUT + 8)[0] == NH.UNSUPPORTED
    assert NH.lib().nh_tiled_mxfp4_weights_bytes(0, 5) == 0 == NH.lib().nh_tiled_mxfp4_weights_bytes(5, 0)
    assert NH.lib().nh_tiled_mxfp4_weights_bytes(1 << 40, 1 << 40) == 0


def linear_status(m=4, n=64, k=256, xd=NH.BF16, od=NH.BF16, w=W, ws=WS, ws_bytes=None, x=X, out=OUT):
    if ws_bytes is None:
        ws_bytes = NH.lib().nh_linear_mxfp4_workspace_size(m, n, k)
    return NH.call_status("nh_linear_mxfp4", None, x, xd, w, None, m, n, k, out, od, ws, ws_bytes, None, None)


def test_linear_refusals():
    assert linear_status(n=0)[0] == linear_status(k=0)[0] == NH.INVALID_SHAPE
    assert linear_status(m=0)[0] == NH.INVALID_ROW_COUNT
    assert linear_status(xd=3)[0] == linear_status(od=-1)[0] == NH.INVALID_PARAMS
    assert linear_status(k=(1 << 17) + 1)[0] == linear_status(m=1 << 24)[0] == linear_status(n=1 << 28)[0] == NH.UNSUPPORTED
    assert linear_status(w=W + 8)[0] == NH.UNSUPPORTED
    need = NH.lib().nh_linear_mxfp4_workspace_size(20, 64, 256)
    st, err = linear_status(m=20, ws_bytes=need - 1)
    assert st == NH.LENGTH_MISMATCH and (err.argument, err.expected, err.actual) == (b"workspace", need, need - 1)
    assert linear_status(m=20, ws=None)[0] == NH.LENGTH_MISMATCH and linear_status(m=20, ws=WS + 4)[0] == NH.UNSUPPORTED
    assert linear_status(out=X)[0] == NH.INVALID_PARAMS  # over its own rows
    assert linear_status(out=X + 4 * 256 * 2 - 2)[0] == NH.INVALID_PARAMS
    assert linear_status(out=X + 4 * 256 * 2)[1].message == b"null context"
    assert NH.lib().nh_linear_mxfp4_workspace_size(16, 64, 16384) == 0 < NH.lib().nh_linear_mxfp4_workspace_size(1, 64, 16385)


def test_moe_refusals():
    def moe(t=4, h=64, i=32, e=8, k=2, biases=None, ws=WS, ws_bytes=None, up=W, xd=NH.BF16, od=NH.BF16):
        if ws_bytes is None:
            ws_bytes = NH.lib().nh_moe_forward_mxfp4_workspace_size(t, h, i, e, k)
        return NH.call_status("nh_moe_forward_mxfp4", None, X, xd, S, t, h, i, e, k, 1, 1.0, up, W2, biases, None, OUT, od, ws,
                              ws_bytes, None, None)
    assert moe(t=0)[0] == NH.INVALID_ROW_COUNT
    assert all(moe(**{v: 0})[0] == NH.INVALID_SHAPE for v in "hiek") and moe(k=9)[0] == NH.INVALID_SHAPE
    assert moe(xd=2)[0] == moe(od=2)[0] == NH.INVALID_PARAMS
    assert moe(h=8193)[0] == moe(i=8193)[0] == moe(e=1025)[0] == moe(e=100, k=65)[0] == NH.UNSUPPORTED
    assert moe(ws=None)[0] == NH.LENGTH_MISMATCH and moe(ws_bytes=100)[0] == NH.LENGTH_MISMATCH
    assert moe(up=W + 4)[0] == moe(ws=WS + 8)[0] == NH.UNSUPPORTED
    assert moe(biases=C.byref(NH.MoeBiases(None, None, BIAS, None)))[0] == NH.INVALID_PARAMS
    assert moe()[1].message == b"null context"


def test_balance_refusals():
    def both(s=1, t=64, e=8, k=2, c=0.1, seq=S, ws_bytes=None):
        if ws_bytes is None:
            ws_bytes = NH.lib().nh_moe_balance_loss_workspace_size(s, t, e)
        a = NH.call_status("nh_moe_balance_loss", None, X, W, seq, s, t, e, k, 0, c, OUT, BIAS, WS, ws_bytes, None)
        b = NH.call_status("nh_moe_balance_loss_backward", None, X, W, seq, s, t, e, k, 0, c, BIAS, OUT, None)
        return a[0], b[0], a[1].message, b[1].message
    for args, want in (({"e": 0}, NH.INVALID_SHAPE), ({"k": 0}, NH.INVALID_SHAPE), ({"s": 0}, NH.INVALID_SHAPE),
                       ({"s": 2, "seq": None}, NH.INVALID_SHAPE), ({"c": float("nan")}, NH.INVALID_PARAMS),
                       ({"c": float("inf")}, NH.INVALID_PARAMS), ({"e": 1025}, NH.UNSUPPORTED), ({"t": 1 << 30}, NH.UNSUPPORTED)):
        assert both(**args)[:2] == (want, want), args
    assert both(ws_bytes=16)[0] == NH.LENGTH_MISMATCH
    assert both()[2:] == (b"null context",) * 2


# ---- dispatch -----------------------------------------------------------------

def mx_kernels(rec, m, n, k, x_dtype=NH.BF16):
    ws = NH.lib().nh_linear_mxfp4_workspace_size(m, n, k)
    return rec.launches("nh_linear_mxfp4", X, x_dtype, W, BIAS, m, n, k, OUT, NH.F32, WS if ws else None, ws, None, None)


def test_linear_without_a_workspace_is_one_launch(rec):
    for k in (1, 1024, 1025, 4096, 8192, 16384):
        for m in (1, 16):
            assert len(mx_kernels(rec, m, 4096, k)) == 1
    assert [v[0] for v in mx_kernels(rec, 17, 4096, 4096)][0] == "quantize_mxfp4_tiles"


def moe_launches(rec, t, h, i, e, k):
    ws = NH.lib().nh_moe_forward_mxfp4_workspace_size(t, h, i, e, k)
    return rec.launches("nh_moe_forward_mxfp4", X, NH.F32, S, t, h, i, e, k, 1, 1.0, W, W2, None, None, OUT, NH.F32, WS, ws, None,
                        None)


def test_every_kernel_is_reached_by_the_device_tests(rec):
    """The products' and the layer's shapes of the device tests launch every MXFP4 kernel between them."""
    seen = {v[0] for m, n, k in G.LINEAR for dt in (NH.F32, NH.BF16) for v in mx_kernels(rec, m, n, k, dt)}
    seen |= {v[0] for shape in G.MOE for v in moe_launches(rec, *shape)}
    src = open(os.path.join(os.path.dirname(NH.__file__), "csrc", "runtime", "context.cpp")).read()
    names = set(re.findall(r'"nh_(mx_\w+)_kernel"', src))
    assert len(names) > 25 and names <= seen, names - seen


# Tiles by the rounds they take (launch_mx_gemm): large ones where they fill the chip, small ones where K is long and they do not.
@pytest.mark.parametrize("m,n,k,tile,grid", [(2048, 21504, 4096, "256x256", 256), (8192, 8192, 8192, "256x256", 256),
                                             (2048, 4096, 4096, "128x128", 512), (300, 4096, 8192, "64x64", 320),
                                             (65, 64, 512, "64x64", 2), (1 << 23, 16, 128, "64x64", 512)])
def test_gemm_tiles(rec, m, n, k, tile, grid):
    assert mx_kernels(rec, m, n, k)[-1] == (f"mx_gemm_{tile}", grid, 1)


# Each pass of an expert's rows has a workgroup of its own where the mean expert has several; a round of the 256 CUs at most.
@pytest.mark.parametrize("shape", [(8, 2048, 1792, 128, 6), (500, 2688, 1856, 128, 6), (700, 4096, 1792, 8, 2), (1, 4096, 1792, 8, 2)])
def test_moe_workgroups(rec, shape):
    for name, gx, gy in moe_launches(rec, *shape):
        if name.startswith("mx_stream"):
            assert gx * min(gy, shape[0] * shape[4]) <= 256


# One workgroup for few logits of one sequence, else a chunk per workgroup and a workgroup per sequence.
def test_balance_launches(rec):
    def launches(t, e, s=1, seq=None):
        ws = NH.lib().nh_moe_balance_loss_workspace_size(s, t, e)
        a = rec.launches("nh_moe_balance_loss", X, W, seq, s, t, e, 2, 0, 0.1, OUT, BIAS, WS, ws, None)
        b = rec.launches("nh_moe_balance_loss_backward", X, OUT, seq, s, t, e, 2, 0, 0.1, BIAS, OUT, None)
        return a, [v[0] for v in b]
    back = ["moe_balance_backward"]
    assert launches(256, 128) == ([("moe_balance_partial", 1, 1)], back)
    assert launches(257, 128) == ([("moe_balance_partial", 5, 1), ("moe_balance_reduce", 1, 1)], back)
    assert launches(64, 128, 3, S) == ([("moe_balance_partial", 4, 1), ("moe_balance_reduce", 3, 1)], back)
    assert launches(131072, 128) == ([("moe_balance_partial", 257, 1), ("moe_balance_reduce", 1, 1)], back)


def test_null_operands_are_refused(rec):
    """Found before a launch: on a recording context, which would note it."""
    def refused(name, args, operands):
        for at in operands:
            st, err = NH.call_status(name, rec.ctx, *(None if i == at else v for i, v in enumerate(args)))
            assert st == NH.INVALID_PARAMS and err.message == b"null operand", (name, at)
        assert NH.call_status(name, rec.ctx, *args)[0] == NH.OK
    ws = NH.lib().nh_moe_forward_mxfp4_workspace_size(4, 64, 32, 8, 2)
    bws = NH.lib().nh_moe_balance_loss_workspace_size(1, 64, 8)
    refused("nh_quantize_rows_mxfp4", (X, NH.F32, 4, 64, OUT, S, None, None), (0, 4, 5))
    refused("nh_dequantize_mxfp4", (X, S, 4, 64, OUT, NH.F32, None), (0, 1, 4))
    refused("nh_linear_mxfp4", (X, NH.F32, W, None, 4, 64, 256, OUT, NH.F32, None, 0, None, None), (0, 2, 7))
    refused("nh_moe_forward_mxfp4", (X, NH.F32, S, 4, 64, 32, 8, 2, 1, 1.0, W, W2, None, None, OUT, NH.F32, WS, ws, None, None),
            (0, 2, 10, 11, 14))
    refused("nh_moe_balance_loss", (X, W, None, 1, 64, 8, 2, 0, 0.1, OUT, BIAS, WS, bws, None), (0, 1, 9, 10))
    refused("nh_moe_balance_loss_backward", (X, W, None, 1, 64, 8, 2, 0, 0.1, BIAS, OUT, None), (0, 1, 9, 10))
    assert NH.call_status("nh_moe_balance_loss", rec.ctx, None, None, None, 1, 0, 8, 2, 0, 0.1, OUT, BIAS, WS, bws, None)[0] == NH.OK


def test_many_sequences_are_refused(rec):
    """Every workgroup walks the offsets."""
    size = NH.lib().nh_moe_balance_loss_workspace_size
    assert size(16384, 1 << 20, 128) > 0 == size(16385, 1 << 20, 128)
    st, _ = NH.call_status("nh_moe_balance_loss", rec.ctx, X, W, S, 16385, 1 << 20, 128, 2, 0, 0.1, OUT, BIAS, WS, 1 << 40, None)
    assert st == NH.UNSUPPORTED


def test_host_twins_without_memory_are_an_error():
    """A size that no allocation meets comes back as a status, never as an exception through the C entry."""
    logits, idx = np.zeros((1, 4), np.float32), np.zeros((1, 1), np.int32)
    counts, loss = np.zeros((1, 4), np.int32), np.zeros(1, np.float32)
    st, err = NH.call_status("nh_moe_balance_loss_host", logits.ctypes.data, idx.ctypes.data, None, 1, 0, 1 << 60, 1, 0, 0.1,
                             counts.ctypes.data, loss.ctypes.data)
    assert st == NH.DEVICE_ERROR and err.message == b"out of host memory"


def test_moe_host_of_weights_without_a_value():
    """A weight block of scale 255 makes h NaN in its column: an intermediate with no value, as on the device."""
    t, h, i, e, k = 2, 64, 32, 2, 1
    rng = np.random.default_rng(0)
    x, logits = rng.standard_normal((t, h)).astype(np.float32), np.array([[1, -1], [-1, 1]], np.float32)
    tiles = [tile_host(*R.quantize(rng.standard_normal(s))[:2], *s) for s in ((i, h), (i, h), (h, i), (h, i))]
    up, down = np.concatenate(tiles[:2]), np.concatenate(tiles[2:])
    out = np.empty((t, h), np.float32)
    args = (x.ctypes.data, NH.F32, logits.ctypes.data, t, h, i, e, k, 0, 1.0, up.ctypes.data, down.ctypes.data, None, None,
            out.ctypes.data, NH.F32)
    assert NH.call_status("nh_moe_forward_mxfp4_host", *args)[0] == NH.OK
    up[tiles[0].size + 1024 + 4 * 3] = 255  # expert 1, row 3, block 0
    st, err = NH.call_status("nh_moe_forward_mxfp4_host", *args)
    assert st == NH.NON_FINITE_INPUT and err.argument == b"intermediate" and err.index == i + 3
