"""The MXFP4 kernels through the C ABI against plain 64-bit forms.

Most products run on values whose sums f32 holds exactly (grid elements, a few powers of two of scale: every partial
sum is a whole number of quanta below 2^24), so the kernels' outputs have to be equal, whatever the order of the sums."""
import ctypes as C

import numpy as np
import pytest

import mx_reference as R
import nemotron_hip as NH

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
GUARD = 256  # bytes in front of and behind a buffer that a kernel must leave alone


@pytest.fixture(scope="module")
def ctx():
    c = NH.Context(0)
    yield c
    c.close()


def note(msg):
    print(f"[gpu-case] {msg}", flush=True)


class Guarded:
    """A device array between guard bytes, `shift` elements off alignment."""

    def __init__(self, ctx, shape, dtype, shift=0):
        self.shape, self.dtype = shape, np.dtype(dtype)
        self.nbytes = int(np.prod(shape, dtype=np.int64)) * self.dtype.itemsize
        self.at = GUARD + shift * self.dtype.itemsize
        self.buf = ctx.upload(np.full(self.at + self.nbytes + GUARD, 0xA5, np.uint8))
        self.ptr = self.buf.ptr + self.at

    def numpy(self):
        b = self.buf.numpy()
        assert (b[:self.at] == 0xA5).all() and (b[self.at + self.nbytes:] == 0xA5).all(), "written outside the output"
        return b[self.at:self.at + self.nbytes].view(self.dtype).reshape(self.shape)


def shifted(ctx, array, shift):
    """The array on the device, `shift` elements off alignment."""
    array = np.ascontiguousarray(array)
    pad = np.full(shift * array.itemsize, 0xFF, np.uint8)
    buf = ctx.upload(np.concatenate([pad, array.view(np.uint8).reshape(-1), np.full(64, 0xFF, np.uint8)]))
    return buf, buf.ptr + pad.size


def edge_rows(rng, cols):
    rows = [np.zeros(cols), -np.zeros(cols), rng.standard_normal(cols), rng.standard_normal(cols) * 1e-38,
            rng.integers(-8, 9, cols) * 2.0 ** -149, rng.choice([3.4028234663852886e38, -1e38, 1.0], cols)]
    for e in (-149, -130, -127, -126, -125, -20, 0, 100, 125):
        tie = rng.choice(R.MIDDLE, cols) * 2.0 ** e * rng.choice([-1, 1], cols)
        tie[::32] = 4 * 2.0 ** e
        rows += [tie, np.nextafter(tie.astype(np.float32), np.float32(0)), np.nextafter(tie.astype(np.float32), np.float32(np.inf))]
    return np.array(rows).astype(np.float32)


def quantize(ctx, x, dtype, shift=0, nonfinite=None):
    rows, cols = x.shape
    buf, at = shifted(ctx, x, shift)
    codes = Guarded(ctx, (rows, -(-cols // 2)), np.uint8, shift)
    scales = Guarded(ctx, (rows, -(-cols // 32)), np.uint8, shift)
    NH.call("nh_quantize_rows_mxfp4", ctx.handle, at, dtype, rows, cols, codes.ptr, scales.ptr, nonfinite, None)
    ctx.synchronize()
    return codes, scales


@pytest.mark.parametrize("cols", [1, 2, 7, 8, 31, 32, 33, 64, 97, 128, 1000, 4096])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shift", [0, 1])
def test_quantize_is_the_definition(ctx, cols, dtype, shift):
    note(f"quantize cols={cols} {dtype} shift={shift}")
    x = edge_rows(np.random.default_rng(cols), cols)
    if dtype == "bf16":
        b = np.minimum(R.to_bf16_bits(x) & 0x7FFF, 0x7F7F) | (R.to_bf16_bits(x) & 0x8000)  # the largest round to infinity
        x, d, src = R.from_bf16_bits(b), NH.BF16, b.astype(np.uint16)
    else:
        d, src = NH.F32, x
    codes, scales = quantize(ctx, src, d, shift)
    rc, rs, rv = R.quantize(x)
    assert np.array_equal(scales.numpy(), rs) and np.array_equal(codes.numpy(), rc)
    out = Guarded(ctx, x.shape, src.dtype, shift)
    NH.call("nh_dequantize_mxfp4", ctx.handle, codes.ptr, scales.ptr, *x.shape, out.ptr, d, None)
    ctx.synchronize()
    want = rv.astype(np.float32).view(np.uint32)
    assert np.array_equal(out.numpy().view(np.uint16 if d == NH.BF16 else np.uint32),
                          (want >> 16).astype(np.uint16) if d == NH.BF16 else want)


def test_quantize_every_bf16_value(ctx):
    """Each finite bf16 as the second value of a block whose first is the largest power under it and up to 2^8 above."""
    note("quantize every bf16")
    bits = np.arange(65536, dtype=np.uint32)
    bits = bits[(bits & 0x7F80) != 0x7F80]
    x = np.zeros((bits.size, 32), np.uint16)
    for j in range(8):
        x[:, 4 * j] = 0
    x[:, 1] = bits
    rise = np.arange(bits.size) % 9
    x[:, 0] = np.minimum(((bits & 0x7F80) + (rise << 7)), 0x7F00).astype(np.uint16)
    codes, scales = quantize(ctx, x, NH.BF16)
    rc, rs, _ = R.quantize(R.from_bf16_bits(x))
    assert np.array_equal(scales.numpy(), rs) and np.array_equal(codes.numpy(), rc)


def test_dequantize_every_code_and_scale(ctx):
    note("dequantize every code and scale")
    codes = np.tile(np.tile(np.arange(256, dtype=np.uint8), (16, 1)).reshape(256, 16), (16, 1))
    scales = np.repeat(np.arange(256, dtype=np.uint8), 16).reshape(-1, 1)
    dc, ds = ctx.upload(codes), ctx.upload(scales)
    with np.errstate(over="ignore"):
        want = R.decode(codes, scales, 32).astype(np.float32)
    for dtype in (NH.F32, NH.BF16):
        out = Guarded(ctx, (4096, 32), np.float32 if dtype == NH.F32 else np.uint16)
        NH.call("nh_dequantize_mxfp4", ctx.handle, dc.ptr, ds.ptr, 4096, 32, out.ptr, dtype, None)
        ctx.synchronize()
        got = out.numpy() if dtype == NH.F32 else R.from_bf16_bits(out.numpy())
        assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_bad_values_mark_their_block(ctx, bad, dtype):
    note(f"quantize non-finite {bad} {dtype}")
    x = np.random.default_rng(2).standard_normal((5, 100)).astype(np.float32)
    x[1, 40] = x[3, 99] = x[3, 98] = bad
    b = R.to_bf16_bits(x)
    src, d = (b, NH.BF16) if dtype == "bf16" else (x, NH.F32)
    word = ctx.upload(np.zeros(1, np.uint64))
    codes, scales = quantize(ctx, src, d, nonfinite=word.ptr)
    rc, rs, _ = R.quantize(R.from_bf16_bits(b) if dtype == "bf16" else x)
    assert np.array_equal(scales.numpy(), rs) and np.array_equal(codes.numpy(), rc)
    assert (scales.numpy() == 255).sum() == 2
    st, err = NH.call_status("nh_take_nonfinite", ctx.handle, word.ptr, None)
    assert st == NH.NON_FINITE_INPUT and err.index == 140
    assert np.isnan(err.value) if np.isnan(bad) else err.value == bad


def test_quantize_of_nothing(ctx):
    for rows, cols in ((0, 64), (4, 0)):
        NH.call("nh_quantize_rows_mxfp4", ctx.handle, None, NH.F32, rows, cols, None, None, None, None)
        NH.call("nh_dequantize_mxfp4", ctx.handle, None, None, rows, cols, None, NH.F32, None)


@pytest.mark.parametrize("n,k", [(1, 1), (16, 128), (17, 129), (5, 500), (33, 512), (40, 513), (16, 1023), (300, 1856)])
def test_tile_is_the_documented_layout(ctx, n, k):
    note(f"tile n={n} k={k}")
    codes, scales, _ = R.quantize(np.random.default_rng(n).standard_normal((n, k)))
    if k % 2:
        codes[:, -1] |= 0xF0  # what lies behind the last value stays out
    (bc, pc), (bs, ps) = shifted(ctx, codes, 1), shifted(ctx, scales, 3)
    size = NH.lib().nh_tiled_mxfp4_weights_bytes(n, k)
    out = Guarded(ctx, (size,), np.uint8)
    NH.call("nh_tile_weights_mxfp4", ctx.handle, pc, ps, n, k, out.ptr, size, None)
    ctx.synchronize()
    if k % 2:
        codes[:, -1] &= 0x0F
    assert np.array_equal(out.numpy(), R.tile(codes, scales, n, k))


def weights(ctx, w):
    """(tiled device weights, values) of an f32 matrix that MXFP4 holds or rounds."""
    codes, scales, v = R.quantize(w)
    return NH.tile_weights_mxfp4(ctx, ctx.upload(codes), ctx.upload(scales), *w.shape), v


def run_linear(ctx, x, tiled, n, bias=None, x_dtype=NH.F32, out_dtype=NH.F32, shift=0, nonfinite=None, stream=None):
    m, k = x.shape
    src = R.to_bf16_bits(x) if x_dtype == NH.BF16 else x.astype(np.float32)
    bx, px = shifted(ctx, src, shift)
    out = Guarded(ctx, (m, n), np.float32 if out_dtype == NH.F32 else np.uint16, shift)
    need = NH.lib().nh_linear_mxfp4_workspace_size(m, n, k)
    # a workspace of what earlier calls left: NaN scales everywhere
    ws = ctx.upload(np.full(max(need, 16), 0xFF, np.uint8))
    db = ctx.upload(bias) if bias is not None else None
    NH.call("nh_linear_mxfp4", ctx.handle, px, x_dtype, tiled.ptr, NH.ptr(db), m, n, k, out.ptr, out_dtype, ws.ptr, need,
            nonfinite, stream)
    ctx.synchronize(stream)
    return out.numpy()


# every kernel: K tiles per wave 1, 2, 4, 8, 16 with K at both ends and ragged, rows 1 / 16 / 17 / 64 / past them, the
# three tiles of the large product, K past what the streaming forms take
LINEAR = [(1, 16, 32), (1, 1, 1), (3, 17, 33), (16, 48, 1024), (16, 40, 1025), (2, 100, 2048), (15, 33, 2049),
          (16, 272, 4096), (1, 4099, 2701), (5, 64, 4097), (9, 130, 8192), (4, 16, 8200), (16, 35, 16384), (1, 5000, 512),
          (3, 40, 16385), (16, 16, 20000), (17, 16, 128), (17, 40, 1000), (64, 33, 2000), (50, 70, 4095), (33, 100, 4096),
          (64, 50, 8192), (31, 19, 5000), (64, 24, 9000), (65, 64, 512), (65, 1, 1), (100, 130, 300), (300, 515, 130),
          (129, 200, 2701), (1040, 2050, 256), (1040, 2047, 700), (4100, 4100, 128), (4097, 4200, 384), (2050, 17000, 64),
          (20, 50, 3000), (1030, 8000, 128), (520, 16300, 1100), (2040, 16300, 384)]


@pytest.mark.parametrize("m,n,k", LINEAR)
@pytest.mark.parametrize("kind", ["bf16-bf16", "f32-f32"])
def test_linear_exact(ctx, m, n, k, kind):
    note(f"linear m={m} n={n} k={k} {kind}")
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    # quanta of 2^-2 * 4^-spread, products up to 36 * 4^spread: k * 144 * 16^spread < 2^24
    spread = 1 if k * 144 * 16 < 1 << 24 else 0
    x, w = R.grid_matrix(rng, m, k, spread), R.grid_matrix(rng, n, k, spread)
    bias = R.grid_matrix(rng, 1, n, 0)[0] if kind == "f32-f32" else None
    tiled, wv = weights(ctx, w)
    assert np.array_equal(wv, w)
    bf16 = kind == "bf16-bf16"
    got = run_linear(ctx, x, tiled, n, bias, NH.BF16 if bf16 else NH.F32, NH.BF16 if bf16 else NH.F32, shift=n % 2)
    want = x.astype(np.float32) @ w.T.astype(np.float32)  # exact, as the kernel's
    if bias is not None:
        want = want + bias
    want = R.to_bf16_bits(want) if bf16 else want
    assert np.array_equal(got, want), f"{(got != want).sum()} differ"


@pytest.mark.parametrize("m,n,k", [(1, 300, 4096), (16, 64, 2701), (40, 100, 3000), (200, 300, 2701), (1100, 1030, 512)])
def test_linear_of_normal_rows(ctx, m, n, k):
    note(f"linear normal m={m} n={n} k={k}")
    rng = np.random.default_rng(k)
    x = (rng.standard_normal((m, k)) * np.where(rng.random(k) < 0.01, 30, 1)).astype(np.float32)
    w = (rng.standard_normal((n, k)) * 0.02).astype(np.float32)
    bias = rng.standard_normal(n).astype(np.float32)
    tiled, wv = weights(ctx, w)
    xv = R.quantize(x)[2]
    y, size = xv @ wv.T + bias, np.abs(xv) @ np.abs(wv).T + np.abs(bias)
    # one rounding per addition at most: k products, eight waves' parts, the bias
    tol = (k + 9) * U * size
    assert (np.abs(run_linear(ctx, x, tiled, n, bias) - y) <= tol).all()
    got = R.from_bf16_bits(run_linear(ctx, x, tiled, n, bias, out_dtype=NH.BF16))
    assert (np.abs(got - y) <= tol + 2.0 ** -8 * (np.abs(y) + tol)).all()


@pytest.mark.parametrize("m,n,k", [(2, 40, 300), (20, 40, 300), (90, 40, 300), (3, 20, 20000)])
def test_linear_bad_values(ctx, m, n, k):
    """A non-finite x makes its row NaN and is reported; other rows are as before.  Weight scales of 255 make columns."""
    note(f"linear non-finite m={m} n={n} k={k}")
    rng = np.random.default_rng(k)
    x, w = R.grid_matrix(rng, m, k, 0), R.grid_matrix(rng, n, k, 0)
    codes, scales, _ = R.quantize(w)
    scales[3, 2] = 255
    tiled = NH.tile_weights_mxfp4(ctx, ctx.upload(codes), ctx.upload(scales), n, k)
    x[1, k - 1] = np.inf
    word = ctx.upload(np.zeros(1, np.uint64))
    got = run_linear(ctx, x, tiled, n, nonfinite=word.ptr)
    ok = np.ones((m, n), bool)
    ok[1], ok[:, 3] = False, False
    assert np.isnan(got[~ok]).all()
    x[1] = 0
    assert np.array_equal(got[ok], (x @ w.T)[ok])
    st, err = NH.call_status("nh_take_nonfinite", ctx.handle, word.ptr, None)
    assert (st, err.argument, err.index, err.value) == (NH.NON_FINITE_INPUT, b"input", k + k - 1, np.inf)


def moe_case(ctx, t, h, i, e, k, seed, spread=0, dense_w=False):
    rng = np.random.default_rng(seed)
    x = R.grid_matrix(rng, t, h, spread)
    logits = rng.standard_normal((t, e)).astype(np.float32)
    make = (lambda n, c: rng.standard_normal((n, c)).astype(np.float32)) if dense_w else (lambda n, c: R.grid_matrix(rng, n, c, 0))
    ups, downs = [make(i, h) for _ in range(e)], [make(h, i) for _ in range(e)]
    return rng, x, logits, ups, downs


def tile_all(ctx, ws):
    parts = []
    for w in ws:
        codes, scales, _ = R.quantize(w)
        parts.append(NH.tile_weights_mxfp4(ctx, ctx.upload(codes), ctx.upload(scales), *w.shape).numpy())
    return ctx.upload(np.concatenate(parts))


def route(logits, k, renormalize, scaling):
    t, e = logits.shape
    idx, wts = np.empty((t, k), np.int32), np.empty((t, k), np.float32)
    NH.call("nh_moe_route_sigmoid_topk_host", logits.ctypes.data, t * e, t, e, k, renormalize, scaling, idx.ctypes.data, t * k,
            wts.ctypes.data, t * k)
    return idx, wts


# rows per expert from none to past one pass of 64; widths ragged against 32, 128 and 512; all five splits of K
MOE = [(1, 64, 32, 8, 2), (3, 100, 70, 4, 1), (8, 1040, 200, 16, 6), (16, 333, 129, 3, 3), (17, 96, 33, 8, 2), (40, 256, 130, 60, 4),
       (70, 128, 96, 2, 1), (200, 160, 64, 2, 2), (33, 512, 1100, 5, 2), (20, 2100, 40, 4, 2), (5, 4200, 50, 4, 2), (24, 60, 4200, 3, 2),
       (12, 48, 2200, 3, 2), (9, 8192, 32, 2, 1), (90, 7000, 36, 2, 2), (6, 60, 4200, 3, 2), (40, 2100, 40, 4, 2),
       (10, 64, 32, 200, 4), (40, 32, 32, 300, 8)]


@pytest.mark.parametrize("t,h,i,e,k", MOE)
def test_moe_layer(ctx, t, h, i, e, k):
    note(f"moe t={t} h={h} i={i} e={e} k={k}")
    rng, x, logits, ups, downs = moe_case(ctx, t, h, i, e, k, t + h)
    bu, bd = R.grid_matrix(rng, e, i, 0), R.grid_matrix(rng, e, h, 0)
    shared = rng.standard_normal((t, h)).astype(np.float32)
    du, dd = tile_all(ctx, ups), tile_all(ctx, downs)
    idx, wts = route(logits, k, 1, 2.5)
    with_bias = t % 2 == 0
    dbu, dbd, dsh = ctx.upload(bu), ctx.upload(bd), ctx.upload(shared)
    biases = C.byref(NH.MoeBiases(dbu.ptr, dbd.ptr, None, None)) if with_bias else None
    dx, dl = ctx.upload(x), ctx.upload(logits)
    need = NH.lib().nh_moe_forward_mxfp4_workspace_size(t, h, i, e, k)
    ws = ctx.upload(np.full(need, 0xFF, np.uint8))
    out = Guarded(ctx, (t, h), np.float32)
    word = ctx.upload(np.zeros(1, np.uint64))
    NH.call("nh_moe_forward_mxfp4", ctx.handle, dx.ptr, NH.F32, dl.ptr, t, h, i, e, k, 1, 2.5, du.ptr, dd.ptr, biases,
            dsh.ptr if with_bias else None, out.ptr, NH.F32, ws.ptr, need, word.ptr, None)
    ctx.synchronize()
    got = out.numpy()
    at = (C.c_size_t * 5)()
    NH.lib().nh_moe_mxfp4_workspace_layout(t, h, i, e, k, at)
    assert np.array_equal(ws.numpy()[at[0]:at[0] + idx.nbytes].view(np.int32).reshape(idx.shape), idx)
    want, size = np.zeros((t, h)), np.zeros((t, h))
    if with_bias:
        want, size = shared.astype(np.float64), np.abs(shared).astype(np.float64)
    for a in range(t):
        for j in range(k):
            n = idx[a, j]
            # sums of quarters: exact in f32, so h and its codes are the kernel's (the square rounds once)
            y = (x[a].astype(np.float32) @ ups[n].T + (bu[n] if with_bias else 0)).astype(np.float32)
            hv = R.quantize((np.maximum(y, 0) ** 2).astype(np.float32).reshape(1, -1))[2][0]
            d, s = downs[n] @ hv, np.abs(downs[n]) @ np.abs(hv)
            if with_bias:
                d, s = d + bd[n], s + np.abs(bd[n])
            want[a] += wts[a, j].astype(np.float64) * d
            size[a] += wts[a, j].astype(np.float64) * s
    # i products, eight parts, a bias; the weight's product and the sum over the routes
    assert (np.abs(got - want) <= (i + 10 + 2 * k) * U * size).all()
    assert NH.call_status("nh_take_nonfinite", ctx.handle, word.ptr, None)[0] == NH.OK


def test_moe_layer_bf16_against_the_host_twin(ctx):
    """Ordinary rows and weights in bf16: the twin sums in 64 bits, so a code of h may fall to the other side of a tie."""
    t, h, i, e, k = 20, 256, 192, 8, 3
    note("moe bf16 host twin")
    rng, x, logits, ups, downs = moe_case(ctx, t, h, i, e, k, 9, dense_w=True)
    x = R.to_bf16_bits(rng.standard_normal((t, h)))
    du, dd = tile_all(ctx, ups), tile_all(ctx, downs)
    need = NH.lib().nh_moe_forward_mxfp4_workspace_size(t, h, i, e, k)
    ws, dx, dl = ctx.empty(need, np.uint8), ctx.upload(x), ctx.upload(logits)
    out = Guarded(ctx, (t, h), np.uint16)
    NH.call("nh_moe_forward_mxfp4", ctx.handle, dx.ptr, NH.BF16, dl.ptr, t, h, i, e, k, 0, 1.0, du.ptr, dd.ptr, None, None,
            out.ptr, NH.BF16, ws.ptr, need, None, None)
    ctx.synchronize()
    want = np.empty((t, h), np.uint16)
    hu, hd = du.numpy(), dd.numpy()
    NH.call("nh_moe_forward_mxfp4_host", x.ctypes.data, NH.BF16, logits.ctypes.data, t, h, i, e, k, 0, 1.0, hu.ctypes.data,
            hd.ctypes.data, None, None, want.ctypes.data, NH.BF16)
    got, want = R.from_bf16_bits(out.numpy()), R.from_bf16_bits(want)
    # sums in f32 against 64 bits: 2^-24 * 256 of the sum's size, and two bf16 roundings; h's 11520 values have a chance
    # of about 1e-5 each to change a code, so one that does (a step of its block) stays within a row's tenth
    off = np.linalg.norm(got - want, axis=1) / np.linalg.norm(want, axis=1)
    assert (off < 0.1).all() and np.median(off) < 2.0 ** -8


def test_moe_weights_without_a_value(ctx):
    """A weight block of scale 255: a NaN column of h is a bad intermediate, a NaN column of the experts' output is none."""
    t, h, i, e, k = 6, 96, 64, 4, 2
    note("moe weight scale 255")
    _, x, logits, ups, downs = moe_case(ctx, t, h, i, e, k, 5)
    idx, _ = route(logits, k, 0, 1.0)
    du, dd = tile_all(ctx, ups).numpy(), tile_all(ctx, downs).numpy()
    need = NH.lib().nh_moe_forward_mxfp4_workspace_size(t, h, i, e, k)
    bad_expert = int(idx[0, 0])
    hit = (idx == bad_expert).any(axis=1)
    assert hit.any() and not hit.all()
    for which in ("up", "down"):
        w = {"up": du.copy(), "down": dd.copy()}
        n, cols = (i, h) if which == "up" else (h, i)
        per = w[which].size // e
        # row 5 of the expert's second 16 (r = 5 of row tile 1): block 1 of its one K tile, piece byte 4 lane
        region = 1024 + 256
        w[which][bad_expert * per + region + 1024 + 4 * (16 * 1 + 5)] = 255
        up, down = ctx.upload(w["up"]), ctx.upload(w["down"])
        ws, dx, dl = ctx.upload(np.full(need, 0xFF, np.uint8)), ctx.upload(x), ctx.upload(logits)
        out, word = Guarded(ctx, (t, h), np.float32), ctx.upload(np.zeros(1, np.uint64))
        NH.call("nh_moe_forward_mxfp4", ctx.handle, dx.ptr, NH.F32, dl.ptr, t, h, i, e, k, 0, 1.0, up.ptr, down.ptr, None, None,
                out.ptr, NH.F32, ws.ptr, need, word.ptr, None)
        ctx.synchronize()
        got, (st, err) = out.numpy(), NH.call_status("nh_take_nonfinite", ctx.handle, word.ptr, None)
        host = np.empty((t, h), np.float32)
        hst, herr = NH.call_status("nh_moe_forward_mxfp4_host", x.ctypes.data, NH.F32, logits.ctypes.data, t, h, i, e, k, 0, 1.0,
                                   w["up"].ctypes.data, w["down"].ctypes.data, None, None, host.ctypes.data, NH.F32)
        if which == "up":
            assert st == hst == NH.NON_FINITE_INPUT and err.argument == herr.argument == b"intermediate"
            assert err.index == herr.index and err.index % i == 21
            assert np.isnan(got[hit]).all() and np.isfinite(got[~hit]).all()
        else:
            assert st == hst == NH.OK
            assert np.isnan(got[hit, 21]).all() and np.isnan(host[hit, 21]).all()
            got[hit, 21] = 0
            assert np.isfinite(got).all()


@pytest.mark.parametrize("m", [3, 40, 200])
def test_linear_in_flight_twice_and_replayed(ctx, m):
    """Calls in flight on two streams with a workspace each, eager and as graphs replayed over new rows."""
    n, k = 300, 700
    note(f"linear on two streams, captured and replayed, m={m}")
    rng = np.random.default_rng(4)
    w = R.grid_matrix(rng, n, k, 0)
    tiled, _ = weights(ctx, w)
    need = NH.lib().nh_linear_mxfp4_workspace_size(m, n, k)
    graphs, runs = NH.HipGraphs(), []

    class Run:
        def __init__(self):
            self.stream = NH.P()
            NH.call("nh_stream_create", ctx.handle, C.byref(self.stream))
            self.dx = ctx.empty((m, k), np.float32)
            self.out, self.ws = Guarded(ctx, (m, n), np.float32), ctx.upload(np.full(max(need, 16), 0xFF, np.uint8))
            self.graph = graphs.capture(self.stream, self.issue)
            self.new_rows()

        def new_rows(self):
            self.x = R.grid_matrix(rng, m, k, 0).astype(np.float32)
            self.dx.copy_from(self.x)

        def issue(self):
            NH.call("nh_linear_mxfp4", ctx.handle, self.dx.ptr, NH.F32, tiled.ptr, None, m, n, k, self.out.ptr, NH.F32,
                    self.ws.ptr, need, None, self.stream)

    runs = [Run(), Run()]
    ctx.synchronize()
    for turn in range(4):
        for r in runs * 2:
            r.issue() if turn == 0 else graphs.launch(r.graph[1], r.stream)
        for r in runs:
            ctx.synchronize(r.stream)
            assert np.array_equal(r.out.numpy(), r.x @ w.T.astype(np.float32)), turn
            r.new_rows()
    for r in runs:
        graphs.destroy(*r.graph)
        NH.call("nh_stream_destroy", ctx.handle, r.stream)


def test_moe_bad_values_stay_in_their_rows(ctx):
    t, h, i, e, k = 6, 96, 64, 4, 2
    note("moe non-finite")
    _, x, logits, ups, downs = moe_case(ctx, t, h, i, e, k, 5)
    du, dd = tile_all(ctx, ups), tile_all(ctx, downs)
    need = NH.lib().nh_moe_forward_mxfp4_workspace_size(t, h, i, e, k)

    def run(x):
        ws, dx, dl = ctx.upload(np.full(need, 0xFF, np.uint8)), ctx.upload(x), ctx.upload(logits)
        out, word = Guarded(ctx, (t, h), np.float32), ctx.upload(np.zeros(1, np.uint64))
        NH.call("nh_moe_forward_mxfp4", ctx.handle, dx.ptr, NH.F32, dl.ptr, t, h, i, e, k, 0, 1.0, du.ptr, dd.ptr, None, None,
                out.ptr, NH.F32, ws.ptr, need, word.ptr, None)
        ctx.synchronize()
        return out.numpy(), NH.call_status("nh_take_nonfinite", ctx.handle, word.ptr, None)

    clean, (st, _) = run(x)
    assert st == NH.OK
    bad = x.copy()
    bad[2, 50] = np.nan
    got, (st, err) = run(bad)
    assert st == NH.NON_FINITE_INPUT and err.argument == b"input" and err.index == 2 * h + 50
    assert np.isnan(got[2]).all() and np.array_equal(np.delete(got, 2, 0), np.delete(clean, 2, 0))
    big = x.copy()
    big[4] = x[4] * np.float32(2.0 ** 100)  # its squares leave f32
    got, (st, err) = run(big)
    assert st == NH.NON_FINITE_INPUT and err.argument == b"intermediate"
    assert np.isnan(got[4]).all() and np.array_equal(np.delete(got, 4, 0), np.delete(clean, 4, 0))
