"""The MXFP4 products of large tiles over several output tiles per workgroup: the ring of stages and the ring of scale
pieces run on from one tile into the next, and a tile's last piece of scales may hold one stage, two or four."""
import numpy as np
import pytest

import mx_reference as R
import nemotron_hip as NH
from dispatch import BIAS, OUT, W, WS, X, Recorder

# K tiles of 128: 4 (one whole piece), 5 (its last piece is one stage, next to the next tile's first), 6, 8, 9 and 13
RING = [(2050, 8200, 507, 128), (2050, 8200, 635, 128), (2050, 8200, 763, 128), (2050, 14400, 1019, 128),
        (2050, 14400, 1147, 128), (2050, 16400, 507, 256), (2050, 16400, 635, 256), (2050, 16400, 1019, 256),
        (2050, 16400, 1147, 256), (2050, 14400, 1659, 256)]


@pytest.mark.parametrize("m,n,k,tile", RING)
def test_ring_shapes_have_several_tiles_per_workgroup(m, n, k, tile):
    rec = Recorder()
    ws = NH.lib().nh_linear_mxfp4_workspace_size(m, n, k)
    name, grid, _ = rec.launches("nh_linear_mxfp4", X, NH.F32, W, BIAS, m, n, k, OUT, NH.F32, WS, ws, None, None)[-1]
    rec.close()
    assert name == f"mx_gemm_{tile}x{tile}" and -(-m // tile) * -(-n // tile) >= 2 * grid


@pytest.fixture(scope="module")
def ctx():
    c = NH.Context(0)
    yield c
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,tile", RING)
def test_linear_exact_over_tiles(ctx, m, n, k, tile):
    """Values whose sums f32 holds (multiples of 1/16 up to 144 k, below 2^20): equal, whatever the order of the sums.
    Blocks have one of three scales, so a block of another's scale shows."""
    print(f"[gpu-case] linear over tiles m={m} n={n} k={k} tile={tile}", flush=True)
    rng = np.random.default_rng(k + tile)
    x, w = R.grid_matrix(rng, m, k, 1), R.grid_matrix(rng, n, k, 1)
    bias = R.grid_matrix(rng, 1, n, 0)[0]
    dx, dw, db = ctx.upload(x), ctx.upload(w), ctx.upload(bias)
    codes, scales = ctx.empty((n, -(-k // 2)), np.uint8), ctx.empty((n, -(-k // 32)), np.uint8)
    NH.call("nh_quantize_rows_mxfp4", ctx.handle, dw.ptr, NH.F32, n, k, codes.ptr, scales.ptr, None, None)
    tiled = NH.tile_weights_mxfp4(ctx, codes, scales, n, k)
    need = NH.lib().nh_linear_mxfp4_workspace_size(m, n, k)
    ws, out = ctx.upload(np.full(need, 0xFF, np.uint8)), ctx.empty((m, n), np.float32)
    want = x @ w.T + bias
    for _ in range(2):
        out.fill_bytes(0xFF)
        NH.call("nh_linear_mxfp4", ctx.handle, dx.ptr, NH.F32, tiled.ptr, db.ptr, m, n, k, out.ptr, NH.F32, ws.ptr, need, None,
                None)
        ctx.synchronize()
        got = out.numpy()
        assert np.array_equal(got, want), f"{(got != want).sum()} differ, first at {np.argwhere(got != want)[0]}"
