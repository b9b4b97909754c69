"""Rows by expert and low-rank adapters whose arrays pass 2^31 elements and 4 GiB: zeros but for rows at both ends."""
import numpy as np
import pytest

import adapters_reference as A
import nemotron_hip as NH
from test_gpu_mxfp4 import note
from test_gpu_mxfp4_far import free, get, put, zeros  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = NH.Context(0)
    yield c
    c.close()


def ends(ctx, buf, rows, cols, ends_of, values):
    """Writes `values` into the first and the last rows of a bf16 array."""
    half = len(values) // 2
    put(ctx, buf, 0, values[:half])
    put(ctx, buf, (rows - (len(values) - half)) * cols * 2, values[half:])


def read_ends(ctx, buf, rows, cols, n, dtype=np.uint16):
    size = np.dtype(dtype).itemsize
    half = n // 2
    return np.concatenate([get(ctx, buf, 0, (half, cols), dtype), get(ctx, buf, (rows - (n - half)) * cols * size, (n - half, cols), dtype)])


@pytest.mark.parametrize("tokens,hidden", [((1 << 19) + 37, 4100), (3, (1 << 30) + 1), (1, (1 << 31) - 1)])
def test_rows(ctx, free, tokens, hidden):  # noqa: F811
    note(f"far rows {tokens} x {hidden}")
    rng = np.random.default_rng(0)
    n = 8 if tokens > 8 else 0
    x, rows, out = [zeros(ctx, (tokens, hidden), np.uint16, free) for _ in range(3)]
    pos = ctx.upload(np.arange(tokens, dtype=np.int32)[::-1].copy())
    free.append(pos)
    w = rng.uniform(0.5, 1, tokens).astype(np.float32)
    dw = ctx.upload(w)
    sizes = (tokens, 1, hidden, tokens)
    if n:
        xs, v = A.held(rng.standard_normal((n, hidden)), "bf16")
        ends(ctx, x, tokens, hidden, n, xs)
        wn = np.concatenate([w[:n // 2], w[-(n - n // 2):]]).astype(np.float64)[:, None]
    else:  # the last values of long rows
        xs, v = A.held(rng.standard_normal((1, 1000)), "bf16")
        put(ctx, x, x.nbytes - 2000, xs)
        wn = w[-1:].astype(np.float64)[:, None]
    near = lambda got, want, times: (np.abs(A.values(got) - want) <= 1.01 * times * (2.0 ** -8 + A.U) * np.abs(want)).all()  # noqa: E731
    rows.fill_bytes(0xA5)
    NH.call("nh_moe_dispatch", ctx.handle, x.ptr, NH.BF16, pos.ptr, dw.ptr, *sizes, rows.ptr, NH.BF16, None)
    ctx.synchronize()
    if n:
        assert near(read_ends(ctx, rows, tokens, hidden, n)[::-1], wn * v, 1)  # pos turns them round
    else:
        assert near(get(ctx, rows, 2 * hidden - 2000, (1, 1000), np.uint16), wn * v, 1)
        assert (get(ctx, rows, rows.nbytes - 4000, 1000, np.uint16) == 0).all()
    NH.call("nh_moe_combine_rows", ctx.handle, rows.ptr, NH.BF16, pos.ptr, None, x.ptr, *sizes, out.ptr, NH.BF16, None)
    ctx.synchronize()
    if n:
        assert near(read_ends(ctx, out, tokens, hidden, n), (1 + wn) * v, 2)
        assert (get(ctx, out, (tokens // 2) * hidden * 2, hidden, np.uint16) == 0).all()
    else:
        assert near(get(ctx, out, out.nbytes - 2000, (1, 1000), np.uint16), (1 + wn) * v, 2)


def test_dweights_of_the_longest_rows(ctx, free):  # noqa: F811
    hidden = (1 << 31) - 1
    note("far dweights")
    rows, out = zeros(ctx, (1, hidden), np.uint16, free), zeros(ctx, (1, hidden), np.uint16, free)
    for b, v in ((rows, 2.0), (out, 3.0)):
        put(ctx, b, b.nbytes - 20, A.held(np.full(10, v), "bf16")[0])
    pos, dw = ctx.upload(np.zeros(1, np.int32)), ctx.upload(np.zeros(1, np.float32))
    NH.call("nh_moe_combine_rows_backward", ctx.handle, out.ptr, NH.BF16, rows.ptr, NH.BF16, pos.ptr, None, 1, 1, hidden, 1,
            rows.ptr, dw.ptr, None)
    assert dw.numpy()[0] == 60.0  # exact in f32
    assert np.array_equal(get(ctx, rows, rows.nbytes - 40, 20, np.uint16), get(ctx, out, out.nbytes - 40, 20, np.uint16))


def test_sort_of_the_most_routes(ctx, free):  # noqa: F811
    n = (1 << 31) - 1
    note("far sort")
    ids, perm, pos = [zeros(ctx, (n,), np.int32, free) for _ in range(3)]
    offsets = ctx.upload(np.full(4, -7, np.int32))
    put(ctx, ids, 4 * (n - 5), np.array([2, 9, 1, -1, 0], np.int32))
    NH.call("nh_moe_permute", ctx.handle, ids.ptr, n, 1, 3, offsets.ptr, perm.ptr, pos.ptr, None)
    ctx.synchronize()
    assert offsets.numpy().tolist() == [0, n - 4, n - 3, n - 2]
    assert get(ctx, perm, 4 * (n - 7), 5, np.int32).tolist() == [n - 7, n - 6, n - 1, n - 3, n - 5]
    assert get(ctx, pos, 4 * (n - 7), 7, np.int32).tolist() == [n - 7, n - 6, n - 3, -1, n - 4, -1, n - 5]
    for at in (0, 12345678, 1 << 30, (1 << 31) - (1 << 23) - 3):  # chunk ends among them
        assert np.array_equal(get(ctx, pos, 4 * at, 70, np.int32), np.arange(at, at + 70))
        assert np.array_equal(get(ctx, perm, 4 * at, 70, np.int32), np.arange(at, at + 70))


@pytest.mark.parametrize("m,n,k,adapters", [((1 << 20) + 75, 2100, 2056, 2), (2100, 1 << 20, 72, 3), (2100, 72, 1 << 20, 3)])
def test_adapters(ctx, free, m, n, k, adapters):  # noqa: F811
    note(f"far adapters m={m} n={n} k={k}")
    rng = np.random.default_rng(0)
    rank, c = 12, 40  # the first 20 rows and the last 20 hold values
    ids = np.sort(rng.integers(0, adapters, m)).astype(np.int32)
    ids[rng.integers(0, m, m // 10)] = -1
    ids[[0, m - 1]] = [0, adapters - 1]
    pick = np.r_[np.arange(c // 2), np.arange(m - c // 2, m)]
    few = ids[pick]
    x, out, dout, dx = [zeros(ctx, (m, v), np.uint16, free) for v in (k, n, n, k)]
    xs, xv = A.held(rng.standard_normal((c, k)), "bf16")
    ds, dv = A.held(rng.standard_normal((c, n)), "bf16")
    os_, ov = A.held(rng.standard_normal((c, n)), "bf16")
    as_, a = A.held(rng.standard_normal((adapters, rank, k)) / np.sqrt(k), "bf16")
    bs, b = A.held(rng.standard_normal((adapters, n, rank)), "bf16")
    s = rng.uniform(0.5, 2, adapters).astype(np.float32)
    for buf, width, v in ((x, k, xs), (dout, n, ds), (out, n, os_)):
        ends(ctx, buf, m, width, c, v)
    di, da_, db_, dsc = [ctx.upload(v) for v in (ids, as_, bs, s)]
    h, ga, gb = ctx.empty((m, rank), np.float32), ctx.empty(a.shape, np.float32), ctx.empty(b.shape, np.float32)
    sizes, lib = (m, n, k, rank, adapters), NH.lib()
    ws = ctx.empty(max(lib.nh_linear_lora_workspace_size(*sizes), lib.nh_linear_lora_backward_workspace_size(*sizes)), np.uint8)
    free.extend([di, da_, db_, dsc, h, ga, gb, ws])
    head = (x.ptr, NH.BF16, di.ptr, da_.ptr, db_.ptr, NH.BF16, dsc.ptr)
    NH.call("nh_linear_lora", ctx.handle, *head, *sizes, out.ptr, out.ptr, NH.BF16, h.ptr, ws.ptr, ws.nbytes, None)
    ctx.synchronize()
    want, _, parts = A.forward(xv, few, a, b, s, ov)
    got = A.values(read_ends(ctx, out, m, n, c))
    assert (np.abs(got - want) <= A.forward_tolerance(want, parts, k, rank, "bf16", "bf16")).all()
    assert (get(ctx, out, (m // 2) * n * 2, n, np.uint16) == 0).all()
    NH.call("nh_linear_lora_backward", ctx.handle, *head, h.ptr, dout.ptr, NH.BF16, *sizes, None, dx.ptr, ga.ptr, gb.ptr, 0,
            ws.ptr, ws.nbytes, None)
    ctx.synchronize()
    wdx, wda, wdb, parts = A.backward(xv, few, a, b, s, dv, None)
    got = A.values(read_ends(ctx, dx, m, k, c))
    assert (np.abs(got - wdx) <= A.forward_tolerance(wdx, parts, n, rank, "bf16", "bf16")).all()
    # the other rows' terms are exact zeros: at most c count
    assert (np.abs(ga.numpy() - wda) <= A.gradient_tolerance(parts, "da", n, c) + A.U * np.abs(wda)).all()
    assert (np.abs(gb.numpy() - wdb) <= A.gradient_tolerance(parts, "db", k, c) + A.U * np.abs(wdb)).all()
