"""Operands that overlap: what the sort, the rows by expert and the adapters make of them (without a GPU)."""
import numpy as np
import pytest

import nemotron_hip as NH
from dispatch import OUT, S, W, X, Recorder


@pytest.fixture
def rec():
    r = Recorder()
    yield r
    r.close()


@pytest.mark.parametrize("tokens,top_k,experts", [(1, 1, 1), (700, 4, 16), (8192, 6, 128), (9000, 3, 4096), (3, 2, 4096)])
def test_the_sort_in_place(rec, tokens, top_k, experts):
    """pos may be the ids themselves, in the one form that reads an id before anything stands in its place: the others
    would take slots and counts for experts, and write past the slots."""
    routes = 4 * tokens * top_k
    status = lambda ids, offsets, perm, pos: NH.call_status(  # noqa: E731
        "nh_moe_permute", rec.ctx, ids, tokens, top_k, experts, offsets, perm, pos, None)[0]
    assert rec.kernels("nh_moe_permute", X, tokens, top_k, experts, S, W, X, None) == ["moe_permute"]
    assert rec.kernels("nh_moe_permute", X, tokens, top_k, experts, S, W, OUT, None) != []
    assert status(X, S, W, X + routes) == status(X + routes, S, W, X) == NH.OK
    for bad in ((X, X, W, OUT), (X, S, X, OUT), (X, S, W, S), (X, W, W, OUT), (X, S, W, W), (X, S, S, X), (X, X + routes - 4, W, OUT),
                (X, S, W, S + 4 * experts)):
        assert status(*bad) == NH.INVALID_PARAMS, bad
    if tokens * top_k > 1:
        assert status(X, S, W, X + 4) == status(X + 4, S, W, X) == status(X, S, W, W + 4) == NH.INVALID_PARAMS


def test_the_sort_in_place_on_the_host():
    ids = np.array([3, 0, 3, 1, 0], np.int32)
    offsets, perm = np.zeros(5, np.int32), np.zeros(5, np.int32)
    NH.call("nh_moe_permute_host", ids.ctypes.data, 5, 1, 4, offsets.ctypes.data, perm.ctypes.data, ids.ctypes.data)
    assert offsets.tolist() == [0, 2, 3, 3, 5] and perm.tolist() == [1, 4, 3, 0, 2] and ids.tolist() == [3, 0, 4, 2, 1]


def test_the_sort_on_the_host_refuses_other_overlaps():
    buf = np.zeros(64, np.int32)
    at = lambda i: buf.ctypes.data + 4 * i  # noqa: E731
    call = lambda ids, offsets, perm, pos: NH.call_status("nh_moe_permute_host", ids, 5, 1, 4, offsets, perm, pos)[0]  # noqa: E731
    assert call(at(0), at(10), at(20), at(30)) == call(at(0), at(10), at(20), at(0)) == NH.OK
    for bad in ((0, 4, 20, 30), (0, 10, 4, 30), (0, 10, 20, 4), (0, 10, 20, 24), (0, 10, 14, 30), (0, 10, 20, 14)):
        assert call(*[at(i) for i in bad]) == NH.INVALID_PARAMS, bad


def host_status(name, *args):
    return NH.call_status(name, *args)[0]


def test_rows_on_the_host_refuse_what_the_device_refuses():
    """An output over another operand would be read where it has been written: 4 tokens, 2 routes, 3 wide, 8 slots in f32."""
    buf = np.zeros(1024, np.float32)
    pos = np.arange(8, dtype=np.int32)
    a = lambda i: buf.ctypes.data + 4 * i  # noqa: E731
    p, size, f = pos.ctypes.data, (4, 2, 3, 8), NH.F32
    x, rows, w, out, dw = a(0), a(100), a(200), a(300), a(400)
    near = (-4, 0, 4)

    def dispatch(to):
        return host_status("nh_moe_dispatch_host", x, f, p, w, *size, to, f)

    def dispatch_back(dx, dweights, with_x=x):
        return host_status("nh_moe_dispatch_backward_host", rows, f, with_x, f, p, w, *size, dx, dweights)

    def combine(to, shared):
        return host_status("nh_moe_combine_rows_host", rows, f, p, w, shared, *size, to, f)

    def combine_back(drows, dweights, y=rows):
        return host_status("nh_moe_combine_rows_backward_host", x, f, y, f, p, w, *size, drows, dweights)

    assert dispatch(rows) == dispatch_back(out, dw) == combine(out, x) == combine(out, None) == combine_back(out, dw) == NH.OK
    for d in near:
        assert dispatch(x + d) == dispatch(w + d) == NH.INVALID_PARAMS
        assert dispatch_back(rows + d, dw) == dispatch_back(x + d, dw) == dispatch_back(w + d, dw) == NH.INVALID_PARAMS
        assert dispatch_back(out, x + d) == dispatch_back(out, w + d) == dispatch_back(out, out + d) == NH.INVALID_PARAMS
        assert combine(rows + d, None) == combine(w + d, None) == NH.INVALID_PARAMS
        assert combine_back(x + d, dw) == combine_back(w + d, dw) == combine_back(out, out + d) == NH.INVALID_PARAMS
        assert (combine(x + d, x) == NH.OK) == (combine_back(rows + d, dw) == NH.OK) == (d == 0)
    assert dispatch_back(x, None, None) == combine_back(rows + 4, None, None) == NH.OK  # not asked for


def test_adapters_on_the_host_refuse_what_the_device_refuses():
    """3 rows of two adapters, 5 -> 4 wide, rank 2, in f32."""
    buf = np.zeros(2048, np.float32)
    ids = np.array([0, 1, -1], np.int32)
    at = lambda i: buf.ctypes.data + 400 * i  # noqa: E731
    x, a, b, s, base, out, h, dout, dx, da, db = [at(i) for i in range(11)]
    size, f, i = (3, 4, 5, 2, 2), NH.F32, ids.ctypes.data

    def forward(to=out, on=base, low=h):
        return host_status("nh_linear_lora_host", x, f, i, a, b, f, s, *size, on, to, f, low)

    def backward(to=dx, on=base, ga=da, gb=db, low=h):
        return host_status("nh_linear_lora_backward_host", x, f, i, a, b, f, s, low, dout, f, *size, on, to, ga, gb, 0)

    assert forward() == forward(on=None, low=None) == forward(to=base) == NH.OK
    assert backward() == backward(on=None, low=None) == backward(to=base) == NH.OK
    for other in (x, a, b, s):
        for d in (-4, 0, 4):
            assert forward(to=other + d) == forward(low=other + d) == NH.INVALID_PARAMS
            assert backward(to=other + d) == backward(ga=other + d) == backward(gb=other + d) == NH.INVALID_PARAMS
    assert forward(to=base + 4) == forward(low=base) == forward(low=out) == backward(to=base + 4) == NH.INVALID_PARAMS
    for d in (dout, h):
        assert backward(to=d) == backward(ga=d) == backward(gb=d) == NH.INVALID_PARAMS
    assert backward(ga=dx) == backward(gb=dx) == backward(ga=db) == NH.INVALID_PARAMS
