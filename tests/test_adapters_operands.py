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
