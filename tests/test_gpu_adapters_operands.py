"""The sort with pos over its ids, and the adapters' workspaces at their ends."""
import numpy as np
import pytest

import nemotron_hip as NH
from test_gpu_mxfp4 import Guarded, note

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = NH.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (700, 16, 3), (1500, 128, 8), (9000, 128, 4), (7000, 4096, 3), (33000, 600, 5)])
def test_sort_in_place(ctx, t, e, k):
    note(f"permute in place t={t} e={e} k={k}")
    rng = np.random.default_rng(t)
    ids = rng.integers(0, e, t * k).astype(np.int32)
    if t > 1:
        ids[rng.integers(0, t * k, 9)] = rng.choice([-1, e, 2 ** 31 - 1, -2 ** 31])
    outs = [Guarded(ctx, (n,), np.int32) for n in (e + 1, t * k, t * k)]
    outs[2].buf.copy_from(np.concatenate([np.full(outs[2].at, 0xA5, np.uint8), ids.view(np.uint8), np.full(256, 0xA5, np.uint8)]))
    NH.call("nh_moe_permute", ctx.handle, outs[2].ptr, t, k, e, *[o.ptr for o in outs], None)
    off, perm, pos = [o.numpy() for o in outs]
    valid = (ids >= 0) & (ids < e)
    order = np.flatnonzero(valid)[np.argsort(ids[valid], kind="stable")]
    where = np.full(t * k, -1)
    where[order] = np.arange(order.size)
    assert np.array_equal(off, np.concatenate([[0], np.cumsum(np.bincount(ids[valid], minlength=e))]))
    assert np.array_equal(perm[:order.size], order) and np.array_equal(pos, where)
