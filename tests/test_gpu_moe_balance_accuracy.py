"""How far the router's balance loss and gradient may be off where single roundings show: values that the kernels hold
exactly but for the one that is looked at."""
import numpy as np
import pytest

import mx_reference as R
import nemotron_hip as NH
from test_gpu_moe_balance import run
from test_gpu_mxfp4 import U, note

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = NH.Context(0)
    yield c
    c.close()


def test_chunks_are_added_in_64_bits(ctx):
    """32768 tokens of 1024 experts in 256 chunks of 128, every route to expert 0.  One token of a chunk is uniform
    (p = 2^-10, exactly), the others have expert 0 alone (p = 1): a chunk's sum is 127 + 2^-10, which f32 holds, and 256
    of them 32512.25, which it holds too.  Added in f32, a step past 16384 is 2^-9 and half of it is lost each time:
    0.12 of 32512, 64 half steps.  In 64 bits only the loss is rounded."""
    t, e = 32768, 1024
    note("balance chunk sums")
    z = np.full((t, e), -np.inf, np.float32)
    z[:, 0] = 0
    z[::128] = 0
    loss = run(ctx, z, np.zeros((t, 1), np.int32), None, 1, coefficient=1.0)[1]
    want = e / t * 256 * (127 + 2.0 ** -10)  # E / (k T^2) * counts_0 * sum p_0
    assert abs(float(loss) - want) <= U * want
