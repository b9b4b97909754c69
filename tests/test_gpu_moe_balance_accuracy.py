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


@pytest.mark.parametrize("softmax", [0, 1])
def test_exp_of_far_logits(ctx, softmax):
    """Rows of two experts, 0 and -z: p_1 is e^-z (twice that for sigmoids) to 2^-36 of it, and with every route to expert
    0 its gradient is -2 e^-z, the other factors and sums being powers of two that nothing rounds.  So the gradient is
    off by what the exponential is: 1 ulp (two half steps) of the instruction and one rounding, however large z is; an
    argument that is rounded first is off by up to z half steps."""
    t = 256
    note(f"balance exp softmax={softmax}")
    z = np.zeros((t, 2), np.float32)
    z[:, 1] = -np.linspace(25, 80, t)
    idx = np.zeros((t, 1), np.int32)
    grad = run(ctx, z, idx, None, softmax, coefficient=1.0, dloss=256.0)[2]
    want = R.balance(z, idx, None, softmax, 1.0, 256.0)[2]
    assert (np.abs(grad[:, 1] - want[:, 1]) <= 3.01 * U * np.abs(want[:, 1])).all()


def test_sigmoids_over_their_sum(ctx):
    """Rows of 16 sigmoids of ordinary logits, every route to expert 0 of an f of 16: p_e f is the gradient's size, and
    p_e is off by the exponential (3 half steps, of a term that is at most half of 1 + t, so 1.5), 1 + t (1), the
    reciprocal (2), the product with t (3 + 1), the sum of 16 (4 additions of a lane and 2 lane moves, 6, and what each
    term has), its reciprocal (2) and the last product (1)."""
    t, e = 512, 16
    note("balance sigmoids")
    rng = np.random.default_rng(0)
    z = (rng.standard_normal((t, e)) * 2).astype(np.float32)
    idx = np.zeros((t, 1), np.int32)
    grad = run(ctx, z, idx, None, 0, coefficient=1.0, dloss=512.0)[2]
    want = R.balance(z, idx, None, 0, 1.0, 512.0)[2]
    term = 1.5 + 1 + 2 + 4
    p = 2 * term + 6 + 3
    # the others' gradient: -16 p_0 p_e d_e, three products, and d = r t or r
    others = 2 * p + 3 + term
    assert (np.abs(grad - want)[:, 1:] <= others * U * np.abs(want[:, 1:])).all()
