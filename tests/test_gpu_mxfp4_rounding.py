"""The device's conversion to MXFP4 against the definition, value by value."""
import numpy as np
import pytest

import mx_reference as R
import nemotron_hip as NH
from test_gpu_mxfp4 import note, quantize

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = NH.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("rise", range(9))
def test_every_bf16_value_under_every_scale(ctx, rise):
    """Each finite bf16 beside a power of two of its own exponent and `rise` above: with 5 and more it is below a quarter
    of the scale and rounds to zero, so these are all scales that matter."""
    note(f"every bf16, rise {rise}")
    bits = np.arange(65536, dtype=np.uint32)
    bits = bits[(bits & 0x7F80) != 0x7F80]
    x = np.zeros((bits.size, 32), np.uint16)
    x[:, 1] = x[:, 30] = bits
    x[:, 8] = np.minimum((bits & 0x7F80) + (rise << 7), 0x7F00)
    codes, scales = quantize(ctx, x, NH.BF16)
    rc, rs, _ = R.quantize(R.from_bf16_bits(x))
    assert np.array_equal(scales.numpy(), rs) and np.array_equal(codes.numpy(), rc)


@pytest.mark.parametrize("seed", range(4))
def test_f32_values_of_all_exponents(ctx, seed):
    """2^22 values in blocks whose largest has any exponent: random mantissas down to 2^-12 of it, and the midpoints of the
    grid with their neighbours."""
    note(f"f32 sweep {seed}")
    rng = np.random.default_rng(seed)
    blocks = (1 << 22) // 32
    top = rng.integers(0, 255, blocks)  # the exponent field
    top[:255] = np.arange(255)
    field = np.maximum(top[:, None] - rng.integers(0, 13, (blocks, 32)), 0).astype(np.uint32)
    bits = (field << 23) | rng.integers(0, 1 << 23, (blocks, 32)).astype(np.uint32)
    with np.errstate(over="ignore"):
        tie = np.ldexp(rng.choice(R.MIDDLE, (blocks, 32)), np.maximum(top, 2)[:, None] - 2 - 127).astype(np.float32)
    tie = np.where(np.isfinite(tie), tie, 0).astype(np.float32).view(np.uint32)
    tie = np.maximum(tie.astype(np.int64) + rng.integers(-1, 2, (blocks, 32)), 0).astype(np.uint32)
    bits = np.where(rng.random((blocks, 32)) < 0.5, bits, tie)
    bits[:, 0] = (top.astype(np.uint32) << 23) | (bits[:, 0] & 0x7FFFFF)  # the largest has this exponent
    x = (bits | (rng.integers(0, 2, bits.shape).astype(np.uint32) << 31)).view(np.float32)
    x = np.where(np.isfinite(x), x, np.float32(1)).astype(np.float32)
    codes, scales = quantize(ctx, x, NH.F32)
    rc, rs, _ = R.quantize(x)
    assert np.array_equal(scales.numpy(), rs) and np.array_equal(codes.numpy(), rc)
