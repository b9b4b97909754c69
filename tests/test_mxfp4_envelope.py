"""The sizes that the MXFP4 entry points accept are sizes that they can launch (without a GPU)."""
import random

import pytest

import nemotron_hip as NH
from dispatch import OUT, S, W, W2, WS, X, Recorder

@pytest.fixture(scope="module")
def rec():
    r = Recorder()
    yield r
    r.close()


def workgroup(kernel):
    """Its threads, or more."""
    return 256 if "quantize" in kernel or "combine" in kernel else 512 if kernel.startswith("mx_stream") or "gemm" in kernel else 1024


def sizes(rng, top):
    """1 .. 2^top, powers of two and their neighbours among them."""
    v = 1 << rng.randrange(top + 1)
    return max(1, rng.choice([v, v - 1, v + 1, rng.randint(1, v)]))


def test_moe_prep_fits_a_launch(rec):
    """2^26 tokens: 5242880 workgroups of 1024 threads, past the 2^32 of a launch."""
    supports = NH.lib().nh_supports_moe_forward_mxfp4
    assert supports(1 << 26, 32, 32, 2, 1) == 0
    size = NH.lib().nh_moe_forward_mxfp4_workspace_size(1 << 26, 32, 32, 2, 1)
    st, err = NH.call_status("nh_moe_forward_mxfp4", rec.ctx, X, NH.F32, S, 1 << 26, 32, 32, 2, 1, 1, 1.0, W, W2, None, None,
                             OUT, NH.F32, WS, size, None, None)
    assert st == NH.UNSUPPORTED
    # the most: 16 * 2^22 * 4 / 5 tokens of up to 512 columns, less one workgroup
    most = max(t for t in range(53687000, 53687200) if supports(t, 512, 32, 2, 1))
    blocks = lambda t: (t + 15) // 16 + ((t + 15) // 16 + 3) // 4  # noqa: E731
    assert blocks(most) < 1 << 22 <= blocks(most + 1)
    # the flat index of an intermediate value: 38 bits of the non-finite word
    assert supports(1 << 19, 32, 8192, 128, 63) == 1 and supports(1 << 19, 32, 8192, 128, 64) == 0


def test_linear_quantization_fits_a_launch():
    supports = NH.lib().nh_supports_linear_mxfp4
    assert supports((1 << 24) - 1, 16, 512 * 15) == 1 and supports((1 << 24) - 1, 16, 512 * 15 + 1) == 0
    assert NH.lib().nh_linear_mxfp4_workspace_size((1 << 24) - 1, 16, 512 * 15 + 1) == 0


def test_conversions_fit_a_launch():
    def both(rows, cols):
        a = NH.call_status("nh_quantize_rows_mxfp4", None, X, NH.BF16, rows, cols, OUT, S, None, None)
        b = NH.call_status("nh_dequantize_mxfp4", None, X, S, rows, cols, OUT, NH.BF16, None)
        assert a[0] == b[0]
        return a[0], a[1].message
    blocks = (1 << 32) - 256
    assert both(blocks // 2, 64)[1] == both(blocks // 2, 33)[1] == b"null context"
    assert both(blocks // 2 + 1, 64)[0] == both(blocks // 2 + 1, 33)[0] == NH.UNSUPPORTED
    assert both(1 << 20, 1 << 20)[0] == NH.UNSUPPORTED


def test_accepted_sizes_launch(rec):
    rng = random.Random(1)
    lib, seen = NH.lib(), set()
    for _ in range(20000):
        t, h, i, e = sizes(rng, rng.choice([21, 30])), sizes(rng, 13), sizes(rng, 13), sizes(rng, 10)
        k = min(e, sizes(rng, 6))
        launches = []
        if lib.nh_supports_moe_forward_mxfp4(t, h, i, e, k):
            ws = lib.nh_moe_forward_mxfp4_workspace_size(t, h, i, e, k)
            args = (X, NH.F32, S, t, h, i, e, k, 1, 1.0, W, W2, None, None, OUT, NH.F32, WS, ws, None, None)
            if t <= 50 * 65535:  # the recorder keeps 64 launches, the combine has one per 65535 tokens
                launches += rec.launches("nh_moe_forward_mxfp4", *args)
        m, n, k = sizes(rng, 24), sizes(rng, 28), sizes(rng, 17)
        if lib.nh_supports_linear_mxfp4(m, n, k):
            ws = lib.nh_linear_mxfp4_workspace_size(m, n, k)
            far = 1 << 60  # an output that no rows reach into
            launches += rec.launches("nh_linear_mxfp4", X, NH.BF16, W, None, m, n, k, far, NH.BF16, WS if ws else None, ws,
                                     None, None)
        rows, cols = sizes(rng, 31), sizes(rng, 31)
        if NH.call_status("nh_quantize_rows_mxfp4", rec.ctx, X, NH.F32, rows, cols, OUT, S, None, None)[0] == NH.OK:
            launches += rec.launches("nh_dequantize_mxfp4", X, S, rows, cols, OUT, NH.F32, None)
        for kernel, gx, gy in launches:
            assert gx * workgroup(kernel) < 1 << 32 and gy <= 65535, (kernel, gx, gy)
            seen.add(kernel)
    assert {"mx_moe_prep", "quantize_mxfp4_tiles", "dequantize_mxfp4", "mx_gemm_64x64"} <= seen


@pytest.mark.parametrize("hidden", [40, 41])
def test_combine_of_more_tokens_than_a_grid_has_rows(rec, hidden):
    for tokens, rows in ((1, [1]), (65535, [65535]), (65536, [65535, 1]), (200000, [65535] * 3 + [3395])):
        launches = rec.launches("nh_moe_combine", X, W, S, tokens, 1, hidden, OUT, NH.F32, None)
        assert [v[1:] for v in launches] == [(1, r) for r in rows]
