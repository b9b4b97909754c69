"""Which form of an MXFP4 operator a size takes, on both sides of each rule (without a GPU)."""
import pytest

import nemotron_hip as NH
from dispatch import OUT, S, W, W2, WS, X, Recorder


@pytest.fixture(scope="module")
def rec():
    r = Recorder()
    yield r
    r.close()


# Rows of codes: streamed where K is long and the columns few, 32 or 64 rows a pass; else the GEMM.
@pytest.mark.parametrize("m,n,k,kernel", [
    (17, 4096, 2048, "mx_gemm_64x64"), (17, 4096, 2049, "mx_stream_tok4_32"), (32, 32768, 4096, "mx_stream_tok4_32"),
    (32, 32768, 8192, "mx_stream_tok8_32"), (32, 4096, 8193, "mx_gemm_64x64"), (33, 8192, 4096, "mx_stream_tok4_64"),
    (33, 8193, 4096, "mx_gemm_64x64"), (64, 8192, 2049, "mx_stream_tok4_64"), (64, 4096, 4097, "mx_stream_tok8_32"),
    (64, 4097, 4097, "mx_gemm_64x64"), (64, 4096, 1024, "mx_gemm_64x64"), (65, 4096, 4096, "mx_gemm_64x64"),
    (16, 4096, 1024, "mx_stream_bf16_2"), (16, 4096, 4096, "mx_stream_bf16_4")])
def test_streamed_or_tiled(rec, m, n, k, kernel):
    ws = NH.lib().nh_linear_mxfp4_workspace_size(m, n, k)
    launches = rec.kernels("nh_linear_mxfp4", X, NH.BF16, W, None, m, n, k, OUT, NH.BF16, WS if ws else None, ws, None, None)
    assert launches == (["quantize_mxfp4_tiles"] if ws else []) + [kernel]


# The MoE layer's routes: sorted by the workgroup that routes them, one turn of 16 tokens and 64 routes at most.
@pytest.mark.parametrize("t,k,inside", [(1, 64, True), (8, 8, True), (16, 4, True), (16, 5, False), (17, 1, False), (8, 9, False),
                                        (32, 2, False)])
def test_routes_sorted_in_the_first_launch(rec, t, k, inside):
    ws = NH.lib().nh_moe_forward_mxfp4_workspace_size(t, 512, 256, 128, k)
    launches = rec.launches("nh_moe_forward_mxfp4", X, NH.F32, S, t, 512, 256, 128, k, 1, 1.0, W, W2, None, None, OUT, NH.F32, WS,
                            ws, None, None)
    assert launches[0][0] == "mx_moe_prep" and ("permute" in launches[1][0]) == (not inside)
    assert launches[0][1] == (1 if inside else -(-t // 16)) + -(--(-t // 16) // 4)


# The balance loss: one workgroup for few logits and routes of one sequence.
@pytest.mark.parametrize("t,e,k,one", [(256, 128, 8, True), (257, 128, 8, False), (4096, 8, 4, True), (4096, 8, 5, False),
                                       (16384, 1, 1, True), (16385, 1, 1, False), (32, 1024, 8, True), (0, 1024, 8, True)])
def test_balance_in_one_workgroup(rec, t, e, k, one):
    ws = NH.lib().nh_moe_balance_loss_workspace_size(1, t, e)
    launches = rec.kernels("nh_moe_balance_loss", X, W, None, 1, t, e, k, 0, 0.1, OUT, S, WS, ws, None)
    assert launches == ["moe_balance_partial"] + ([] if one else ["moe_balance_reduce"])
