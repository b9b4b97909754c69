"""What the MXFP4 and balance entry points have in common with the library's others (without a GPU)."""
import ctypes as C
import os
import re

import numpy as np

import nemotron_hip as NH

HEADER = os.path.join(os.path.dirname(__file__), "..", "include", "nemotron_hip.h")


def test_registry_lists_every_entry_point():
    lib, names = NH.lib(), {}
    for i in range(lib.nh_kernel_count()):
        backend = C.c_int(-1)
        name = lib.nh_kernel_name(i, C.byref(backend)).decode()
        names[name] = backend.value
    entries = re.findall(r"^nh_status nh_(\w*(?:mxfp4|balance)\w*)\(", open(HEADER).read(), re.M)
    assert len(entries) == 14
    for e in entries:
        assert names.get(e) == (0 if e.endswith("_host") else 1), e


def test_host_twins_refuse_null_operands():
    """As the device's entry points do; the operands that a call has no use for may be NULL."""
    t, h, i, e, k = 4, 64, 32, 8, 2
    keep = [np.zeros(1 << 16, d) for d in (np.float32, np.float32, np.uint8, np.uint8, np.int32, np.float32)]
    f, out, b, s, ids, up = (v.ctypes.data for v in keep)
    size = NH.lib().nh_tiled_mxfp4_weights_bytes(t, h)

    def refused(name, args, operands):
        for at in operands:
            st, err = NH.call_status(name, *(None if n == at else v for n, v in enumerate(args)))
            assert st == NH.INVALID_PARAMS and err.message == b"null operand", (name, at)
        assert NH.call_status(name, *args)[0] == NH.OK, name

    refused("nh_quantize_rows_mxfp4_host", (f, NH.F32, t, h, b, s), (0, 4, 5))
    refused("nh_dequantize_mxfp4_host", (b, s, t, h, out, NH.F32), (0, 1, 4))
    refused("nh_tile_weights_mxfp4_host", (b, s, t, h, out, size), (0, 1, 4))
    refused("nh_linear_mxfp4_host", (f, NH.F32, b, None, t, 16, h, out, NH.F32), (0, 2, 7))
    refused("nh_moe_forward_mxfp4_host", (f, NH.F32, f, t, h, i, e, k, 1, 1.0, b, b, None, None, out, NH.F32), (0, 2, 10, 11, 14))
    refused("nh_moe_balance_loss_host", (f, ids, None, 1, t, e, k, 0, 0.1, s, out), (0, 1, 9, 10))
    refused("nh_moe_balance_loss_backward_host", (f, ids, None, 1, t, e, k, 0, 0.1, up, out), (0, 1, 9, 10))
    assert NH.call_status("nh_quantize_rows_mxfp4_host", None, NH.F32, 0, h, None, None)[0] == NH.OK
    assert NH.call_status("nh_dequantize_mxfp4_host", None, None, t, 0, None, NH.F32)[0] == NH.OK
    assert NH.call_status("nh_moe_balance_loss_host", None, None, None, 1, 0, e, k, 0, 0.1, s, out)[0] == NH.OK
    assert NH.call_status("nh_moe_balance_loss_backward_host", None, None, None, 1, 0, e, k, 0, 0.1, None, None)[0] == NH.OK


def test_balance_has_an_envelope():
    """nh_supports_moe_balance_loss is 1 exactly where neither call is refused, and where the workspace has a size."""
    lib = NH.lib()
    p = 1 << 40  # an operand that no call here gets to: there is no context
    for s, t, e, k in ((1, 64, 8, 2), (16384, 1 << 20, 1024, 8), (16385, 64, 8, 2), (1, 64, 1025, 2), (1, 1 << 30, 8, 1),
                       (1, (1 << 30) - 1, 8, 2), (1, (1 << 30) - 1, 8, 3), (1, 0, 8, 2), (1, 64, 8, 1024), (1, 64, 8, 1025),
                       (0, 64, 8, 2), (1, 64, 0, 2), (1, 64, 8, 0), (2, (1 << 64) - 1, 1, 1)):
        yes = lib.nh_supports_moe_balance_loss(s, t, e, k)
        size = lib.nh_moe_balance_loss_workspace_size(s, t, e)
        a = NH.call_status("nh_moe_balance_loss", None, p, p, p, s, t, e, k, 0, 0.1, p, p, p, size, None)
        b = NH.call_status("nh_moe_balance_loss_backward", None, p, p, p, s, t, e, k, 0, 0.1, p, p, None)
        for st, err in (a, b):
            if yes:
                assert size > 0 and err.message == b"null context", (s, t, e, k)
            else:
                assert st in (NH.UNSUPPORTED, NH.INVALID_SHAPE) and err.message != b"null context", (s, t, e, k)


def test_rust_comments_are_the_headers():
    """Each MXFP4 and balance declaration of the Rust crate stands under its header comment, word for word."""
    words = lambda t: re.findall(r"\w+", t)  # noqa: E731
    header, crate = open(HEADER).read(), open(os.path.join(os.path.dirname(HEADER), "..", "rust", "nemotron-hip-sys", "src",
                                                           "lib.rs")).read()
    comments = re.findall(r"/\*((?:[^*]|\*(?!/))*)\*/\n[^;{}/]*?\b(nh_\w*(?:mxfp4|balance)\w*)\s*\(", header)
    assert len(comments) > 10
    for text, name in comments:
        rust = re.search(r"((?:    ///[^\n]*\n)+)    pub fn " + name + r"\b", crate)
        assert rust, name
        assert words(rust.group(1)) == words(re.sub(r"\n \*", "\n", text)), name
