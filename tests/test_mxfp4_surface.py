"""What the MXFP4 and balance entry points have in common with the library's others (without a GPU)."""
import ctypes as C
import os
import re

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
