"""The host twins of the rows by expert and of the low-rank adapters against plain 64-bit forms, what the entry points
refuse, and the envelopes (without a GPU)."""
import ctypes as C
import os
import random
import re

import numpy as np
import pytest

import adapters_reference as A
import nemotron_hip as NH
from dispatch import OUT, S, W, W2, WS, X, Recorder

HEADER = os.path.join(os.path.dirname(__file__), "..", "include", "nemotron_hip.h")
DT = {"f32": NH.F32, "bf16": NH.BF16}
ptr = lambda a: None if a is None else a.ctypes.data  # noqa: E731


@pytest.fixture
def rec():
    r = Recorder()
    yield r
    r.close()


# ---- host twins -------------------------------------------------------------------

@pytest.mark.parametrize("t,k,h", [(1, 1, 1), (5, 3, 9), (7, 10, 20)])
@pytest.mark.parametrize("token,row", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("weights", [True, False])
def test_rows_host(t, k, h, token, row, weights):
    rng = np.random.default_rng(t)
    slots = t * k + 2
    pos = rng.permutation(slots)[:t * k].reshape(t, k).astype(np.int32)
    if t > 1:
        pos[1, 0], pos[2, 1] = -1, slots
    w = rng.uniform(-1, 1, (t, k)).astype(np.float32) if weights else None
    x, vx = A.held(rng.standard_normal((t, h)), token)
    y, vy = A.held(rng.standard_normal((slots, h)), row)
    shared, vs = A.held(rng.standard_normal((t, h)), token)
    size = (t, k, h, slots)
    rows, out, dw = A.empty((slots, h), row), A.empty((t, h), token), np.zeros((t, k), np.float32)
    NH.call("nh_moe_dispatch_host", ptr(x), DT[token], ptr(pos), ptr(w), *size, ptr(rows), DT[row])
    want, touched, _, _ = A.scatter(vx, pos, w, slots)
    tol = 1.01 * (A.HALF[row] + A.U) * np.abs(want)
    assert (np.abs(A.values(rows) - want) <= tol).all() and (A.values(rows)[~touched] == 0).all()
    NH.call("nh_moe_dispatch_backward_host", ptr(y), DT[row], ptr(x), DT[token], ptr(pos), ptr(w), *size, ptr(out), ptr(dw))
    want, total, g, g_abs = A.gather(vy, pos, w, dot=vx)
    assert (np.abs(A.values(out) - want) <= 1.01 * (A.HALF[token] + A.U) * np.abs(want) + 1e-40).all()
    assert (np.abs(dw - g) <= A.U * np.abs(g) + 1e-40).all()
    NH.call("nh_moe_combine_rows_host", ptr(y), DT[row], ptr(pos), ptr(w), ptr(shared), *size, ptr(out), DT[token])
    want, _, _, _ = A.gather(vy, pos, w, shared=vs)
    assert (np.abs(A.values(out) - want) <= 1.01 * (A.HALF[token] + A.U) * np.abs(want) + 1e-40).all()
    rows[:] = 0
    NH.call("nh_moe_combine_rows_backward_host", ptr(x), DT[token], ptr(y), DT[row], ptr(pos), ptr(w), *size, ptr(rows), ptr(dw))
    want, touched, g, _ = A.scatter(vx, pos, w, slots, rows=vy)
    assert (np.abs(A.values(rows) - want) <= 1.01 * (A.HALF[row] + A.U) * np.abs(want)).all()
    assert (np.abs(dw - g) <= A.U * np.abs(g) + 1e-40).all()


def lora_inputs(m, n, k, rank, adapters, x, w, out, seed):
    rng = np.random.default_rng(seed)
    ids = rng.integers(-1, adapters + 1, m).astype(np.int32)
    stored, exact = {}, {}
    for name, shape, d in (("x", (m, k), x), ("a", (adapters, rank, k), w), ("b", (adapters, n, rank), w), ("base", (m, n), out),
                           ("dout", (m, n), out), ("dx_base", (m, k), x)):
        stored[name], exact[name] = A.held(rng.standard_normal(shape), d)
    return ids, stored, exact, rng.uniform(-2, 2, adapters).astype(np.float32)


@pytest.mark.parametrize("m,n,k,rank,adapters", [(1, 1, 1, 1, 1), (9, 7, 5, 3, 2), (20, 33, 18, 130, 4)])
@pytest.mark.parametrize("x,w,out", [("bf16", "bf16", "bf16"), ("f32", "f32", "f32"), ("bf16", "f32", "bf16"),
                                     ("f32", "bf16", "f32")])
def test_lora_host(m, n, k, rank, adapters, x, w, out):
    ids, st, v, s = lora_inputs(m, n, k, rank, adapters, x, w, out, m + rank)
    size = (m, n, k, rank, adapters)
    y, h = A.empty((m, n), out), np.zeros((m, rank), np.float32)
    NH.call("nh_linear_lora_host", ptr(st["x"]), DT[x], ptr(ids), ptr(st["a"]), ptr(st["b"]), DT[w], ptr(s), *size,
            ptr(st["base"]), ptr(y), DT[out], ptr(h))
    want, wh, parts = A.forward(v["x"], ids, v["a"], v["b"], s, v["base"])
    # h is rounded once, out once in f32 and once to its type
    assert (np.abs(h - wh) <= A.U * np.abs(wh) + 1e-40).all()
    assert (np.abs(A.values(y) - want) <= 1.01 * ((A.HALF[out] + A.U) * np.abs(want) + A.U * parts["low"]) + 1e-40).all()
    dx, da, db = A.empty((m, k), x), np.full((adapters, rank, k), 3.0, np.float32), np.full((adapters, n, rank), 3.0, np.float32)
    wdx, wda, wdb, parts = A.backward(v["x"], ids, v["a"], v["b"], s, v["dout"], v["dx_base"])
    for given, accumulate in ((h, 0), (None, 1)):
        before = (da.astype(np.float64), db.astype(np.float64)) if accumulate else (0.0, 0.0)
        NH.call("nh_linear_lora_backward_host", ptr(st["x"]), DT[x], ptr(ids), ptr(st["a"]), ptr(st["b"]), DT[w], ptr(s),
                ptr(given), ptr(st["dout"]), DT[out], *size, ptr(st["dx_base"]), ptr(dx), ptr(da), ptr(db), accumulate)
        assert (np.abs(A.values(dx) - wdx) <= 1.01 * ((A.HALF[x] + A.U) * np.abs(wdx) + A.U * parts["low"]) + 1e-40).all()
        for got, g, low, b in ((da, wda, parts["da_low"], before[0]), (db, wdb, parts["db_low"], before[1])):
            assert (np.abs(got - (g + b)) <= 1.01 * A.U * (np.abs(g + b) + 2 * low) + 1e-40).all()


def test_lora_host_gradients_are_differences():
    """out is linear in x, a and b each: a central difference along any direction is exact but for f32's roundings."""
    m, n, k, rank, adapters = 12, 9, 11, 3, 2
    ids, st, v, s = lora_inputs(m, n, k, rank, adapters, "f32", "f32", "f32", 3)
    dx, da, db = np.zeros((m, k), np.float32), np.zeros((adapters, rank, k), np.float32), np.zeros((adapters, n, rank), np.float32)
    NH.call("nh_linear_lora_backward_host", ptr(st["x"]), NH.F32, ptr(ids), ptr(st["a"]), ptr(st["b"]), NH.F32, ptr(s), None,
            ptr(st["dout"]), NH.F32, m, n, k, rank, adapters, None, ptr(dx), ptr(da), ptr(db), 0)
    rng = np.random.default_rng(4)
    for name, grad in (("x", dx), ("a", da), ("b", db)):
        d = rng.standard_normal(grad.shape)
        f = [A.forward(**{**{q: v[q] for q in "xab"}, name: v[name] + e * d}, ids=ids, s=s, base=None)[0] for e in (1.0, -1.0)]
        diff = (v["dout"] * (f[0] - f[1])).sum() / 2
        assert abs((grad * d).sum() - diff) <= 8 * A.U * (np.abs(grad) * np.abs(d)).sum()


# ---- refusals ---------------------------------------------------------------------

P1, P2, P3, P4, P5 = (i << 44 for i in range(1, 6))  # operands apart from each other
ROWS = {  # arguments after the context; positions of operands, dtypes and sizes
    "nh_moe_dispatch": ([P1, NH.BF16, P2, P3, 4, 2, 64, 8, P4, NH.BF16], (0, 2, 8), (1, 9)),
    "nh_moe_dispatch_backward": ([P1, NH.BF16, P2, NH.BF16, P3, None, 4, 2, 64, 8, P4, P5], (0, 2, 4, 10), (1, 3)),
    "nh_moe_combine_rows": ([P1, NH.BF16, P2, P3, None, 4, 2, 64, 8, P4, NH.BF16], (0, 2, 9), (1, 10)),
    "nh_moe_combine_rows_backward": ([P1, NH.BF16, P2, NH.BF16, P3, None, 4, 2, 64, 8, P4, P5], (0, 2, 4, 10), (1, 3)),
}


@pytest.mark.parametrize("name", ROWS)
def test_rows_refusals(rec, name):
    args, operands, dtypes = ROWS[name]
    size = args.index(4)  # tokens, top_k, hidden, slots

    def status(*changes):
        a = list(args)
        for at, v in changes:
            a[at] = v
        return NH.call_status(name, rec.ctx, *a, None)[0]
    assert status() == NH.OK
    for at in operands:
        assert status((at, None)) == NH.INVALID_PARAMS
    for at in dtypes:
        assert status((at, 2)) == NH.INVALID_PARAMS
    for at in (size + 1, size + 2):
        assert status((at, 0)) == NH.INVALID_SHAPE
    big = ((size, 1 << 31), (size, 1 << 62), (size + 1, 1 << 30), (size + 2, 1 << 31), (size + 2, 1 << 38), (size + 3, 1 << 31),
           (size + 3, (1 << 34)))
    for change in big:
        assert status(change) == NH.UNSUPPORTED, change
    assert NH.call_status(name, None, *args, None)[0] == NH.INVALID_PARAMS
    # an output over an input: 4 x 64 and 8 x 64 values of two bytes
    out, first = size + 4, args[0]
    assert status((out, first)) == NH.INVALID_PARAMS and status((out, first + 64)) == NH.INVALID_PARAMS
    assert status((out, first + 4096)) == NH.OK
    if name == "nh_moe_combine_rows_backward":
        assert status((out, args[2])) == NH.OK and status((out, args[2] + 2)) == NH.INVALID_PARAMS
        assert status((out, args[2] + 2), (out + 1, None), (2, None)) == NH.OK
    if name == "nh_moe_dispatch_backward":
        assert status((out, args[2])) == NH.INVALID_PARAMS and status((2, None), (out + 1, None)) == NH.OK
    for at in range(size):  # over positions and weights, and a second output over anything
        if args[at] in (P1, P2, P3) and (name, at) != ("nh_moe_combine_rows_backward", 2):
            assert status((out, args[at])) == NH.INVALID_PARAMS
        if name.endswith("_backward") and args[at] in (P1, P2, P3):
            assert status((out + 1, args[at])) == NH.INVALID_PARAMS
    if name.endswith("_backward"):
        assert status((out + 1, P4)) == NH.INVALID_PARAMS and status((5, P5)) == NH.INVALID_PARAMS
    if name == "nh_moe_combine_rows":
        assert status((4, P4)) == NH.OK and status((4, P4 + 2)) == NH.INVALID_PARAMS
    host = [a for a in args]
    host[size] = 0
    assert NH.call_status(name + "_host", *host)[0] == NH.OK
    for at in operands:
        host = [None if i == at else a for i, a in enumerate(args)]
        assert NH.call_status(name + "_host", *host)[0] == NH.INVALID_PARAMS


def lora_args(m, n, k, rank, adapters, ws=None, **over):
    need = NH.lib().nh_linear_lora_workspace_size(m, n, k, rank, adapters) if ws is None else ws
    a = dict(x=X, xd=NH.BF16, ids=S, a=W, b=W2, wd=NH.BF16, s=None, m=m, n=n, k=k, rank=rank, adapters=adapters, base=P4, out=OUT,
             od=NH.BF16, h=None, ws=WS, wsb=need, stream=None)
    a.update(over)
    return list(a.values())


def back_args(m, n, k, rank, adapters, ws=None, **over):
    need = NH.lib().nh_linear_lora_backward_workspace_size(m, n, k, rank, adapters) if ws is None else ws
    a = dict(x=X, xd=NH.BF16, ids=S, a=W, b=W2, wd=NH.BF16, s=None, h=P5, dout=P4, dd=NH.BF16, m=m, n=n, k=k, rank=rank,
             adapters=adapters, dx_base=None, dx=OUT, da=P2, db=P3, accumulate=0, ws=WS, wsb=need, stream=None)
    a.update(over)
    return list(a.values())


def test_lora_refusals(rec):
    size = (100, 64, 48, 8, 3)
    for name, make in (("nh_linear_lora", lora_args), ("nh_linear_lora_backward", back_args)):
        def status(*s, **over):
            return NH.call_status(name, rec.ctx, *make(*(s or size), **over))[0]
        assert status() == NH.OK
        for at in range(1, 5):
            assert status(*[0 if i == at else v for i, v in enumerate(size)]) == NH.INVALID_SHAPE
        assert status(0, *size[1:]) == NH.INVALID_ROW_COUNT
        for bad in ((1 << 24, 8, 8, 4, 1), (8, (1 << 20) + 1, 8, 4, 1), (8, 8, (1 << 20) + 1, 4, 1), (8, 8, 8, 129, 1),
                    (8, 8, 8, 4, 1025), ((1 << 24) - 1, 1 << 20, 8, 4, 1), ((1 << 24) - 1, 8, 1 << 20, 4, 1), (1 << 62, 4, 4, 4, 4)):
            assert status(*bad) == NH.UNSUPPORTED and NH.lib().nh_supports_linear_lora(*bad) == 0
        assert NH.call_status(name, None, *make(*size))[0] == NH.INVALID_PARAMS
        for d in ("xd", "wd", "od" if make is lora_args else "dd"):
            assert status(**{d: 7}) == NH.INVALID_PARAMS
    f = lambda **o: NH.call_status("nh_linear_lora", rec.ctx, *lora_args(*size, **o))[0]  # noqa: E731
    for operand in ("x", "ids", "a", "b", "out"):
        assert f(**{operand: None}) == NH.INVALID_PARAMS
    assert f(base=None) == f(base=OUT) == f(s=P2) == f(h=P2) == NH.OK
    for operand in (X, S, W, W2, P4, OUT):
        assert f(h=operand) == f(h=operand + 4) == NH.INVALID_PARAMS
    assert f(s=P2, h=P2) == f(out=S) == f(out=W) == f(out=W2 + 16) == NH.INVALID_PARAMS
    assert f(base=OUT + 2) == f(out=X) == f(out=X + 4800) == NH.INVALID_PARAMS
    g = lambda **o: NH.call_status("nh_linear_lora_backward", rec.ctx, *back_args(*size, **o))[0]  # noqa: E731
    for operand in ("x", "ids", "a", "b", "dout"):
        assert g(**{operand: None}) == NH.INVALID_PARAMS
    assert g(dx=None, da=None, db=None) == NH.INVALID_PARAMS
    # what nothing asks for
    assert g(da=None, db=None, x=None, h=None) == g(dx=None, db=None, a=None, h=None) == NH.OK
    assert g(dx=None, da=None, a=None, b=None, x=P1) == g(dx=None, da=None, db=P3, b=None, h=None) == NH.OK
    assert g(dx=None, da=None, h=None, x=None) == g(dx=None, da=None, h=None, a=None) == NH.INVALID_PARAMS
    for operand in (X, S, W, W2, P4, P5, OUT):
        assert g(da=operand) == g(db=operand) == NH.INVALID_PARAMS and (operand == OUT or g(dx=operand) == NH.INVALID_PARAMS)
    assert g(da=P3) == g(dx=P2) == NH.INVALID_PARAMS
    assert g(dx=X) == g(dx=P4) == g(dx_base=OUT + 2) == NH.INVALID_PARAMS and g(dx_base=OUT) == NH.OK


def test_lora_workspace_is_checked(rec):
    size = (100, 64, 48, 8, 3)
    for name, make, at in (("nh_linear_lora", lora_args, -3), ("nh_linear_lora_backward", back_args, -3)):
        a = make(*size)
        for p, n, want in ((None, a[-2], NH.LENGTH_MISMATCH), (WS + 8, a[-2], NH.UNSUPPORTED), (WS, a[-2] - 1, NH.LENGTH_MISMATCH),
                           (WS, a[-2], NH.OK)):
            b = list(a)
            b[at], b[-2] = p, n
            assert NH.call_status(name, rec.ctx, *b)[0] == want


def test_lora_host_refusals():
    keep = [np.zeros(4096, np.float32) for _ in range(9)]
    p = [v.ctypes.data for v in keep]
    ok = [p[0], NH.F32, p[1], p[2], p[3], NH.F32, None, 4, 6, 5, 2, 2, None, p[4], NH.F32, None]
    assert NH.call_status("nh_linear_lora_host", *ok)[0] == NH.OK
    for at in (0, 2, 3, 4, 13):
        assert NH.call_status("nh_linear_lora_host", *[None if i == at else v for i, v in enumerate(ok)])[0] == NH.INVALID_PARAMS
    for at, st in ((7, NH.INVALID_ROW_COUNT), (8, NH.INVALID_SHAPE), (9, NH.INVALID_SHAPE), (10, NH.INVALID_SHAPE), (11, NH.INVALID_SHAPE)):
        assert NH.call_status("nh_linear_lora_host", *[0 if i == at else v for i, v in enumerate(ok)])[0] == st
    back = [p[0], NH.F32, p[1], p[2], p[3], NH.F32, None, None, p[4], NH.F32, 4, 6, 5, 2, 2, None, p[5], p[6], p[7], 0]
    assert NH.call_status("nh_linear_lora_backward_host", *back)[0] == NH.OK
    for at in (0, 2, 3, 4, 8):
        assert NH.call_status("nh_linear_lora_backward_host", *[None if i == at else v for i, v in enumerate(back)])[0] == NH.INVALID_PARAMS


# ---- envelopes ----------------------------------------------------------------------

def sizes(rng, top):
    v = 1 << rng.randrange(top + 1)
    return max(1, rng.choice([v, v - 1, v + 1, rng.randint(1, v)]))


def test_accepted_sizes_can_be_launched(rec):
    rng, lib, seen = random.Random(2), NH.lib(), set()
    far = 1 << 60
    for _ in range(6000):
        launches = []
        size = (sizes(rng, 24), sizes(rng, 20), sizes(rng, 20), sizes(rng, 7), sizes(rng, 10))
        yes = lib.nh_supports_linear_lora(*size)
        assert (lib.nh_linear_lora_workspace_size(*size) > 0) == (lib.nh_linear_lora_backward_workspace_size(*size) > 0) == bool(yes)
        if yes:
            launches += rec.launches("nh_linear_lora", *lora_args(*size, x=1 << 56, out=far, base=None))
            launches += rec.launches("nh_linear_lora_backward", *back_args(*size, x=1 << 56, dout=1 << 58, dx=far, h=None))
        t, k, h = sizes(rng, 31), sizes(rng, 6), sizes(rng, 31)
        if lib.nh_supports_moe_rows(t, k, h, t):
            launches += rec.launches("nh_moe_dispatch", 1 << 50, NH.BF16, S, None, t, k, h, t, far, NH.F32, None)
            launches += rec.launches("nh_moe_combine_rows", far, NH.F32, S, None, None, t, k, h, t, 1 << 50, NH.BF16, None)
        for kernel, gx, gy in launches:
            threads = 1024 if kernel == "lora_plan" else 512 if "rows" in kernel or "shrink" in kernel else 256
            assert gx >= 1 and gx * (threads if "rows" not in kernel else 64) < 1 << 32 and 1 <= gy <= 65535, (kernel, gx, gy)
            seen.add(kernel)
    assert len([k for k in seen if "lora_shrink" in k]) >= 4


@pytest.mark.parametrize("m,plan", [(1, False), (64, False), (65, True), (5000, True)])
def test_few_rows_need_no_plan(rec, m, plan):
    launches = rec.kernels("nh_linear_lora", *lora_args(m, 512, 512, 16, 4))
    assert launches == (["lora_plan"] if plan else []) + [f"lora_{f}_bf16_{'tiles' if plan else 'few'}_1" for f in ("shrink", "expand")]


@pytest.mark.parametrize("rank,form", [(1, 1), (16, 1), (17, 2), (32, 2), (33, 4), (64, 4), (65, 8), (128, 8)])
@pytest.mark.parametrize("xd,wd,kinds", [(NH.BF16, NH.BF16, ("bf16", "bf16", "bf16")), (NH.F32, NH.BF16, ("f32", "bf16", "f32")),
                                         (NH.BF16, NH.F32, ("f32", "f32", "bf16")), (NH.F32, NH.F32, ("f32", "f32", "f32"))])
def test_forms_by_rank_and_type(rec, rank, form, xd, wd, kinds):
    launches = rec.kernels("nh_linear_lora", *lora_args(200, 512, 512, rank, 4, xd=xd, wd=wd))
    assert launches[1:] == [f"lora_shrink_{kinds[0]}_tiles_{form}", f"lora_expand_{kinds[1]}_tiles_{form}"]
    launches = rec.kernels("nh_linear_lora_backward", *back_args(200, 512, 512, rank, 4, xd=xd, wd=wd, dd=xd))
    assert {f"lora_shrink_{kinds[0]}_back_{form}", f"lora_expand_{kinds[1]}_back_{form}", f"lora_outer_{kinds[2]}_{form}"} <= set(launches)


# ---- the surface ----------------------------------------------------------------------

NAMES = r"nh_(?:moe_dispatch|moe_combine_rows|linear_lora)\w*"


def test_registry_lists_every_entry_point():
    lib, names = NH.lib(), {}
    for i in range(lib.nh_kernel_count()):
        backend = C.c_int(-1)
        name = lib.nh_kernel_name(i, C.byref(backend)).decode()
        names[name] = backend.value
    entries = re.findall(rf"^nh_status ({NAMES})\(", open(HEADER).read(), re.M)
    assert len(entries) == 12
    for e in entries:
        assert names.get(e[3:]) == (0 if e.endswith("_host") else 1), e


def test_rust_comments_are_the_headers():
    words = lambda t: re.findall(r"\w+", t)  # noqa: E731
    header = open(HEADER).read()
    crate = open(os.path.join(os.path.dirname(HEADER), "..", "rust", "nemotron-hip-sys", "src", "lib.rs")).read()
    names = rf"(?:nh_supports_moe_rows|nh_supports_linear_lora|{NAMES})"
    comments = re.findall(r"/\*((?:[^*]|\*(?!/))*)\*/\n[^;{}/]*?\b(" + names + r")\s*\(", header)
    assert len(comments) >= 8
    for text, name in comments:
        rust = re.search(r"((?:    ///[^\n]*\n)+)    pub fn " + name + r"\b", crate)
        assert rust, name
        assert words(rust.group(1)) == words(re.sub(r"\n \*", "\n", text)), name
