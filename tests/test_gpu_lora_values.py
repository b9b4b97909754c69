"""What the adapters' products make of their low-rank values: every bit of them, whatever the result's type, and
infinities as the formulas have them."""
import numpy as np
import pytest

import adapters_reference as A
import nemotron_hip as NH
from test_gpu_lora import DT, NP, TYPES, Case
from test_gpu_mxfp4 import Guarded, note

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = NH.Context(0)
    yield c
    c.close()


def cancelling(ctx, base, product, dtype):
    """A base that leaves of base + product what rounding the product to `dtype` leaves over, at the address of `base`."""
    stored, v = A.held(-product, dtype)
    buf, at = base
    raw = buf.numpy()
    raw[at - buf.ptr:][:stored.nbytes] = stored.view(np.uint8).reshape(-1)
    buf.copy_from(raw)
    return v


@pytest.mark.parametrize("m,n,k,rank,adapters,kind", [
    (1, 300, 8, 1, 1, "one"), (40, 200, 16, 8, 3, "each"), (64, 130, 8, 24, 2, "runs"), (33, 90, 8, 64, 2, "each"),
    (20, 96, 8, 100, 1, "one"), (100, 130, 16, 8, 3, "runs"), (200, 200, 8, 20, 3, "each"), (130, 129, 16, 33, 2, "runs"),
    (70, 192, 8, 100, 1, "one"), (90, 128, 8, 128, 2, "each")])
@pytest.mark.parametrize("x,out", [("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32")])
def test_a_product_that_its_base_cancels(ctx, m, n, k, rank, adapters, kind, x, out):
    """What is left of base + product is some 2^-9 of the product, so its own rounding to bf16 leaves nothing of the
    terms' errors out: they are f32's alone (3 rank products' sums and the first product's), no 2^-15 of a low-rank
    value."""
    note(f"lora cancelled m={m} n={n} k={k} rank={rank} adapters={adapters} {kind} {x} {out}")
    c = Case(ctx, m, n, k, rank, adapters, x, "bf16", out, kind)
    wide = np.random.default_rng(m).standard_normal((m, n))  # dout, of few columns that count: dh's sum is short
    wide[:, 8:] = 0
    stored, c.dout = A.held(wide, out)
    buf, at = c.keep["dout"]
    raw = buf.numpy()
    raw[at - buf.ptr:][:stored.nbytes] = stored.view(np.uint8).reshape(-1)
    buf.copy_from(raw)
    with np.errstate(invalid="ignore"):
        c.base = cancelling(ctx, c.keep["base"], A.forward(c.x, c.ids, c.a, c.b, c.s, None)[0], out)
        want, _, parts = A.forward(c.x, c.ids, c.a, c.b, c.s, c.base)
        c.dx_base = cancelling(ctx, c.keep["dx_base"], A.backward(c.x, c.ids, c.a, c.b, c.s, c.dout, None)[0], x)
        wdx, _, _, dparts = A.backward(c.x, c.ids, c.a, c.b, c.s, c.dout, c.dx_base)
    y, dx = Guarded(ctx, (m, n), NP[out]), Guarded(ctx, (m, k), NP[x])
    c.forward(y.ptr)
    c.backward(None, dx.ptr, None, None)
    # f32 matrices' tolerance: no part of a value cut away; of dout's sums eight terms are not zero
    assert (np.abs(A.values(y.numpy()) - want) <= A.forward_tolerance(want, parts, k, rank, "f32", out)).all()
    assert (np.abs(A.values(dx.numpy()) - wdx) <= A.forward_tolerance(wdx, dparts, 8, rank, "f32", x)).all()


def put(keep, stored):
    buf, at = keep
    raw = buf.numpy()
    raw[at - buf.ptr:][:stored.nbytes] = stored.view(np.uint8).reshape(-1)
    buf.copy_from(raw)


def same(got, want, half):
    """Finite values as near as their type allows, infinities of the same sign, NaN where the formula gives it."""
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    assert (np.abs(got[fine] - want[fine]) <= half * np.abs(want[fine])).all()


@pytest.mark.parametrize("m,n,k,rank,adapters", [(1, 70, 9, 1, 1), (30, 100, 70, 8, 2), (64, 130, 40, 40, 3), (20, 64, 64, 100, 1),
                                                 (90, 70, 66, 8, 2), (150, 130, 130, 20, 3), (200, 96, 96, 64, 2), (80, 90, 70, 100, 1),
                                                 (2500, 64, 66, 16, 1)])
@pytest.mark.parametrize("x,w,out", TYPES)
@pytest.mark.parametrize("where", ["a", "b", "x", "dout"])
def test_infinities_are_those_of_the_formulas(ctx, m, n, k, rank, adapters, x, w, out, where):
    """Whole numbers whose sums f32 holds, most low-rank values of few bits, with infinities of both signs in one
    operand: what stands beside a zero is NaN, what stands beside anything else infinite."""
    note(f"lora infinities m={m} n={n} k={k} rank={rank} adapters={adapters} {x} {w} {out} in {where}")
    rng = np.random.default_rng(m + n + k + rank)
    c = Case(ctx, m, n, k, rank, adapters, x, w, out, "one" if adapters == 1 else "each", scales=False)
    c.ids = np.where(c.ids >= adapters, -1, c.ids)
    shapes = {"a": ((adapters, rank, k), w), "b": ((adapters, n, rank), w), "x": ((m, k), x), "dout": ((m, n), out),
              "base": ((m, n), out), "dx_base": ((m, k), x)}
    v = {}
    for name, (shape, dtype) in shapes.items():
        value = rng.integers(-2, 3, shape).astype(np.float32)
        if name == where:
            for sign in (1, -1):
                value[tuple(rng.integers(0, s, 2) for s in shape)] = sign * np.inf
        stored, v[name] = A.held(value, dtype)
        put(c.keep[name], stored)
    with np.errstate(invalid="ignore"):
        y, dx = v["base"].copy(), v["dx_base"].copy()
        da, db = np.zeros_like(v["a"]), np.zeros_like(v["b"])
        for l in range(adapters):
            i = np.flatnonzero(c.ids == l)
            if i.size == 0:
                continue
            h, dh = v["x"][i] @ v["a"][l].T, v["dout"][i] @ v["b"][l]
            y[i] += h @ v["b"][l].T
            dx[i] += dh @ v["a"][l]
            da[l], db[l] = dh.T @ v["x"][i], v["dout"][i].T @ h
    for value in (y, dx, da, db):  # f32 holds every sum on the way
        assert np.abs(value[np.isfinite(value)]).max(initial=0) < 2 ** 24
    outs = [Guarded(ctx, shape, NP[d]) for shape, d in (((m, n), out), ((m, k), x), (da.shape, "f32"), (db.shape, "f32"))]
    c.forward(outs[0].ptr)
    c.backward(None, *[o.ptr for o in outs[1:]])
    for got, want, dtype in zip(outs, (y, dx, da, db), (out, x, "f32", "f32")):
        same(A.values(got.numpy()), want, A.HALF["bf16"] if dtype == "bf16" else 0.0)
