"""Rows by expert and low-rank adapters in 64 bits, from their definitions (numpy), and how far a kernel may be off.

u = 2^-24 (f32).  A sum of n terms in f32, in any order, is off by at most n u of the terms' absolute sum (first order;
the factors below leave room for the second).  A value rounded to bf16 is off by 2^-8 of it, to f32 by 2^-24."""
import numpy as np

from mx_reference import from_bf16_bits, to_bf16_bits

U = 2.0 ** -24
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}


def held(x, dtype):
    """f32 values -> (as stored, as the f64 values that they stand for)."""
    x = np.asarray(x, np.float32)
    if dtype == "bf16":
        b = to_bf16_bits(x)
        return b, from_bf16_bits(b).astype(np.float64)
    return x, x.astype(np.float64)


def values(stored):
    return (from_bf16_bits(stored) if stored.dtype == np.uint16 else stored).astype(np.float64)


def empty(shape, dtype):
    return np.zeros(shape, np.uint16 if dtype == "bf16" else np.float32)


# ---- rows by expert -----------------------------------------------------------

def placed(pos, slots):
    return (pos >= 0) & (pos < slots)


def scatter(v, pos, w, slots, rows=None):
    """(rows [slots][H] and which of them are written, their tolerance for an output type's half step, dweights and its)."""
    t, k = pos.shape
    out, touched = np.zeros((slots, v.shape[1])), np.zeros(slots, bool)
    dw, dw_abs = np.zeros((t, k)), np.zeros((t, k))
    for i in range(t):
        for j in range(k):
            if placed(pos[i, j], slots):
                s = pos[i, j]
                out[s] = v[i] * (1.0 if w is None else w[i, j])
                touched[s] = True
                if rows is not None:
                    dw[i, j], dw_abs[i, j] = rows[s] @ v[i], np.abs(rows[s]) @ np.abs(v[i])
    return out, touched, dw, dw_abs


def gather(rows, pos, w, shared=None, dot=None):
    """(out, the absolute sum of its terms, dweights, the absolute sum of its)."""
    t, k = pos.shape
    out = np.zeros((t, rows.shape[1])) if shared is None else shared.copy()
    size, dw, dw_abs = np.abs(out), np.zeros((t, k)), np.zeros((t, k))
    for i in range(t):
        for j in range(k):
            if placed(pos[i, j], len(rows)):
                y = rows[pos[i, j]] * (1.0 if w is None else w[i, j])
                out[i] += y
                size[i] += np.abs(y)
                if dot is not None:
                    dw[i, j] = rows[pos[i, j]] @ dot[i]
                    dw_abs[i, j] = np.abs(rows[pos[i, j]]) @ np.abs(dot[i])
    return out, size, dw, dw_abs


# ---- low-rank adapters ----------------------------------------------------------

def _rows(ids, adapters):
    """An adapter's rows; one without takes no part, whatever its scale."""
    return [(n, np.flatnonzero(ids == n)) for n in range(adapters) if (ids == n).any()]


def forward(x, ids, a, b, s, base):
    """out, h, and what their tolerances are made of: sums of absolute terms."""
    adapters, rank, k = a.shape
    n = b.shape[1]
    out = np.zeros((len(x), n)) if base is None else base.copy()
    h, h_abs = np.zeros((len(x), rank)), np.zeros((len(x), rank))
    low, far = np.zeros_like(out), np.zeros_like(out)
    for l, i in _rows(ids, adapters):
        scale = 1.0 if s is None else float(s[l])
        h[i], h_abs[i] = x[i] @ a[l].T, np.abs(x[i]) @ np.abs(a[l]).T
        out[i] += scale * (h[i] @ b[l].T)
        low[i] = abs(scale) * (np.abs(h[i]) @ np.abs(b[l]).T)   # the terms of the second product
        far[i] = abs(scale) * (h_abs[i] @ np.abs(b[l]).T)       # what the first one's errors reach
    return out, h, {"h": h_abs, "low": low, "far": far}


# Where matrices and result are bf16, the bf16 matrix cores see a low-rank value as two parts of eight bits (what the
# first leaves over starts no higher than its ninth bit), so what is lost stays under 2^-15 of it; three parts are the
# value.
def forward_tolerance(out, parts, k, rank, w_dtype, out_dtype):
    cut = 2.0 ** -15 if w_dtype == out_dtype == "bf16" else 0.0
    low = (3 * rank + 8) * U + cut
    return 1.01 * (HALF[out_dtype] * (np.abs(out) + low * parts["low"]) + low * parts["low"]
                   + (k + 40) * U * parts["far"] + U * np.abs(out)) + 1e-40


def h_tolerance(parts, k):
    return 1.01 * (k + 40) * U * parts["h"] + 1e-40


def backward(x, ids, a, b, s, dout, dx_base):
    adapters, rank, k = a.shape
    dx = np.zeros_like(x) if dx_base is None else dx_base.copy()
    low, far = np.zeros_like(dx), np.zeros_like(dx)
    da, db = np.zeros(a.shape), np.zeros(b.shape)
    da_low, da_far, db_low, db_far = np.zeros(a.shape), np.zeros(a.shape), np.zeros(b.shape), np.zeros(b.shape)
    for l, i in _rows(ids, adapters):
        scale = 1.0 if s is None else float(s[l])
        h, h_abs = x[i] @ a[l].T, np.abs(x[i]) @ np.abs(a[l]).T
        dh, dh_abs = scale * (dout[i] @ b[l]), abs(scale) * (np.abs(dout[i]) @ np.abs(b[l]))
        dx[i] += dh @ a[l]
        low[i], far[i] = np.abs(dh) @ np.abs(a[l]), dh_abs @ np.abs(a[l])
        da[l], db[l] = dh.T @ x[i], scale * (dout[i].T @ h)
        da_low[l], da_far[l] = np.abs(dh).T @ np.abs(x[i]), dh_abs.T @ np.abs(x[i])
        db_low[l], db_far[l] = abs(scale) * (np.abs(dout[i]).T @ np.abs(h)), abs(scale) * (np.abs(dout[i]).T @ h_abs)
    parts = {"low": low, "far": far, "da_low": da_low, "da_far": da_far, "db_low": db_low, "db_far": db_far}
    return dx, da, db, parts


def gradient_tolerance(parts, which, length, m):
    """da (length n: dh's sums) or db (length k: h's sums), f32: three parts a term, sums over at most m rows."""
    return 1.01 * ((3 * m + 40) * U * parts[which + "_low"] + (length + 40) * U * parts[which + "_far"]) + 1e-40
