"""Plain 64-bit forms of the MXFP4 operators and of the router's balance loss, from their definitions (numpy)."""
import numpy as np

BLOCK = 32
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# between neighbours; a tie goes to the one of even mantissa: down at the even places, up at the odd ones
MIDDLE = (GRID[1:] + GRID[:-1]) / 2


def to_bf16_bits(x):
    """f32 -> bf16 bits, nearest even (finite values, infinities and NaNs)."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), ((u >> 16) | 0x40).astype(np.uint16), r)


def from_bf16_bits(b):
    return (np.ascontiguousarray(b).astype(np.uint32) << 16).view(np.float32)


def quantize(x):
    """[rows][cols] -> codes [rows][ceil(cols / 2)], scales [rows][ceil(cols / 32)], values (f64)."""
    x = np.asarray(x, dtype=np.float64)
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    b = np.zeros((rows, blocks * BLOCK))
    b[:, :cols] = x
    b = b.reshape(rows, blocks, BLOCK)
    bad = ~np.isfinite(b).all(axis=2)
    b = np.where(bad[:, :, None], 0.0, b)
    amax = np.abs(b).max(axis=2)
    exponent = np.frexp(amax)[1] - 1  # floor(log2), of a positive amax
    e = np.where(amax > 0, np.maximum(exponent - 2 + 127, 0), 0)
    scale = np.ldexp(1.0, e - 127)[:, :, None]
    a = np.abs(b) / scale
    index = np.zeros(b.shape, dtype=np.int64)
    for i, mid in enumerate(MIDDLE):
        index += (a >= mid) if i % 2 else (a > mid)
    code = (index | (np.signbit(b) * 8)).astype(np.uint8)
    code[bad] = 0
    value = GRID[index] * np.where(np.signbit(b), -1.0, 1.0) * scale
    value[bad] = np.nan
    e = np.where(bad, 255, e).astype(np.uint8)
    code = code.reshape(rows, -1)[:, :cols]
    if cols % 2:
        code = np.concatenate([code, np.zeros((rows, 1), np.uint8)], axis=1)
    return (code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8), e, value.reshape(rows, -1)[:, :cols]


def decode(codes, scales, cols):
    c = np.stack([codes & 15, codes >> 4], axis=2).reshape(codes.shape[0], -1)[:, :cols]
    e = np.repeat(scales.astype(np.int64), BLOCK, axis=1)[:, :cols]
    v = GRID[c & 7] * np.where(c & 8, -1.0, 1.0) * np.ldexp(1.0, e - 127)
    return np.where(e == 255, np.nan, v)


def tile(codes, scales, n, k):
    """The documented tiled form, byte by byte."""
    kt, nt = -(-k // 128), -(-n // 16)
    kq = -(-kt // 4)
    out = np.zeros((nt, kt * 1024 + kq * 256), np.uint8)
    for row in range(n):
        region, r = out[row // 16], row % 16
        for b in range(-(-k // BLOCK)):
            t, g = divmod(b, 4)
            piece = codes[row, 16 * b:16 * b + 16]
            at = t * 1024 + 16 * (16 * g + r)
            region[at:at + piece.size] = piece
            q, j = divmod(t, 4)
            region[kt * 1024 + q * 256 + 4 * (16 * g + r) + j] = scales[row, b]
    return out.reshape(-1)


def grid_matrix(rng, rows, cols, spread):
    """Values that MXFP4 holds exactly: grid elements times 2^-spread .. 2^spread, one power per block."""
    s = np.repeat(rng.integers(-spread, spread + 1, (rows, -(-cols // BLOCK))), BLOCK, axis=1)[:, :cols]
    return np.ldexp(GRID[rng.integers(0, 8, (rows, cols))] * rng.choice([-1.0, 1.0], (rows, cols)), s).astype(np.float32)


def offsets_of(seq, tokens):
    return [(0, tokens)] if seq is None else list(zip(seq[:-1], seq[1:]))


def balance(z, idx, seq, softmax, coefficient, dloss=1.0):
    """(counts, loss, dlogits) in 64 bits."""
    z = np.asarray(z, dtype=np.float64)
    t, e = z.shape
    k = idx.shape[1]
    spans = offsets_of(seq, t)
    counts, loss, grad = np.zeros((len(spans), e), np.int32), 0.0, np.zeros((t, e))
    for s, (lo, hi) in enumerate(spans):
        if hi <= lo:
            continue
        ids = idx[lo:hi].reshape(-1)
        ids = ids[(ids >= 0) & (ids < e)]
        counts[s] = np.bincount(ids, minlength=e)
        f = counts[s] * e / (k * (hi - lo))
        part = coefficient / (len(spans) * (hi - lo))
        for row in range(lo, hi):
            p, slope = probabilities(z[row], softmax)
            loss += part * float(f @ p)
            grad[row] = part * dloss * p * (f - f @ p) * slope
    return counts, loss, grad


def probabilities(z, softmax):
    """p and d of one row; a row of -inf alone has none."""
    m = np.max(z)
    if m == -np.inf:
        return np.zeros_like(z), np.ones_like(z)
    if softmax:
        w, slope = np.exp(z - m), np.ones_like(z)
    else:  # log sigmoid, so that no row underflows
        with np.errstate(over="ignore"):
            ls = np.minimum(z, 0) - np.log1p(np.exp(-np.abs(z)))
            slope = np.exp(np.minimum(-z, 0) - np.log1p(np.exp(-np.abs(z))))
        w = np.exp(ls - np.max(ls))
    return w / w.sum(), slope
