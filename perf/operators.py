"""The MXFP4 operators and the router's balance loss as measurable passes, with their plain forms.

MXFP4 (OCP microscaling): 4-bit e2m1 elements in blocks of 32 along a row, each block with one power-of-two scale
byte (e8m0).  The scale is 2^(floor(log2(largest |x| of the block)) - 2); elements are rounded to nearest even on
the grid 0, 0.5, 1, 1.5, 2, 3, 4, 6 and saturate at 6.

Sizes are those of the repository's own workloads (bench.py: the 4096-wide hybrid stack, the 2688-wide MoE layer
with 128 experts of 1856, top-6) and generic ragged ones.  A serving program keeps, per layer, its tiled weights,
workspace and output buffers, and calls the C ABI on them.
"""
import ctypes
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
BLOCK = 32          # values that share a scale
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one decode token's activations, quantized and read back: the smallest call, latency bound
        {"name": "quant_1row", "op": "quant", "rows": 1, "cols": 4096, "x": "bf16"},
        # a prompt's activations of odd width: rows of any alignment, a last block of part of a scale
        {"name": "quant_ragged", "op": "quant", "rows": 613, "cols": 2701, "x": "bf16"},
        # a projection's f32 weights, as a checkpoint is converted
        {"name": "quant_weights", "op": "quant", "rows": 16384, "cols": 4096, "x": "f32"},
        # single-stream decode: the SSM in_proj
        {"name": "linear_m1", "op": "linear", "m": 1, "k": 4096, "n": 16384, "x": "bf16", "out": "bf16",
         "bias": False},
        # batch-8 decode: logits over a large vocabulary, weights larger than any cache
        {"name": "linear_m8_head", "op": "linear", "m": 8, "k": 4096, "n": 131072, "x": "bf16", "out": "f32",
         "bias": False},
        # a ragged f32 prompt through a layer of odd width and depth, with a bias
        {"name": "linear_m300_ragged", "op": "linear", "m": 300, "k": 2701, "n": 4099, "x": "f32", "out": "f32",
         "bias": True},
        # prefill of 2048 tokens: the widest projection
        {"name": "linear_m2048_up", "op": "linear", "m": 2048, "k": 4096, "n": 21504, "x": "bf16", "out": "bf16",
         "bias": False},
        # batch-8 decode through the experts: about 40 of 128 are reached
        {"name": "moe_t8", "op": "moe", "tokens": 8, "hidden": 2688, "inter": 1856, "experts": 128, "top_k": 6,
         "x": "bf16"},
        # a 500-token prompt through the same experts
        {"name": "moe_t500", "op": "moe", "tokens": 500, "hidden": 2688, "inter": 1856, "experts": 128, "top_k": 6,
         "x": "bf16"},
        # a small batch's load balance: launches are what it costs
        {"name": "balance_t64", "op": "balance", "tokens": 64, "experts": 128, "top_k": 6, "sequences": 1, "pad": 0,
         "softmax": False},
        # a fine-tuning micro-batch of packed sequences, each balanced by itself, with padding behind the last
        {"name": "balance_packed", "op": "balance", "tokens": 8191, "experts": 128, "top_k": 6, "sequences": 13,
         "pad": 311, "softmax": False},
        # a large batch through a softmax router
        {"name": "balance_t131072", "op": "balance", "tokens": 131072, "experts": 128, "top_k": 8, "sequences": 1,
         "pad": 0, "softmax": True},
    ]


MAX_FLOPS = 3.6e11                    # the listed prefill's
MAX_HEAD = 4096 * 131072              # the listed vocabulary's weights
MAX_EXPERT_WEIGHTS = 128 * 2688 * 1856


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A row length: whole 128s, whole 32s or any."""
    v = _log(rng, lo, hi)
    unit = rng.choice([128, 32, 1])
    return max(unit, v // unit * unit)


def draw(rng):
    while True:
        op = rng.choices(["quant", "linear", "moe", "balance"], [20, 40, 20, 20])[0]
        x = rng.choice(["bf16", "bf16", "bf16", "f32"])
        if op == "quant":
            case = {"op": op, "rows": _log(rng, 1, 16384), "cols": _width(rng, 32, 21504), "x": x}
            if case["rows"] * case["cols"] > 16384 * 4096:
                continue
        elif op == "linear":
            case = {"op": op, "m": _log(rng, 1, 2048), "k": _width(rng, 128, 21504), "n": _log(rng, 64, 32768), "x": x,
                    "out": rng.choice(["bf16", "bf16", "f32"]), "bias": rng.random() < 0.4}
            if rng.random() < 0.5:
                case["n"] = max(64, case["n"] // 64 * 64)
            if case["n"] * case["k"] > MAX_HEAD or work(case)["flops"] > MAX_FLOPS:
                continue
        elif op == "moe":
            experts = rng.choice([8, 16, 60, 64, 128])
            case = {"op": op, "tokens": _log(rng, 1, 768), "hidden": _width(rng, 256, 4096),
                    "inter": _width(rng, 256, 1856), "experts": experts, "top_k": rng.randint(1, 8), "x": x}
            if experts * case["hidden"] * case["inter"] > MAX_EXPERT_WEIGHTS or work(case)["flops"] > MAX_FLOPS:
                continue
        else:
            experts = rng.choice([8, 16, 60, 64, 128, 256, 512])
            tokens = _log(rng, 1, 131072)
            if tokens * experts > 131072 * 128:
                continue
            sequences = 1 if rng.random() < 0.5 else _log(rng, 1, 64)
            case = {"op": op, "tokens": tokens, "experts": experts, "top_k": rng.randint(1, 8), "sequences": sequences,
                    "pad": 0 if rng.random() < 0.7 else tokens // 10, "softmax": rng.random() < 0.4}
        return case


# ---- inputs -----------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, shape, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(dtype)


def _activations(gen, rows, cols, dtype):
    """Normal rows with a few channels twenty times as large, as activations have them."""
    wide = torch.rand(cols, generator=gen, device="cuda") < 1 / 256
    return (_normal(gen, (rows, cols)) * torch.where(wide, 20.0, 1.0)).to(dtype)


def _encode(values, scales):
    """Values on the MXFP4 grid and their scale bytes -> packed codes, low nibble first."""
    rows, cols = values.shape
    q = (values * _power(127 - scales.int()).repeat_interleave(BLOCK, 1)[:, :cols]).abs()
    c = torch.where(q < 2, 2 * q, torch.where(q < 4, q + 2, q / 2 + 4)).to(torch.uint8)
    c = c | (torch.signbit(values).to(torch.uint8) << 3)
    c = torch.nn.functional.pad(c, (0, cols % 2))
    return c[:, 0::2] | (c[:, 1::2] << 4)


def _weights(gen, n, k):
    """A trained matrix in MXFP4: packed codes [n][ceil(k / 2)] and scale bytes [n][ceil(k / 32)]."""
    values, scales = _mx(_normal(gen, (n, k), 0.02))
    return _encode(values, scales), scales


def _tile(codes, scales, n, k):
    """The library's tiled form of MXFP4 weights (nh_tile_weights_mxfp4): per 16 rows, KT = ceil(k / 128) tiles of
    1 KiB of codes (byte 16 (16 g + r) + b of a tile: row r, values 32 g + 2 b and 2 b + 1 of its 128), then
    ceil(KT / 4) pieces of 256 scale bytes (byte 4 (16 g + r) + j: row r, block 4 (4 q + j) + g)."""
    nt, kt = -(-n // 16), -(-k // 128)
    kq = -(-kt // 4)
    c = torch.nn.functional.pad(codes, (0, kt * 64 - codes.shape[1], 0, nt * 16 - n))
    c = c.reshape(nt, 16, kt, 4, 16).permute(0, 2, 3, 1, 4).reshape(nt, kt * 1024)
    s = torch.nn.functional.pad(scales, (0, kq * 16 - scales.shape[1], 0, nt * 16 - n))
    s = s.reshape(nt, 16, kq, 4, 4).permute(0, 2, 4, 1, 3).reshape(nt, kq * 256)
    return torch.cat([c, s], 1).reshape(-1)


def _linear_inputs(case, seed):
    gen = _generator(seed)
    m, n, k = case["m"], case["n"], case["k"]
    x = _activations(gen, m, k, DT[case["x"]])
    bias = _normal(gen, (n,), 0.1) if case["bias"] else None
    return x, _weights(gen, n, k), bias


class _MoeInputs:
    def __init__(self, case, seed):
        self.case, self.gen = case, _generator(seed)
        self.x = _activations(self.gen, case["tokens"], case["hidden"], DT[case["x"]])
        self.logits = _normal(self.gen, (case["tokens"], case["experts"]))

    def experts(self):
        h, i = self.case["hidden"], self.case["inter"]
        for _ in range(self.case["experts"]):
            yield _weights(self.gen, i, h), _weights(self.gen, h, i)


def _balance_inputs(case, seed):
    gen = _generator(seed)
    t, e, k, s = (case[v] for v in ("tokens", "experts", "top_k", "sequences"))
    logits = _normal(gen, (t, e)) + _normal(gen, (e,), 0.5)  # some experts are liked more
    indices = logits.topk(min(k, e), dim=1).indices.to(torch.int32).contiguous()
    live = t - case["pad"]
    cuts = torch.randint(0, live + 1, (s - 1,), generator=gen, device="cuda").sort().values
    ends = torch.tensor([0, live], device="cuda")
    offsets = torch.cat([ends[:1], cuts, ends[1:]]).to(torch.int32)
    dloss = _normal(gen, (1,)).abs() + 0.5
    return logits, indices, offsets, dloss


BALANCE_COEFFICIENT = 0.01


def prepare(case, seed):
    if case["op"] == "quant":
        gen = _generator(seed)
        if case["x"] == "f32":
            x = _normal(gen, (case["rows"], case["cols"]), 0.02)
        else:
            x = _activations(gen, case["rows"], case["cols"], DT[case["x"]])
        return {"case": case, "x": x}
    if case["op"] == "linear":
        x, (codes, scales), bias = _linear_inputs(case, seed)
        return {"case": case, "x": x, "codes": codes, "scales": scales, "bias": bias,
                "tiled": _tile(codes, scales, case["n"], case["k"])}
    if case["op"] == "moe":
        inputs = _MoeInputs(case, seed)
        h, i = case["hidden"], case["inter"]
        up, down, tiled_up, tiled_down = [], [], [], []
        for u, d in inputs.experts():
            up.append(u)
            down.append(d)
            tiled_up.append(_tile(*u, i, h))
            tiled_down.append(_tile(*d, h, i))
        stack = lambda pairs: tuple(torch.stack(t) for t in zip(*pairs))  # noqa: E731
        return {"case": case, "x": inputs.x, "logits": inputs.logits, "up": stack(up), "down": stack(down),
                "tiled_up": torch.cat(tiled_up), "tiled_down": torch.cat(tiled_down)}
    logits, indices, offsets, dloss = _balance_inputs(case, seed)
    return {"case": case, "logits": logits, "indices": indices, "offsets": offsets, "dloss": dloss}


def run(state):
    if own:
        return _run_own(state)
    return {"quant": _plain_quant, "linear": _plain_linear, "moe": _plain_moe,
            "balance": _plain_balance}[state["case"]["op"]](state)


# ---- the plain forms: elementary operations in 32 bits ----------------------

def _power(e):
    """2^e as f32 from its bits, e an int32 tensor in [-127, 127]."""
    return torch.where(e > -127, (e + 127) << 23, 0x400000).view(torch.float32)


def _mx(x):
    """f32 [rows][cols] -> (its values on the MXFP4 grid in f32, scale bytes): every step is exact but the rounding."""
    rows, cols = x.shape
    b = torch.nn.functional.pad(x, (0, -cols % BLOCK)).reshape(rows, -1, BLOCK)
    bits = b.abs().amax(dim=2).view(torch.int32)
    byte = ((bits >> 23) - 2).clamp(min=0)
    y = b * _power(127 - byte).unsqueeze(2)
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = (torch.round(a / step) * step).clamp(max=6.0)
    v = torch.copysign(q, y) * _power(byte - 127).unsqueeze(2)
    return v.reshape(rows, -1)[:, :cols], byte.to(torch.uint8)


_pairs = None


def _decode(codes, scales, cols):
    """Packed codes [..., cols / 2] and scale bytes -> f32 [..., cols]."""
    global _pairs
    if _pairs is None:
        grid = torch.tensor(GRID + tuple(-v for v in GRID), device="cuda")
        byte = torch.arange(256, device="cuda")
        _pairs = torch.stack([grid[byte & 15], grid[byte >> 4]], 1)
    v = _pairs[codes.to(torch.int32)].flatten(-2)
    s = _power(scales.to(torch.int32) - 127)
    whole = v.shape[-1] // BLOCK * BLOCK
    if whole == v.shape[-1]:
        return (v.unflatten(-1, (-1, BLOCK)) * s.unsqueeze(-1)).flatten(-2)[..., :cols].contiguous()
    return (v * s.repeat_interleave(BLOCK, -1)[..., :v.shape[-1]])[..., :cols].contiguous()


def _plain_quant(state):
    x = state["x"]
    v, s = _mx(x.float())
    return {"values": v.to(x.dtype), "scales": s}


def _plain_linear(state):
    case = state["case"]
    x, _ = _mx(state["x"].float())
    y = x @ _decode(state["codes"], state["scales"], case["k"]).T
    if state["bias"] is not None:
        y = y + state["bias"]
    return y.to(DT[case["out"]])


def _route(logits, k):
    """Sigmoid top-k, ties to the lowest expert, weights renormalised."""
    w = torch.sigmoid(logits.double()).float()
    order = w.sort(dim=1, descending=True, stable=True)
    w = order.values[:, :k]
    return w / w.sum(dim=1, keepdim=True), order.indices[:, :k]


def _plain_moe(state):
    case = state["case"]
    t, h, i, e, k = (case[v] for v in ("tokens", "hidden", "inter", "experts", "top_k"))
    w, idx = _route(state["logits"], k)
    x, _ = _mx(state["x"].float())
    flat = idx.reshape(-1)
    routes = flat.numel()
    if routes <= e:  # each route against its own expert's weights
        groups, rows = routes, 1
        up, down = (tuple(p[flat] for p in state[v]) for v in ("up", "down"))
        slot = torch.arange(routes, device="cuda")
    else:  # the routes by expert, each expert's padded to the fullest one's
        count = torch.bincount(flat, minlength=e)
        groups, rows = e, int(count.max())
        up, down = state["up"], state["down"]
        order = flat.sort(stable=True)
        rank = torch.arange(routes, device="cuda") - (count.cumsum(0) - count)[order.values]
        slot = torch.empty_like(flat)
        slot[order.indices] = order.values * rows + rank
    a = torch.zeros((groups * rows, h), device="cuda")
    a[slot] = x.repeat_interleave(k, 0)
    y = torch.bmm(_decode(*up, h), a.view(groups, rows, h).transpose(1, 2).contiguous())
    y = torch.relu(y).square().transpose(1, 2).reshape(groups * rows, i)
    y, _ = _mx(y)
    y = torch.bmm(_decode(*down, i), y.view(groups, rows, i).transpose(1, 2).contiguous())
    y = y.transpose(1, 2).reshape(groups * rows, h)[slot].view(t, k, h)
    return (y * w.unsqueeze(2)).sum(dim=1).to(torch.bfloat16)


def _plain_balance(state):
    case = state["case"]
    z, idx, offsets = state["logits"], state["indices"], state["offsets"]
    t, e, s = case["tokens"], case["experts"], case["sequences"]
    k = idx.shape[1]
    seq = torch.searchsorted(offsets[1:], torch.arange(t, device="cuda", dtype=torch.int32), right=True)  # s: padding
    length = (offsets[1:] - offsets[:-1]).clamp(min=1).float()
    at = (seq.unsqueeze(1) * e + idx).reshape(-1)
    counts = torch.zeros((s + 1) * e, dtype=torch.int32, device="cuda")
    counts.scatter_add_(0, at, torch.ones_like(at, dtype=torch.int32))
    counts = counts.view(s + 1, e)[:s]
    f = counts.float() * (e / (k * length)).unsqueeze(1)          # [s][e]
    if case["softmax"]:
        u = torch.exp(z - z.amax(dim=1, keepdim=True))
    else:  # sigmoid, in a form that does not vanish for rows of large negative logits
        u = torch.exp(z.clamp(max=0) - z.amax(dim=1, keepdim=True).clamp(max=0)) / (1 + torch.exp(-z.abs()))
    p = u / u.sum(dim=1, keepdim=True)
    ft = torch.cat([f, torch.zeros_like(f[:1])])[seq]             # [t][e]
    fp = (ft * p).sum(dim=1)
    part = torch.cat([1 / length, torch.zeros(1, device="cuda")])[seq] * (BALANCE_COEFFICIENT / s)
    loss = (part * fp).double().sum().float().reshape(1)
    g = p * (ft - fp.unsqueeze(1))
    if not case["softmax"]:
        g = g * torch.exp(-torch.relu(z)) / (1 + torch.exp(-z.abs()))
    return {"counts": counts, "loss": loss, "dlogits": g * (part * state["dloss"]).unsqueeze(1)}


# ---- the library's calls ----------------------------------------------------

_library = None


def _nh():
    """The binding and the program's one library context."""
    global _library
    if _library is None:
        sys.path.insert(0, os.path.join(ROOT, "nemotron-cutile-rs_amd"))
        import nemotron_hip

        _library = (nemotron_hip, nemotron_hip.Context(0))
    return _library


class _Bound:
    """Entry points with their arguments bound to a layer's buffers, as a serving loop keeps them: all but the stream,
    which is the one that is current when a pass runs."""

    def __init__(self, state):
        NH, ctx = _nh()
        self.NH, self.ctx, self.err, self.calls, self.keep = NH, ctx.handle, NH.NhError(), [], []
        self.outs = getattr(self, "_" + state["case"]["op"])(state["case"], state)

    def add(self, name, *args):
        fn = getattr(self.NH.lib(), name)
        simple = (ctypes.c_size_t, ctypes.c_int, ctypes.c_float, ctypes.c_void_p)
        args = (self.ctx, *[a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args])
        conv = [t(a) if t in simple and not isinstance(a, t) else a for t, a in zip(fn.argtypes, args)]
        self.calls.append((fn, conv))

    def run(self):
        """One pass on the current stream.  Its outputs and its workspace are the state's: a state's passes run one
        after the other, and the next one overwrites what this one returns."""
        # the handle alone: the object of torch.cuda.current_stream() costs 3 us, which is a launch
        stream, err = ctypes.c_void_p(torch._C._cuda_getCurrentRawStream(0)), ctypes.byref(self.err)
        for fn, args in self.calls:
            status = fn(*args, stream, err)
            if status:
                self.NH.check(status, self.err)
        return self.outs

    def empty(self, shape, dtype):
        self.keep.append(torch.empty(shape, dtype=dtype, device="cuda"))
        return self.keep[-1]

    def dtype(self, name):
        return self.NH.BF16 if name == "bf16" else self.NH.F32

    def workspace(self, name, *sizes):
        t = self.empty(max(16, getattr(self.NH.lib(), name)(*sizes)), torch.uint8)
        return t, t.numel()

    def _quant(self, case, state):
        r, c, d = case["rows"], case["cols"], self.dtype(case["x"])
        codes, scales = self.empty((r, -(-c // 2)), torch.uint8), self.empty((r, -(-c // BLOCK)), torch.uint8)
        values = self.empty((r, c), DT[case["x"]])
        self.add("nh_quantize_rows_mxfp4", state["x"], d, r, c, codes, scales, None)
        self.add("nh_dequantize_mxfp4", codes, scales, r, c, values, d)
        return {"values": values, "scales": scales}

    def _linear(self, case, state):
        m, n, k = case["m"], case["n"], case["k"]
        out = self.empty((m, n), DT[case["out"]])
        ws = self.workspace("nh_linear_mxfp4_workspace_size", m, n, k)
        self.add("nh_linear_mxfp4", state["x"], self.dtype(case["x"]), state["tiled"], state["bias"], m, n, k, out,
                 self.dtype(case["out"]), *ws, None)
        return out

    def _moe(self, case, state):
        sizes = [case[v] for v in ("tokens", "hidden", "inter", "experts", "top_k")]
        out = self.empty((case["tokens"], case["hidden"]), torch.bfloat16)
        ws = self.workspace("nh_moe_forward_mxfp4_workspace_size", *sizes)
        self.add("nh_moe_forward_mxfp4", state["x"], self.dtype(case["x"]), state["logits"], *sizes, 1, 1.0,
                 state["tiled_up"], state["tiled_down"], None, None, out, self.NH.BF16, *ws, None)
        return out

    def _balance(self, case, state):
        t, e, s = case["tokens"], case["experts"], case["sequences"]
        k = state["indices"].shape[1]
        counts, loss = self.empty((s, e), torch.int32), self.empty((1,), torch.float32)
        dlogits = self.empty((t, e), torch.float32)
        ws = self.workspace("nh_moe_balance_loss_workspace_size", s, t, e)
        kind = (s, t, e, k, int(case["softmax"]), BALANCE_COEFFICIENT)
        self.add("nh_moe_balance_loss", state["logits"], state["indices"], state["offsets"], *kind, counts, loss, *ws)
        self.add("nh_moe_balance_loss_backward", state["logits"], counts, state["offsets"], *kind, state["dloss"],
                 dlogits)
        return {"counts": counts, "loss": loss, "dlogits": dlogits}


def _run_own(state):
    bound = state.get("bound")
    if bound is None:
        bound = state["bound"] = _Bound(state)
    return bound.run()


# ---- cost and expected values -----------------------------------------------

def _mx_bytes(rows, cols):
    return rows * (-(-cols // 2) + -(-cols // BLOCK))


def work(case):
    """Inputs, weights and outputs once each; the multiply-adds of the products."""
    size = {"f32": 4, "bf16": 2}
    if case["op"] == "quant":  # the rows in and out, the codes and scales out and in
        r, c = case["rows"], case["cols"]
        return {"bytes": 2.0 * (r * c * size[case["x"]] + _mx_bytes(r, c)), "flops": 4.0 * r * c}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": float(_mx_bytes(n, k) + 4 * n * case["bias"] + m * k * size[case["x"]]
                               + m * n * size[case["out"]]), "flops": 2.0 * m * n * k}
    if case["op"] == "moe":
        t, h, i, e, k = (case[v] for v in ("tokens", "hidden", "inter", "experts", "top_k"))
        touched = e * (1 - (1 - min(k, e) / e) ** t)  # experts that receive a route
        return {"bytes": touched * (_mx_bytes(i, h) + _mx_bytes(h, i)) + 4 * t * e + t * h * (size[case["x"]] + 2),
                "flops": 4.0 * t * k * h * i}
    t, e, k, s = (case[v] for v in ("tokens", "experts", "top_k", "sequences"))
    # forward and backward each read the logits; the counts are written and read
    return {"bytes": 4.0 * (3 * t * e + t * min(k, e) + 2 * s * e + s), "flops": 20.0 * t * e}


def _exact_mx(x):
    """Values on the MXFP4 grid in 64 bits, from the definition: blocks, a power of two, the nearest of eight."""
    rows, cols = x.shape
    pad = -cols % BLOCK
    b = torch.cat([x.double(), x.new_zeros((rows, pad), dtype=torch.float64)], 1).view(rows, -1, BLOCK)
    exponent = torch.frexp(b.abs().amax(dim=2, keepdim=True)).exponent - 1
    byte = torch.where(b.abs().amax(dim=2, keepdim=True) > 0, exponent - 2 + 127, 0).clamp(0, 254)
    scale = torch.exp2((byte - 127).double())
    a = b.abs() / scale
    index = torch.zeros_like(a, dtype=torch.int64)
    for n, (lo, hi) in enumerate(zip(GRID, GRID[1:])):  # a tie goes to the neighbour of even mantissa
        middle = (lo + hi) / 2
        index += (a >= middle) if n % 2 else (a > middle)
    v = torch.tensor(GRID, dtype=torch.float64, device=x.device)[index] * b.sign() * scale
    return v.view(rows, -1)[:, :cols], byte.squeeze(2).to(torch.uint8)


def _exact_weights(codes, scales, cols):
    c = torch.stack([codes & 15, codes >> 4], 2).reshape(codes.shape[0], -1)[:, :cols].long()
    e, m = (c >> 1) & 3, (c & 1).double()
    v = torch.where(e > 0, (1 + m / 2) * torch.exp2((e - 1).double()), m / 2) * (1 - 2 * (c >> 3)).double()
    block = torch.arange(cols, device=c.device) // BLOCK
    return v * torch.exp2(scales.double() - 127)[:, block]


def _exact_moe(case, seed):
    inputs = _MoeInputs(case, seed)
    k = case["top_k"]
    w, idx = torch.sigmoid(inputs.logits.double()).topk(k, dim=1)
    w = w / w.sum(dim=1, keepdim=True)
    x, _ = _exact_mx(inputs.x)
    out = torch.zeros_like(x)
    for n, (up, down) in enumerate(inputs.experts()):
        t, j = (idx == n).nonzero(as_tuple=True)
        if t.numel():
            y = (x[t] @ _exact_weights(*up, case["hidden"]).T).clamp(min=0).square()
            # the layer keeps y in 32 bits before it is quantized
            out[t] += w[t, j][:, None] * (_exact_mx(y.float())[0] @ _exact_weights(*down, case["inter"]).T)
    return out


def _exact_balance(case, seed):
    z, idx, offsets, dloss = _balance_inputs(case, seed)
    z, e, s = z.double(), case["experts"], case["sequences"]
    k, off = idx.shape[1], offsets.tolist()
    weight = z.softmax(dim=1) if case["softmax"] else z.sigmoid()
    p = weight / weight.sum(dim=1, keepdim=True)
    slope = p if case["softmax"] else p * (1 - weight)
    counts = torch.zeros((s, e), dtype=torch.int32, device=z.device)
    loss, grad = 0.0, torch.zeros_like(z)
    for n, (lo, hi) in enumerate(zip(off, off[1:])):
        if hi > lo:
            counts[n] = torch.bincount(idx[lo:hi].reshape(-1).long(), minlength=e).int()
            f = counts[n].double() * e / (k * (hi - lo))
            per_row = p[lo:hi] @ f
            part = BALANCE_COEFFICIENT / (s * (hi - lo))
            loss = loss + part * per_row.sum()
            grad[lo:hi] = slope[lo:hi] * (f - per_row[:, None]) * part * dloss.double()
    return {"counts": counts, "loss": torch.as_tensor(loss, device=z.device).double().reshape(1), "dlogits": grad}


def exact(case, seed):
    if case["op"] == "quant":
        v, s = _exact_mx(prepare(case, seed)["x"])
        return {"values": v, "scales": s}
    if case["op"] == "linear":
        x, (codes, scales), bias = _linear_inputs(case, seed)
        y = _exact_mx(x)[0] @ _exact_weights(codes, scales, case["k"]).T
        return y if bias is None else y + bias.double()
    return _exact_moe(case, seed) if case["op"] == "moe" else _exact_balance(case, seed)
