"""Rows of a mixture of experts sorted by expert and back, and low-rank adapters beside a linear layer, as measurable
passes with their plain forms.

Rows by expert: token t has top_k routes; route (t, j) goes to expert indices[t, j].  The routes are sorted by expert,
stable by route, into slots; rows[slot of (t, j)] = x[t] is what the experts read, and out[t] = sum_j w[t, j] *
y[slot of (t, j)] joins what they answer.  Backward: dy[slot] = w[t, j] dout[t], dw[t, j] = <y[slot], dout[t]>, and
dx[t] = sum_j drows[slot of (t, j)].

Low-rank adapters: row i belongs to adapter l = ids[i] (or to none): out_i = base_i + s_l B_l (A_l x_i), base being the
shared projection's output, A_l [rank][k], B_l [n][rank].  Backward, h_i = A_l x_i: dh_i = s_l B_l^T dout_i,
dx_i = dx_base_i + A_l^T dh_i, dA_l = sum_i dh_i x_i^T, dB_l = s_l sum_i dout_i h_i^T.

Sizes are those of the repository's own workloads (bench.py: the 4096-wide stack and its 16384- and 21504-wide
projections, the 2688-wide MoE layer with 128 experts, top-6) and generic ragged ones.  A program keeps its workspaces
and output buffers, and calls the C ABI on them.
"""
import ctypes
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}


def listed():
    return [
        # batch-8 decode through the experts: launches are what it costs
        {"name": "rows_t8", "op": "rows", "tokens": 8, "hidden": 2688, "experts": 128, "top_k": 6, "x": "bf16"},
        # a ragged f32 prompt of odd width, where rows start at any alignment
        {"name": "rows_ragged", "op": "rows", "tokens": 613, "hidden": 2701, "experts": 60, "top_k": 4, "x": "f32"},
        # a prompt batch of 8192 tokens: the sort of 49152 routes, and rows larger than any cache
        {"name": "rows_t8192", "op": "rows", "tokens": 8192, "hidden": 2688, "experts": 128, "top_k": 6, "x": "bf16"},
        # the gradients of a short fine-tuning sequence
        {"name": "rows_train_t64", "op": "rows_train", "tokens": 64, "hidden": 2688, "experts": 128, "top_k": 6,
         "x": "bf16"},
        # the gradients of a training micro-batch
        {"name": "rows_train_t8192", "op": "rows_train", "tokens": 8192, "hidden": 2688, "experts": 128, "top_k": 6,
         "x": "bf16"},
        # single-stream decode of one fine-tune
        {"name": "lora_m1", "op": "lora", "m": 1, "k": 4096, "n": 4096, "rank": 16, "adapters": 8, "x": "bf16",
         "w": "bf16", "spread": "rows"},
        # a decode batch whose requests each name their own fine-tune, at the widest input projection
        {"name": "lora_m48_each", "op": "lora", "m": 48, "k": 4096, "n": 16384, "rank": 16, "adapters": 64, "x": "bf16",
         "w": "bf16", "spread": "rows"},
        # a ragged f32 prompt batch of odd widths and a small rank
        {"name": "lora_ragged", "op": "lora", "m": 613, "k": 2701, "n": 4099, "rank": 8, "adapters": 5, "x": "f32",
         "w": "f32", "spread": "runs"},
        # prefill of several requests at the widest projection, a large rank
        {"name": "lora_m4096_up", "op": "lora", "m": 4096, "k": 4096, "n": 21504, "rank": 64, "adapters": 12, "x": "bf16",
         "w": "bf16", "spread": "runs"},
        # a short sequence's training step of one adapter
        {"name": "lora_train_m64", "op": "lora_train", "m": 64, "k": 2688, "n": 1856, "rank": 8, "adapters": 1,
         "x": "bf16", "w": "bf16", "spread": "runs"},
        # a ragged f32 training step of several adapters, the rank no multiple of anything
        {"name": "lora_train_ragged", "op": "lora_train", "m": 300, "k": 2701, "n": 1999, "rank": 20, "adapters": 3,
         "x": "f32", "w": "f32", "spread": "runs"},
        # a packed training batch of several adapters at once
        {"name": "lora_train_m8192", "op": "lora_train", "m": 8192, "k": 4096, "n": 4096, "rank": 32, "adapters": 4,
         "x": "bf16", "w": "bf16", "spread": "runs"},
    ]


MAX_ROWS = 8192 * 6 * 2688          # the listed batch's dispatched values
MAX_SERVED = 4096 * (4096 + 21504)  # the listed prefill's activations
MAX_TRAINED = 8192 * (4096 + 4096)  # the listed training batch's


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A row length: whole 64s, whole eights or any."""
    v = _log(rng, lo, hi)
    unit = rng.choice([64, 64, 8, 1])
    return max(unit, v // unit * unit)


def draw(rng):
    while True:
        op = rng.choices(["rows", "rows_train", "lora", "lora_train"], [20, 20, 35, 25])[0]
        if op.startswith("rows"):
            experts = rng.choice([8, 16, 60, 64, 128, 256])
            case = {"op": op, "tokens": _log(rng, 1, 16384), "hidden": _width(rng, 128, 4096), "experts": experts,
                    "top_k": rng.randint(1, 8), "x": rng.choice(["bf16", "bf16", "bf16", "f32"])}
            if case["tokens"] * case["top_k"] * case["hidden"] * SIZE[case["x"]] > 2 * MAX_ROWS:
                continue
            return case
        x, w = rng.choice([("bf16", "bf16")] * 3 + [("f32", "f32"), ("bf16", "f32")])
        case = {"op": op, "m": _log(rng, 1, 8192), "k": _width(rng, 64, 21504), "n": _width(rng, 64, 21504),
                "rank": rng.choice([4, 8, 16, 32, 64, rng.randint(1, 64)]), "adapters": _log(rng, 1, 64), "x": x, "w": w,
                "spread": rng.choice(["rows", "runs"])}
        values = case["m"] * (case["k"] + case["n"]) * SIZE[x] // 2
        if values > (MAX_SERVED if op == "lora" else MAX_TRAINED):
            continue
        if case["adapters"] * case["rank"] * (case["k"] + case["n"]) > 64 * 16 * (4096 + 16384):
            continue  # the listed decode batch's adapters
        return case


# ---- inputs -----------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, shape, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(dtype)


def _routes(gen, case):
    """A router's choice: its experts, some liked more than others, and weights that sum to one."""
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    logits = _normal(gen, (t, e)) + _normal(gen, (e,), 0.5)
    top = torch.sigmoid(logits).topk(k, dim=1)
    weights = top.values / top.values.sum(dim=1, keepdim=True)
    return top.indices.to(torch.int32).contiguous(), weights.contiguous()


def _rows_inputs(case, seed):
    gen, dt = _generator(seed), DT[case["x"]]
    indices, weights = _routes(gen, case)
    t, h, slots = case["tokens"], case["hidden"], case["tokens"] * case["top_k"]
    if case["op"] == "rows":
        return {"indices": indices, "weights": weights, "x": _normal(gen, (t, h), 1.0, dt),
                "y": _normal(gen, (slots, h), 0.5, dt)}
    # the forward pass left where each route went; y: the experts' answers, dout and drows: gradients that arrive
    order = indices.reshape(-1).sort(stable=True).indices
    pos = torch.empty_like(order)
    pos[order] = torch.arange(slots, device="cuda")
    return {"pos": pos.to(torch.int32), "weights": weights, "y": _normal(gen, (slots, h), 0.5, dt),
            "dout": _normal(gen, (t, h), 1e-2, dt), "drows": _normal(gen, (slots, h), 1e-2, dt)}


def _ids(gen, case):
    """Adapters of the rows, about one row in ten without: a row's own each, or runs of rows that share one (the
    prompts of a batch)."""
    m, count = case["m"], case["adapters"]
    if case["spread"] == "rows":
        ids = torch.randint(0, count, (m,), generator=gen, device="cuda")
        bare = torch.rand(m, generator=gen, device="cuda") < 0.1
    else:
        runs = min(m, 2 * count)
        cuts = torch.randint(0, m, (runs - 1,), generator=gen, device="cuda").sort().values
        run = torch.searchsorted(cuts, torch.arange(m, device="cuda"), right=True)
        own_run = torch.arange(runs, device="cuda") % count
        ids = own_run[run]
        bare = (torch.rand(runs, generator=gen, device="cuda") < 0.1)[run]
    if m > 1:
        ids = torch.where(bare, -1, ids)
    return ids.to(torch.int32)


def _lora_inputs(case, seed):
    gen, dt, wt = _generator(seed), DT[case["x"]], DT[case["w"]]
    m, k, n, r, count = (case[v] for v in ("m", "k", "n", "rank", "adapters"))
    s = {"ids": _ids(gen, case), "x": _normal(gen, (m, k), 1.0, dt), "base": _normal(gen, (m, n), 1.0, dt),
         "a": _normal(gen, (count, r, k), k ** -0.5, wt), "b": _normal(gen, (count, n, r), r ** -0.5, wt),
         "scales": torch.rand(count, generator=gen, device="cuda") + 0.5}
    if case["op"] == "lora_train":
        s["dout"] = _normal(gen, (m, n), 1e-2, dt)
        s["dx_base"] = _normal(gen, (m, k), 1e-2, dt)
    return s


def _inputs(case, seed):
    return (_rows_inputs if case["op"].startswith("rows") else _lora_inputs)(case, seed)


def prepare(case, seed):
    return {"case": case, **_inputs(case, seed)}


def run(state):
    if own:
        return _run_own(state)
    return {"rows": _plain_rows, "rows_train": _plain_rows_train, "lora": _plain_lora,
            "lora_train": _plain_lora_train}[state["case"]["op"]](state)


# ---- the plain forms: elementary operations in 32 bits ----------------------

def _plain_rows(state):
    case = state["case"]
    t, e, k, h = (case[v] for v in ("tokens", "experts", "top_k", "hidden"))
    flat = state["indices"].reshape(-1).long()
    order = flat.sort(stable=True).indices
    pos = torch.empty_like(order)
    pos[order] = torch.arange(t * k, device="cuda")
    offsets = torch.zeros(e + 1, dtype=torch.int64, device="cuda")
    offsets.scatter_add_(0, flat + 1, torch.ones_like(flat))
    y = state["y"][pos].view(t, k, h).float()
    return {"offsets": offsets.cumsum(0).int(), "perm": order.int(), "pos": pos.int(), "rows": state["x"][order // k],
            "out": (y * state["weights"].unsqueeze(2)).sum(dim=1).to(DT[case["x"]])}


def _plain_rows_train(state):
    case = state["case"]
    t, k, h, dt = case["tokens"], case["top_k"], case["hidden"], DT[case["x"]]
    pos = state["pos"].long()
    dout = state["dout"].float().unsqueeze(1)
    dy = torch.empty((t * k, h), dtype=dt, device="cuda")
    dy[pos] = (dout * state["weights"].unsqueeze(2)).to(dt).view(t * k, h)
    dweights = (state["y"][pos].view(t, k, h).float() * dout).sum(dim=2)
    dx = state["drows"][pos].view(t, k, h).float().sum(dim=1).to(dt)
    return {"dy": dy, "dweights": dweights, "dx": dx}


class _Groups:
    """Rows gathered by adapter, each adapter's padded to the fullest one's; rows without one go to a group of their
    own that is not computed."""

    def __init__(self, ids, count):
        group = torch.where(ids < 0, count, ids.long())
        sizes = torch.zeros(count + 1, dtype=torch.int64, device="cuda")
        sizes.scatter_add_(0, group, torch.ones_like(group))
        self.count, self.most = count, max(1, int(sizes[:count].max()))
        order = group.sort(stable=True)
        rank = torch.arange(len(ids), device="cuda") - (sizes.cumsum(0) - sizes)[order.values]
        with_one = order.values < count
        self.rows, self.at = order.indices[with_one], (order.values * self.most + rank)[with_one]

    def gather(self, v):
        out = torch.zeros((self.count * self.most, v.shape[1]), device="cuda")
        out[self.at] = v[self.rows].float()
        return out.view(self.count, self.most, -1)

    def added(self, base, v):
        out = base.float()
        out[self.rows] += v.reshape(self.count * self.most, -1)[self.at]
        return out


def _lora_products(state, groups, x):
    a, b, s = state["a"].float(), state["b"].float(), state["scales"].view(-1, 1, 1)
    h = torch.bmm(x, a.transpose(1, 2).contiguous())
    return h, torch.bmm(h, b.transpose(1, 2).contiguous()) * s


def _plain_lora(state):
    case, ids = state["case"], state["ids"]
    dt = DT[case["x"]]
    if case["m"] <= case["adapters"]:  # each row against its own adapter's matrices
        at = ids.long().clamp(min=0)
        h = torch.bmm(state["a"][at].float(), state["x"].float().unsqueeze(2))
        y = torch.bmm(state["b"][at].float(), h).squeeze(2) * state["scales"][at].unsqueeze(1)
        return torch.where(ids.unsqueeze(1) < 0, state["base"].float(), state["base"].float() + y).to(dt)
    groups = _Groups(ids, case["adapters"])
    _, y = _lora_products(state, groups, groups.gather(state["x"]))
    return groups.added(state["base"], y).to(dt)


def _plain_lora_train(state):
    dt = DT[state["case"]["x"]]
    groups = _Groups(state["ids"], state["case"]["adapters"])
    x, dout = groups.gather(state["x"]), groups.gather(state["dout"])
    h, y = _lora_products(state, groups, x)
    out = groups.added(state["base"], y).to(dt)
    s = state["scales"].view(-1, 1, 1)
    dh = torch.bmm(dout, state["b"].float()) * s
    dx = groups.added(state["dx_base"], torch.bmm(dh, state["a"].float())).to(dt)
    da = torch.bmm(dh.transpose(1, 2).contiguous(), x)
    db = torch.bmm(dout.transpose(1, 2).contiguous(), h) * s
    return {"out": out, "dx": dx, "da": da, "db": db}


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
    """Entry points with their arguments bound to a layer's buffers, as a serving or training loop keeps them: all but
    the stream, which is the one that is current when a pass runs."""

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

    def _rows(self, case, s):
        t, k, e, h, d = case["tokens"], case["top_k"], case["experts"], case["hidden"], self.dtype(case["x"])
        offsets, perm, pos = (self.empty(v, torch.int32) for v in (e + 1, t * k, t * k))
        rows, out = self.empty((t * k, h), DT[case["x"]]), self.empty((t, h), DT[case["x"]])
        self.add("nh_moe_permute", s["indices"], t, k, e, offsets, perm, pos)
        self.add("nh_moe_dispatch", s["x"], d, pos, None, t, k, h, t * k, rows, d)
        self.add("nh_moe_combine_rows", s["y"], d, pos, s["weights"], None, t, k, h, t * k, out, d)
        return {"offsets": offsets, "perm": perm, "pos": pos, "rows": rows, "out": out}

    def _rows_train(self, case, s):
        t, k, h, d = case["tokens"], case["top_k"], case["hidden"], self.dtype(case["x"])
        dy, dx = self.empty((t * k, h), DT[case["x"]]), self.empty((t, h), DT[case["x"]])
        dweights = self.empty((t, k), torch.float32)
        self.add("nh_moe_combine_rows_backward", s["dout"], d, s["y"], d, s["pos"], s["weights"], t, k, h, t * k, dy,
                 dweights)
        self.add("nh_moe_dispatch_backward", s["drows"], d, None, d, s["pos"], None, t, k, h, t * k, dx, None)
        return {"dy": dy, "dweights": dweights, "dx": dx}

    def onto(self, case, base):
        """Where a call's result goes.  The plain form adds to an f32 base where it stands, but for the rows that it
        takes one by one: so do the calls."""
        one_by_one = case["op"] == "lora" and case["m"] <= case["adapters"]
        return base if case["x"] == "f32" and not one_by_one else self.empty(base.shape, base.dtype)

    def _forward(self, case, s, h):
        sizes = [case[v] for v in ("m", "n", "k", "rank", "adapters")]
        d, w = self.dtype(case["x"]), self.dtype(case["w"])
        out = self.onto(case, s["base"])
        ws = self.workspace("nh_linear_lora_workspace_size", *sizes)
        self.add("nh_linear_lora", s["x"], d, s["ids"], s["a"], s["b"], w, s["scales"], *sizes, s["base"], out, d, h, *ws)
        return out

    def _lora(self, case, s):
        return self._forward(case, s, None)

    def _lora_train(self, case, s):
        sizes = [case[v] for v in ("m", "n", "k", "rank", "adapters")]
        m, n, k, r, count = sizes
        d, w = self.dtype(case["x"]), self.dtype(case["w"])
        h, dx = self.empty((m, r), torch.float32), self.onto(case, s["dx_base"])
        da, db = self.empty((count, r, k), torch.float32), self.empty((count, n, r), torch.float32)
        out = self._forward(case, s, h)
        ws = self.workspace("nh_linear_lora_backward_workspace_size", *sizes)
        self.add("nh_linear_lora_backward", s["x"], d, s["ids"], s["a"], s["b"], w, s["scales"], h, s["dout"], d, *sizes,
                 s["dx_base"], dx, da, db, 0, *ws)
        return {"out": out, "dx": dx, "da": da, "db": db}


def _run_own(state):
    bound = state.get("bound")
    if bound is None:
        bound = state["bound"] = _Bound(state)
    return bound.run()


# ---- cost and expected values -----------------------------------------------

def work(case):
    """Inputs and outputs once each; the multiply-adds of the products and sums."""
    if case["op"].startswith("rows"):
        t, k, h, e = case["tokens"], case["top_k"], case["hidden"], SIZE[case["x"]]
        if case["op"] == "rows":  # x and y in, rows and out out; indices, weights, perm, pos, offsets
            return {"bytes": 2.0 * t * h * e * (1 + k) + 16 * t * k + 4 * (case["experts"] + 1), "flops": 2.0 * t * k * h}
        # dout, y and drows in, dy and dx out; pos, weights, dweights
        return {"bytes": t * h * e * (2.0 + 3 * k) + 12 * t * k, "flops": 4.0 * t * k * h}
    m, k, n, r, count, e = case["m"], case["k"], case["n"], case["rank"], case["adapters"], SIZE[case["x"]]
    live = count * (1 - (1 - 1 / count) ** m) if case["spread"] == "rows" else min(count, m)  # adapters that have rows
    weights = live * r * (k + n) * SIZE[case["w"]] + 4 * count + 4 * m
    if case["op"] == "lora":
        return {"bytes": m * (k + 2.0 * n) * e + weights, "flops": 2.0 * m * r * (k + n)}
    return {"bytes": m * (3.0 * k + 3.0 * n) * e + weights + 4.0 * count * r * (k + n), "flops": 6.0 * m * r * (k + n)}


def _exact_rows(case, seed):
    s = _rows_inputs(case, seed)
    flat = s["indices"].flatten().tolist()
    perm = sorted(range(len(flat)), key=lambda r: flat[r])
    perm_t = torch.tensor(perm, device="cuda")
    pos = torch.empty_like(perm_t)
    pos.scatter_(0, perm_t, torch.arange(len(perm), device="cuda"))
    held = torch.bincount(s["indices"].flatten(), minlength=case["experts"])
    out = torch.zeros((case["tokens"], case["hidden"]), dtype=torch.float64, device="cuda")
    for j in range(case["top_k"]):
        out += s["weights"][:, j, None].double() * s["y"].double()[pos.view(-1, case["top_k"])[:, j]]
    offsets = torch.cat([held.new_zeros(1), held.cumsum(0)])
    return {"offsets": offsets.int(), "perm": perm_t.int(), "pos": pos.int(),
            "rows": s["x"].double()[torch.div(perm_t, case["top_k"], rounding_mode="floor")], "out": out}


def _exact_rows_train(case, seed):
    s = _rows_inputs(case, seed)
    t, k, h = case["tokens"], case["top_k"], case["hidden"]
    pos, dout = s["pos"].view(t, k).long(), s["dout"].double()
    dy = torch.zeros((t * k, h), dtype=torch.float64, device="cuda")
    dx = torch.zeros((t, h), dtype=torch.float64, device="cuda")
    dweights = torch.zeros((t, k), dtype=torch.float64, device="cuda")
    for j in range(k):
        at = pos[:, j]
        dy[at] = dout * s["weights"].double()[:, j:j + 1]
        dweights[:, j] = (s["y"][at].double() * dout).sum(dim=1)
        dx += s["drows"][at].double()
    return {"dy": dy, "dweights": dweights, "dx": dx}


def _exact_lora(case, seed):
    s = _lora_inputs(case, seed)
    train = case["op"] == "lora_train"
    out = s["base"].double()
    if train:
        dx, da = s["dx_base"].double(), torch.zeros(s["a"].shape, dtype=torch.float64, device="cuda")
        db = torch.zeros(s["b"].shape, dtype=torch.float64, device="cuda")
    for n in range(case["adapters"]):
        i = (s["ids"] == n).nonzero().flatten()
        if i.numel() == 0:
            continue
        a, b, scale = s["a"][n].double(), s["b"][n].double(), s["scales"][n].double()
        x = s["x"][i].double()
        h = x @ a.T
        out[i] += scale * (h @ b.T)
        if train:
            dout = s["dout"][i].double() * scale
            dh = dout @ b
            dx[i] += dh @ a
            da[n] = dh.T @ x
            db[n] = dout.T @ h
    return {"out": out, "dx": dx, "da": da, "db": db} if train else out


def exact(case, seed):
    return {"rows": _exact_rows, "rows_train": _exact_rows_train, "lora": _exact_lora,
            "lora_train": _exact_lora}[case["op"]](case, seed)
