"""Measured cases of the Dense-layer operators: dropout from a counter-based generator, the 8-bit integer product with a
scale per row and channel, and the products grouped by expert with ragged sizes, forward and backward.

`run` computes each of them in its plain form (elementary torch operations in 32 bits), or, where `own` is true, through
weather_model_amd.ops.  `exact` is the same from the definitions, in 64 bits.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}


def listed():
    return [
        # One training step's dropout on the Conv3D model's hidden layer: Dense(640), batch 16 -- the smallest call, all latency.
        {"name": "dropout_layer", "op": "dropout", "rows": 16, "cols": 640, "type": "float32", "p": 0.5, "residual": False, "offset": 0},
        # Activations of a wide layer over a batch of grid points, added to the residual path; forward and backward.
        {"name": "dropout_residual", "op": "dropout", "rows": 32768, "cols": 2048, "type": "bfloat16", "p": 0.1, "residual": True, "offset": 1 << 33},
        # singleRegression's 6^3-cube targets with one more column, an odd row and an odd counter offset; float32.
        {"name": "dropout_odd", "op": "dropout", "rows": 30011, "cols": 217, "type": "float32", "p": 0.37, "residual": False, "offset": 12345},
        # One grid cube answered by the Conv3D model's output layer, Dense(640 -> 8000): a single row.
        {"name": "int8_one_row", "op": "int8", "rows": 1, "cols": 8000, "inner": 640, "type": "float32", "relu": False},
        # A handful of rows through a wide layer: bound by reading the weights.
        {"name": "int8_few_rows", "op": "int8", "rows": 8, "cols": 8192, "inner": 8192, "type": "bfloat16", "relu": True},
        # Odd sizes on every side.
        {"name": "int8_odd", "op": "int8", "rows": 777, "cols": 1001, "inner": 1283, "type": "float16", "relu": False},
        # A whole field's rows at once: bound by the matrix cores.
        {"name": "int8_field", "op": "int8", "rows": 8192, "cols": 8192, "inner": 4096, "type": "bfloat16", "relu": False},
        # A few rows over many experts, some of which get none: bound by reading the weights of the others.
        {"name": "experts_few_rows", "op": "experts", "rows": 48, "cols": 2048, "inner": 2048, "groups": 16, "empty": 4, "behind": 0,
         "split": 1, "type": "bfloat16", "relu": True, "train": False},
        # singleRegression's map 432 -> 216, one for each of data.py's eleven variables, ragged numbers of rows, float32.
        {"name": "experts_regression", "op": "experts", "rows": 45001, "cols": 216, "inner": 432, "groups": 11, "empty": 0, "behind": 7,
         "split": 2, "type": "float32", "relu": False, "train": False},
        # A training step of one layer: forward and the gradients of rows, weights and biases, in the framework's own type.
        {"name": "experts_step_f32", "op": "experts", "rows": 8191, "cols": 1024, "inner": 1024, "groups": 8, "empty": 1, "behind": 0,
         "split": 3, "type": "float32", "relu": False, "train": True},
        # The same in bfloat16 at a size that fills the card.
        {"name": "experts_step_bf16", "op": "experts", "rows": 16384, "cols": 4096, "inner": 2048, "groups": 16, "empty": 0, "behind": 100,
         "split": 4, "type": "bfloat16", "relu": False, "train": True},
        # Small groups with an odd inner size, trained: half precision.
        {"name": "experts_step_odd", "op": "experts", "rows": 2999, "cols": 333, "inner": 515, "groups": 33, "empty": 5, "behind": 3,
         "split": 5, "type": "float16", "relu": False, "train": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("dropout", "int8", "experts"))
    kind = rng.choice(("float32", "bfloat16", "float16"))
    if op == "dropout":
        cols = _log(rng, 16, 8192)
        rows = _log(rng, 1, max(1, min(65536, 60_000_000 // cols)))
        return {"op": op, "rows": rows, "cols": cols, "type": kind, "p": rng.choice((0.05, 0.1, 0.25, 0.5, 0.9)),
                "residual": rng.random() < 0.5, "offset": rng.choice((0, 8 * rng.randrange(1 << 36), rng.randrange(1 << 40)))}
    if op == "int8":
        cols, inner = _log(rng, 16, 8192), _log(rng, 16, 8192)
        rows = _log(rng, 1, 8192)
        rows = max(1, min(rows, 200_000_000_000 // (cols * inner)))
        return {"op": op, "rows": rows, "cols": cols, "inner": inner, "type": kind, "relu": rng.random() < 0.5}
    groups = _log(rng, 1, 64)
    cols, inner = _log(rng, 16, 4096), _log(rng, 16, 4096)
    inner = max(16, min(inner, 200_000_000 // (cols * groups)))
    train = rng.random() < 0.5
    most = (60 if train else 180) * (1 if kind != "float32" else 0.25) * 1e9
    rows = max(1, min(_log(rng, 1, 32768), int(most / (cols * inner))))
    return {"op": op, "rows": rows, "cols": cols, "inner": inner, "groups": groups, "empty": rng.randrange(groups), "behind": rng.randrange(1 + rows // 8),
            "split": rng.randrange(1000), "type": kind, "relu": rng.random() < 0.5 and not train, "train": train}


def _sizes(case):
    """Rows of each group: uneven shares of what `behind` leaves, `empty` groups without any."""
    rng = random.Random(case["split"])
    live = case["groups"] - case["empty"]
    share = [0.25 + rng.random() for _ in range(live)]
    total, rows, sizes, done = sum(share), case["rows"] - case["behind"], [], 0.0
    for s in share:
        before, done = done, done + s
        sizes.append(int(round(rows * done / total)) - int(round(rows * before / total)))
    return sizes + [0] * case["empty"]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["type"]]
    rows, cols = case["rows"], case["cols"]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=gen, device="cuda") * scale

    if case["op"] == "dropout":
        s = {"x": normal(rows, cols).to(kind), "gy": normal(rows, cols).to(kind), "seed": seed % 1000003}
        s["residual"] = normal(rows, cols).to(kind) if case["residual"] else None
        return {"case": case, **s}
    inner = case["inner"]
    if case["op"] == "int8":
        w = normal(cols, inner, scale=inner ** -0.5)
        scale = w.abs().amax(1) / torch.full((cols,), 127.0, device="cuda")
        q = torch.round(w / scale[:, None]).clamp_(-127, 127).to(torch.int8)
        # rows of unlike size, as activations have
        x = normal(rows, inner) * torch.exp(normal(rows, 1))
        return {"case": case, "x": x.to(kind), "q": q, "scale": scale, "bias": normal(cols, scale=0.1)}
    sizes = _sizes(case)
    random.Random(seed).shuffle(sizes)                       # which expert gets how many rows differs from seed to seed
    offsets = torch.tensor([sum(sizes[:g]) for g in range(len(sizes) + 1)], dtype=torch.int64, device="cuda")
    groups = case["groups"]
    x = normal(rows, inner).clamp_(min=0.0).to(kind)         # what a ReLU below leaves
    w = normal(groups, cols, inner, scale=inner ** -0.5).to(kind)
    return {"case": case, "x": x, "w": w, "bias": normal(groups, cols, scale=0.1).to(kind), "offsets": offsets, "sizes": sizes, "most": max(sizes),
            "gy": normal(rows, cols).to(kind) if case["train"] else None}


# ------------------------------------------------------------------ plain forms

def _signed(v):
    return v - (1 << 64) if v >= 1 << 63 else v


def _hash64(seed, index):
    """The framework's counter-based hash (weather_model_amd.synth.hash64) on int64 tensors."""
    z = index + _signed(((seed + 1) & 0xFFFFFFFF) * 0x9E3779B97F4A7C15 & (1 << 64) - 1)
    z = (z ^ ((z >> 30) & (1 << 34) - 1)) * _signed(0xBF58476D1CE4E5B9)
    z = (z ^ ((z >> 27) & (1 << 37) - 1)) * _signed(0x94D049BB133111EB)
    return z ^ ((z >> 31) & (1 << 33) - 1)


def _kept(n, p, seed, offset):
    """Which of the elements offset .. offset + n - 1 stay: element e draws 32 bits, the upper 16 from the hash of e // 4, the
    lower 16 from the hash of that, each at bits 16 (e % 4), and is dropped if they are below p 2^32."""
    first, last = offset // 4, (offset + n - 1) // 4
    upper = _hash64(seed, torch.arange(first, last + 1, device="cuda"))
    lower = _hash64(seed, upper)
    at = torch.arange(0, 64, 16, device="cuda")
    bits = ((upper[:, None] >> at & 0xFFFF) << 16) + (lower[:, None] >> at & 0xFFFF)
    bits = bits.reshape(-1)[offset - 4 * first:][:n]
    return bits >= int(round(p * 2 ** 32))


def _scale(p):
    return 2.0 ** 32 / (2 ** 32 - int(round(p * 2 ** 32)))


def _dropout(s):
    c, x, gy = s["case"], s["x"], s["gy"]
    if own:
        from weather_model_amd import ops
        y = ops.dropout_forward(x, c["p"], s["seed"], offset=c["offset"], residual=s["residual"])
        return {"y": y, "gx": ops.dropout_backward(gy, c["p"], s["seed"], offset=c["offset"])}
    keep = _kept(x.numel(), c["p"], s["seed"], c["offset"]).view(x.shape)
    y = torch.where(keep, x.float() * _scale(c["p"]), 0.0)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"y": y.to(x.dtype), "gx": torch.where(keep, gy.float() * _scale(c["p"]), 0.0).to(x.dtype)}


def _int8(s):
    c, x = s["case"], s["x"]
    if own:
        from weather_model_amd import ops
        return {"y": ops.dense_i8(x, s["q"], s["scale"], s["bias"], relu=c["relu"])}
    x = x.float()
    scale = x.abs().amax(1, keepdim=True) / torch.full((1, 1), 127.0, device="cuda")
    q = torch.where(scale > 0, torch.round(x / scale), 0.0).clamp(-127, 127)
    y = (q @ s["q"].float().t()) * scale * s["scale"] + s["bias"]
    return {"y": (torch.relu(y) if c["relu"] else y).to(s["x"].dtype)}


def _experts(s):
    c, x, w = s["case"], s["x"], s["w"]
    if own:
        from weather_model_amd import ops
        out = {"y": ops.dense_grouped_forward(x, w, s["offsets"], s["bias"], relu=c["relu"])}
        if c["train"]:
            out["gx"], out["gw"], out["gb"] = ops.dense_grouped_backward(x, w, s["offsets"], s["gy"], mask_below=x)
        return out
    rows = torch.arange(c["rows"], device="cuda")
    group = torch.searchsorted(s["offsets"], rows, right=True) - 1
    # rows behind the last group belong to none: zeros
    rows, group = rows[: c["rows"] - c["behind"]], group[: c["rows"] - c["behind"]]
    place = rows - s["offsets"][group]
    packed = x.new_zeros((c["groups"], max(1, s["most"]), c["inner"]), dtype=torch.float32)
    packed[group, place] = x[rows].float()
    full = w.float()
    y = torch.bmm(packed, full.transpose(1, 2)) + s["bias"].float()[:, None]
    y = torch.relu(y) if c["relu"] else y
    out = {"y": x.new_zeros((c["rows"], c["cols"]))}
    out["y"][rows] = y[group, place].to(x.dtype)
    if c["train"]:
        grad = x.new_zeros((c["groups"], max(1, s["most"]), c["cols"]), dtype=torch.float32)
        grad[group, place] = s["gy"][rows].float()
        gx = torch.bmm(grad, full)[group, place]
        out["gx"] = x.new_zeros((c["rows"], c["inner"]))
        out["gx"][rows] = torch.where(x[rows] > 0, gx, 0.0).to(x.dtype)
        out["gw"] = torch.bmm(grad.transpose(1, 2), packed).to(x.dtype)
        out["gb"] = grad.sum(1).to(x.dtype)
    return out


def run(state):
    return {"dropout": _dropout, "int8": _int8, "experts": _experts}[state["case"]["op"]](state)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    rows, cols, size = case["rows"], case["cols"], SIZE[case["type"]]
    if case["op"] == "dropout":                              # x and gy in, y and gx out
        return {"bytes": rows * cols * size * (5 if case["residual"] else 4), "flops": rows * cols * 2}
    inner = case["inner"]
    if case["op"] == "int8":                                 # the weights are bytes, scales and biases float32
        return {"bytes": rows * (inner + cols) * size + cols * inner + 8 * cols, "flops": 2 * rows * cols * inner}
    live, inside = sum(n > 0 for n in _sizes(case)), rows - case["behind"]
    b = (inside * inner + rows * cols + live * cols * (inner + 1)) * size
    if case["train"]:                                        # x, gy and w once more, gx, gw and gb out
        b += (inside * (inner + cols) + rows * inner + live * cols * inner + case["groups"] * cols * (inner + 1)) * size
    return {"bytes": b, "flops": 2 * inside * cols * inner * (3 if case["train"] else 1)}


# ------------------------------------------------------------------ the definitions in 64 bits

def _np_hash(seed, z):
    with np.errstate(over="ignore"):
        z = z + np.uint64((seed + 1) % 2 ** 32) * np.uint64(0x9E3779B97F4A7C15)
        for shift, factor in ((30, 0xBF58476D1CE4E5B9), (27, 0x94D049BB133111EB)):
            z = (z ^ (z >> np.uint64(shift))) * np.uint64(factor)
        return z ^ (z >> np.uint64(31))


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "dropout":
        if x.numel() > 1 << 23:
            return None                                      # minutes of host arithmetic
        e = np.arange(x.numel(), dtype=np.uint64) + np.uint64(case["offset"])
        upper = _np_hash(s["seed"], e >> np.uint64(2))
        at = (e & np.uint64(3)) * np.uint64(16)
        draws = ((upper >> at) % np.uint64(65536)) * np.uint64(65536) + (_np_hash(s["seed"], upper) >> at) % np.uint64(65536)
        least = round(case["p"] * 2 ** 32)
        factor = torch.from_numpy((draws >= np.uint64(least)) * (1.0 / (1.0 - least / 2 ** 32))).cuda().view(x.shape)
        y = x * factor if s["residual"] is None else x * factor + s["residual"].double()
        return {"y": y, "gx": s["gy"].double() * factor}
    if case["op"] == "int8":
        # the row's scale is the float32 nearest to max / 127, its codes round the float32 quotients: both are part of the definition
        top = x.abs().max(dim=1).values
        scale = (top / 127.0).float().double()
        safe = torch.where(scale == 0, torch.ones_like(scale), scale)
        code = torch.round((x / safe.unsqueeze(1)).float().double()).clamp(-127, 127) * (scale != 0).unsqueeze(1)
        y = torch.mm(code, s["q"].double().t().contiguous())
        y = y * scale.unsqueeze(1) * s["scale"].double().unsqueeze(0) + s["bias"].double().unsqueeze(0)
        return {"y": y.clamp(min=0) if case["relu"] else y}
    w, b = s["w"].double(), s["bias"].double()
    y = torch.zeros((case["rows"], case["cols"]), dtype=torch.float64, device="cuda")
    gx, gw, gb = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    at = 0
    for g, n in enumerate(s["sizes"]):
        part = slice(at, at + n)
        at += n
        if n == 0:
            continue
        y[part] = x[part] @ w[g].t().contiguous() + b[g]
        if case["train"]:
            gy = s["gy"][part].double()
            gx[part] = (gy @ w[g]) * (x[part] > 0)
            gw[g] = gy.t().contiguous() @ x[part]
            gb[g] = gy.sum(0)
    if case["relu"]:
        y = y.clamp(min=0)
    return {"y": y, "gx": gx, "gw": gw, "gb": gb} if case["train"] else {"y": y}
