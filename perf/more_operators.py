"""The gated layer of routed experts in training, its gradients clipped, and linear layers in 8-bit integers for serving.

A case names an operator and its shape:
  ``gated``        h = act(x Wg^T) * (x Wu^T) in one call; ``keep``: with both products, as the backward pass takes them
  ``gated_grad``   its gradients for the rows and the weights
  ``int8``         rows quantised to 8-bit integers and multiplied with quantised weights, a scale per row and per channel
  ``clip``         the norm over many gradients, and those scaled into the buffers that the optimiser reads
``rows``, ``hidden``, ``width`` (and ``n``, ``inner``) are the extents. With ``experts``, every one of ``tokens`` goes to ``k`` of them, experts are of
unequal popularity, ``drop`` of all entries have no expert, and the rows are the sorted entries.
``own`` false computes the operators from their definitions with elementary torch operations, true calls ``nacho_b200.nacho``.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
TOP = 127.0            # the largest 8-bit integer on both sides of zero
FLOOR = 2.0 ** -110    # of a row's largest magnitude, so that the factor 127 / m stays finite
GELU = (1.5957691216057308, 0.044715)  # 2 sqrt(2 / pi), and the cubic part of the tanh form


# ------------------------------------------------------------------------------------- cases ----

def listed():
    return [
        # the first half of a feed-forward layer for a single token: the weights' bytes
        {"name": "gated_1", "op": "gated", "rows": 1, "hidden": 4096, "width": 4096, "act": "silu", "keep": False, "dtype": "bf16"},
        # the same in training on sizes that divide by nothing
        {"name": "gated_odd", "op": "gated", "rows": 1003, "hidden": 1501, "width": 1100, "act": "gelu", "keep": True, "dtype": "f16"},
        # a dense layer of a training batch: the tensor cores
        {"name": "gated_4k", "op": "gated", "rows": 4096, "hidden": 8192, "width": 4096, "act": "silu", "keep": True, "dtype": "bf16"},
        # the experts of 64 requests, most of them with a few rows: every expert's weights once
        {"name": "gated_experts_64", "op": "gated", "tokens": 64, "experts": 64, "k": 4, "drop": 0.0, "hidden": 1024, "width": 2048, "act": "silu", "keep": False, "dtype": "bf16"},
        # the experts of a training batch whose experts have a capacity
        {"name": "gated_experts_8k", "op": "gated", "tokens": 8192, "experts": 32, "k": 4, "drop": 0.02, "hidden": 2048, "width": 2048, "act": "silu", "keep": True, "dtype": "bf16"},
        # gradients of a small layer whose rows start anywhere
        {"name": "gated_grad_odd", "op": "gated_grad", "rows": 1003, "hidden": 1101, "width": 1100, "act": "gelu", "dtype": "f16"},
        # gradients of the experts of a training batch
        {"name": "gated_grad_experts_4k", "op": "gated_grad", "tokens": 4096, "experts": 16, "k": 4, "drop": 0.0, "hidden": 2048, "width": 2048, "act": "silu", "dtype": "bf16"},
        # a linear layer served for a single token
        {"name": "int8_1", "op": "int8", "rows": 1, "n": 4096, "inner": 4096, "dtype": "bf16"},
        # a linear layer on sizes that divide by nothing, with a 32-bit result
        {"name": "int8_odd", "op": "int8", "rows": 1003, "n": 1500, "inner": 1100, "dtype": "f32"},
        # a linear layer for the prompts of many requests: the tensor cores
        {"name": "int8_8k", "op": "int8", "rows": 8192, "n": 8192, "inner": 8192, "dtype": "bf16"},
        # the gradients of a small layer: only latency counts
        {"name": "clip_small", "op": "clip", "layers": 2, "width": 128, "hidden": 384, "dtype": "f32"},
        # the gradients of a model of 12 layers, 16-bit matrices and 32-bit vectors: device memory
        {"name": "clip_12", "op": "clip", "layers": 12, "width": 2048, "hidden": 4096, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def _size(rng, lo, hi):
    """A size of that range; two of three are multiples of 128 (64 below 256), as layers have them, the others are as they come."""
    v = _log(rng, lo, hi)
    if rng.random() < 0.67:
        v = max(lo, v // (128 if v >= 256 else 64) * (128 if v >= 256 else 64))
    return v


def draw(rng):
    op = rng.choice(["gated", "gated", "gated", "gated_grad", "gated_grad", "int8", "int8", "clip"])
    if op == "clip":
        while True:
            c = {"op": op, "layers": rng.randint(1, 40), "width": _size(rng, 64, 4096), "hidden": _size(rng, 64, 8192), "dtype": rng.choice(["f32", "bf16", "f16"])}
            if sum(math.prod(shape) * SIZES[t] for shape, t in _shapes(c)) <= 1 << 30:
                return c
    names = ("n", "inner") if op == "int8" else ("hidden", "width")
    while True:
        c = {"op": op}
        if rng.random() < 0.5:
            c["rows"] = rows = _log(rng, 1, 8192)
            groups = 1
        else:
            c.update(tokens=_log(rng, 8, 16384), experts=_log(rng, 4, 128), k=rng.randint(1, 4), drop=rng.choice([0.0, 0.0, 0.05]))
            rows, groups = c["tokens"] * c["k"], c["experts"]
        c.update({names[0]: _size(rng, 64, 8192), names[1]: _size(rng, 64, 8192)})
        wide = c[names[0]] * (1 if op == "int8" else 2)
        if rows * wide * c[names[1]] <= (1 << 37) // (2 if op == "gated_grad" else 1) and groups * wide * c[names[1]] <= 1 << 28 and rows * max(wide, c[names[1]]) <= 1 << 28:
            break
    if op == "int8":
        c["dtype"] = rng.choice(["bf16", "f16", "f32"])
    else:
        c.update(act=rng.choice(["silu", "silu", "gelu"]), dtype=rng.choice(["bf16", "bf16", "f16"]))
    if op == "gated":
        c["keep"] = rng.random() < 0.5
    return c


def _shapes(case):
    """Extents and types of the gradients: per layer four square matrices, a gated block's two, and two vectors; an embedding-like table in front."""
    d, h, t = case["width"], case["hidden"], case["dtype"]
    layer = [((d, d), t)] * 4 + [((2 * h, d), t), ((d, h), t), ((d,), "f32"), ((d + 1,), "f32")]
    return [((997, d), t)] + layer * case["layers"]


# ------------------------------------------------------------------------------------ inputs ----

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32) * scale).to(dtype)


def _routing(case, g):
    """Experts of the entries (token by token, -1: none) from the k best of noisy scores."""
    T, E, k = case["tokens"], case["experts"], case["k"]
    scores = torch.randn(T, E, generator=g, device=DEVICE) + torch.randn(E, generator=g, device=DEVICE) * 0.5
    expert = torch.topk(scores, k, dim=1).indices
    if case["drop"]:
        expert = torch.where(torch.rand(T, k, generator=g, device=DEVICE) < case["drop"], torch.full_like(expert, -1), expert)
    return expert.flatten().to(torch.int32)


def prepare(case, seed):
    g, op, dtype = _generator(seed), case["op"], DTYPES[case["dtype"]]
    s = {"op": op, "dtype": dtype, "act": case.get("act"), "keep": case.get("keep", False), "order": None}
    if op == "clip":
        s["gradients"] = [_normal(g, shape, DTYPES[t], 0.01) for shape, t in _shapes(case)]
        s["max_norm"] = 1.0
        # the optimiser reads one long buffer of every type; the scaled gradients go into their places there
        s["buffers"], s["out"] = {}, []
        for t in dict.fromkeys(x.dtype for x in s["gradients"]):
            s["buffers"][t] = torch.empty(sum(x.numel() for x in s["gradients"] if x.dtype == t), dtype=t, device=DEVICE)
        at = dict.fromkeys(s["buffers"], 0)
        for x in s["gradients"]:
            s["out"].append(s["buffers"][x.dtype][at[x.dtype]:at[x.dtype] + x.numel()].view(x.shape))
            at[x.dtype] += x.numel()
        return s
    rows, groups = case.get("rows"), 1
    if rows is None:
        expert = _routing(case, g)
        rows, groups = expert.numel(), case["experts"]
        counts = torch.bincount(expert[expert >= 0].long(), minlength=groups)
        s["bounds"] = [0] + torch.cumsum(counts, 0).tolist()
    else:
        s["bounds"] = [0, rows]
    if op == "int8":
        s["x"] = _normal(g, (rows, case["inner"]), dtype)
        w = _normal(g, (groups, case["n"], case["inner"]), torch.float32, case["inner"] ** -0.5)
        s["scales"] = w.abs().amax(dim=2) / TOP
        s["codes"] = torch.round(w / s["scales"][:, :, None]).clamp(-TOP, TOP).to(torch.int8)
    else:
        s["x"] = _normal(g, (rows, case["width"]), dtype)
        s["w"] = _normal(g, (groups, 2 * case["hidden"], case["width"]), dtype, case["width"] ** -0.5)
    if op == "gated_grad":
        s["both"] = _normal(g, (rows, 2 * case["hidden"]), dtype)
        s["dh"] = _normal(g, (rows, case["hidden"]), dtype)
    # what else a program has in hand: the order that sorted the rows, the weights as the products take them
    if own:
        from nacho_b200 import nacho
        if "tokens" in case:
            offsets = torch.arange(0, rows + 1, case["k"], dtype=torch.int32, device=DEVICE)
            r = nacho.CSR_gpu(offsets, expert, torch.ones(rows, device=DEVICE), (case["tokens"], groups))
            s["order"] = nacho.gpu_expert_order(r)
        if op == "int8":
            s["weights"] = nacho.to_int8_rows(s["codes"], s["scales"])
    return s


# --------------------------------------------------------------------------------- plain forms ----

def _gate(g, act):
    """sigmoid(p(g)) of act(g) = g sigmoid(p(g)), and the derivative of p."""
    if act == "silu":
        return 1 / (1 + torch.exp(-g)), torch.ones_like(g)
    a, b = GELU
    return 1 / (1 + torch.exp(-a * (g + b * g * g * g))), a * (1 + 3 * b * g * g)


def _by_group(a, w, bounds):
    y = torch.zeros(a.shape[0], w.shape[1], device=DEVICE)
    for e in range(len(bounds) - 1):
        y[bounds[e]:bounds[e + 1]] = a[bounds[e]:bounds[e + 1]] @ w[e].t()
    return y


def _quantised(x):
    m = x.abs().amax(dim=1, keepdim=True).clamp(min=FLOOR)
    top = torch.full_like(m, TOP)
    return torch.round(x * (top / m)), m / top


def _plain(s):
    op, dtype = s["op"], s["dtype"]
    if op == "clip":
        norm = torch.sqrt(sum((x.double() * x.double()).sum() for x in s["gradients"])).float()
        factor = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
        return norm, [torch.cat([(x.float() * factor).to(t).flatten() for x in s["gradients"] if x.dtype == t]) for t in s["buffers"]]
    x, bounds = s["x"].float(), s["bounds"]
    if op == "int8":
        q, scale = _quantised(x)
        y = _by_group(q, s["codes"].float(), bounds)
        for e in range(len(bounds) - 1):
            y[bounds[e]:bounds[e + 1]] *= scale[bounds[e]:bounds[e + 1]] * s["scales"][e]
        return y.to(dtype)
    w = s["w"].float()
    hidden = w.shape[1] // 2
    if op == "gated":
        both = _by_group(x, w, bounds)
        g, u = both[:, :hidden], both[:, hidden:]
        h = (g * _gate(g, s["act"])[0] * u).to(dtype)
        return (h, both.to(dtype)) if s["keep"] else h
    dh, g, u = s["dh"].float(), s["both"][:, :hidden].float(), s["both"][:, hidden:].float()
    soft, slope = _gate(g, s["act"])
    dboth = torch.cat([dh * u * (soft + g * soft * (1 - soft) * slope), dh * g * soft], dim=1)
    dx = _by_group(dboth, w.transpose(1, 2), bounds)
    dw = torch.zeros_like(w)
    for e in range(len(bounds) - 1):
        dw[e] = dboth[bounds[e]:bounds[e + 1]].t() @ x[bounds[e]:bounds[e + 1]]
    return dx.to(dtype), dw.to(dtype)


# ---------------------------------------------------------------------------------- one pass ----

def run(s):
    if not own:
        return _plain(s)
    from nacho_b200 import nacho
    op = s["op"]
    if op == "gated":
        return nacho.gpu_gated_product(s["x"], s["w"], s["order"], activation=s["act"], keep=s["keep"])
    if op == "gated_grad":
        return nacho.gpu_gated_product_grad(s["dh"], s["both"], s["x"], s["w"], s["order"], activation=s["act"])
    if op == "int8":
        return nacho.gpu_int8_product(nacho.to_int8_rows(s["x"]), s["weights"], s["order"], dtype=s["dtype"])
    return nacho.gpu_clip_gradients(s["gradients"], s["max_norm"], out=s["out"]), list(s["buffers"].values())


# ----------------------------------------------------------------------------- work and truth ----

def work(case):
    op, size = case["op"], SIZES[case["dtype"]]
    if op == "clip":
        return {"bytes": sum(2 * SIZES[t] * math.prod(shape) for shape, t in _shapes(case)) + 4, "flops": sum(3 * math.prod(shape) for shape, _ in _shapes(case))}
    rows, used, groups = case.get("rows"), 1.0, 1
    kept = rows
    if rows is None:
        rows, groups = case["tokens"] * case["k"], case["experts"]
        kept = rows * (1.0 - case["drop"])
        used = groups * (1.0 - (1.0 - 1.0 / groups) ** kept)  # experts that have rows at all
    if op == "int8":
        n, k = case["n"], case["inner"]
        return {"bytes": int(size * (kept * k + rows * n) + used * n * (k + 4)), "flops": int(2 * kept * n * k)}
    h, d = case["hidden"], case["width"]
    if op == "gated":
        return {"bytes": int(size * (kept * d + used * 2 * h * d + rows * h * (3 if case["keep"] else 1))), "flops": int(4 * kept * h * d)}
    return {"bytes": int(size * (kept * (3 * h + d) + used * 2 * h * d + rows * d + groups * 2 * h * d)), "flops": int(8 * kept * h * d)}


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "clip":
        squares = torch.stack([torch.linalg.vector_norm(x.double()) ** 2 for x in s["gradients"]])
        norm = torch.sqrt(squares.sum())
        factor = min(1.0, s["max_norm"] / (norm.item() + 1e-6))
        return norm, [torch.cat([x.double().flatten() for x in s["gradients"] if x.dtype == t]) * factor for t in s["buffers"]]
    bounds, x = s["bounds"], s["x"].double()
    parts = [slice(a, b) for a, b in zip(bounds[:-1], bounds[1:])]
    if op == "int8":
        # the two factors of a row are 32-bit numbers by definition, and so is the product that is rounded to a whole number
        m = s["x"].float().abs().max(dim=1, keepdim=True).values.double().clamp(min=FLOOR)
        codes = torch.round(s["x"].float() * (TOP / m).float()).double()
        y = torch.zeros(x.shape[0], case["n"], dtype=torch.float64, device=DEVICE)
        for e, part in enumerate(parts):
            y[part] = (codes[part] @ s["codes"][e].double().t()) * (m[part] / TOP).float().double() * s["scales"][e].double()
        return y
    h = case["hidden"]
    if op == "gated":
        y, both = (torch.zeros(x.shape[0], n, dtype=torch.float64, device=DEVICE) for n in (h, 2 * h))
        for e, part in enumerate(parts):
            both[part] = x[part] @ s["w"][e].double().t()
        g = both[:, :h]
        y = g * torch.sigmoid(g if case["act"] == "silu" else 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)) * both[:, h:]
        return (y, both) if s["keep"] else y
    g, u, dh = s["both"][:, :h].double(), s["both"][:, h:].double(), s["dh"].double()
    if case["act"] == "silu":
        act, slope = g * torch.sigmoid(g), torch.sigmoid(g) * (1 + g * torch.sigmoid(-g))
    else:
        z = math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
        t = torch.tanh(z)
        act, slope = 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g * g)
    dg, du = dh * u * slope, dh * act
    dx = torch.zeros_like(x)
    dw = torch.zeros(s["w"].shape, dtype=torch.float64, device=DEVICE)
    for e, part in enumerate(parts):
        w = s["w"][e].double()
        dx[part] = dg[part] @ w[:h] + du[part] @ w[h:]
        dw[e] = torch.cat([dg[part].t() @ x[part], du[part].t() @ x[part]])
    return dx, dw
