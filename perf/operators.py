"""The operators around a router whose decision is a CSR matrix (tokens x experts, values = gate weights): tokens sorted by expert,
8-bit products of the sorted rows with every expert's weights, and the way back, with their gradients.

A case names an operator and its shape:
  ``tokens``, ``experts``, ``k``   each token goes to ``k`` experts (with ``ragged`` to 0 .. k of them; ``drop`` of all entries have no
                                   expert, as where a capacity overflows). Experts are of unequal popularity.
  ``width``                        the tokens' width (sort, unsort)
  ``rows``, ``n``, ``inner``       rows x inner times (n x inner) transposed (products; by expert, the rows are the sorted tokens)
``own`` false computes the operators from their definitions with elementary torch operations, true calls ``nacho_b200.nacho``.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 128
TOP = 448.0            # the largest e4m3 number
FLOOR = 2.0 ** -110    # of a block's largest magnitude, so that the factor 448 / m stays finite


# ------------------------------------------------------------------------------------- cases ----

def listed():
    return [
        # one step of serving 16 requests: only latency counts
        {"name": "sort_16", "op": "sort", "tokens": 16, "experts": 64, "k": 4, "width": 2048, "dtype": "bf16", "ragged": False, "drop": 0.0},
        # a training batch on its way to the experts, bound by device memory
        {"name": "sort_32k", "op": "sort", "tokens": 32768, "experts": 64, "k": 4, "width": 4096, "dtype": "bf16", "ragged": False, "drop": 0.0},
        # the gradient of that on ragged sizes: rows that start anywhere, tokens without an expert
        {"name": "sort_grad_odd", "op": "sort_grad", "tokens": 5003, "experts": 60, "k": 3, "width": 1001, "dtype": "f32", "ragged": True, "drop": 0.05},
        # the way back while serving 64 requests
        {"name": "unsort_64", "op": "unsort", "tokens": 64, "experts": 128, "k": 8, "width": 2048, "dtype": "f16", "ragged": False, "drop": 0.0},
        # the way back of a training batch whose experts have a capacity
        {"name": "unsort_16k", "op": "unsort", "tokens": 16384, "experts": 128, "k": 8, "width": 4096, "dtype": "bf16", "ragged": False, "drop": 0.1},
        # and its gradient, for the experts' results and the gate weights
        {"name": "unsort_grad_8k", "op": "unsort_grad", "tokens": 8192, "experts": 32, "k": 4, "width": 4096, "dtype": "bf16", "ragged": True, "drop": 0.0},
        # a linear layer for a single token: the weights' bytes
        {"name": "product_1", "op": "product", "rows": 1, "n": 4096, "inner": 4096, "dtype": "bf16"},
        # a linear layer on sizes that divide by nothing, with a 32-bit result
        {"name": "product_odd", "op": "product", "rows": 1003, "n": 1500, "inner": 1100, "dtype": "f32"},
        # a linear layer of a large batch: the tensor cores
        {"name": "product_8k", "op": "product", "rows": 8192, "n": 8192, "inner": 8192, "dtype": "bf16"},
        # the experts of 64 requests, most of them with a few rows: every expert's weights once
        {"name": "experts_64", "op": "experts", "tokens": 64, "experts": 64, "k": 4, "n": 2048, "inner": 2048, "dtype": "bf16", "ragged": False, "drop": 0.0},
        # the experts of a training batch
        {"name": "experts_8k", "op": "experts", "tokens": 8192, "experts": 32, "k": 4, "n": 4096, "inner": 2048, "dtype": "bf16", "ragged": False, "drop": 0.02},
        # and the gradients of their rows and weights
        {"name": "experts_grad_4k", "op": "experts_grad", "tokens": 4096, "experts": 16, "k": 4, "n": 2048, "inner": 2048, "dtype": "bf16", "ragged": False, "drop": 0.0},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def _size(rng, lo, hi):
    """A size of that range; two of three are multiples of 128 (64 below 256), as layers have them, the others are as they come."""
    v = _log(rng, lo, hi)
    step = 256 if v >= 2048 else 128 if v >= 256 else 64
    if rng.random() < 0.67:
        v = v // step * step
    return v + step if v == 3072 else v  # as this repository's configurations, which do not have that size


def draw(rng):
    op = rng.choice(["sort", "sort_grad", "unsort", "unsort_grad", "product", "product", "experts", "experts", "experts_grad"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "product":
        while True:
            c = {"op": op, "rows": _log(rng, 1, 8192), "n": _size(rng, 200, 8192), "inner": _size(rng, 200, 8192), "dtype": dtype}
            if c["rows"] * c["n"] * c["inner"] <= 1 << 38:
                return c
    while True:
        c = {"op": op, "tokens": _log(rng, 8, 32768), "experts": _log(rng, 4, 256), "k": rng.randint(1, 8)}
        c["k"] = min(c["k"], c["experts"])
        if op.startswith("experts"):
            c.update(n=_size(rng, 200, 4096), inner=_size(rng, 200, 4096))
            fits = c["tokens"] * c["k"] * c["n"] * c["inner"] <= 1 << 38 and c["experts"] * c["n"] * c["inner"] <= 1 << 29 and \
                c["tokens"] * c["k"] * max(c["n"], c["inner"]) <= 1 << 28
        else:
            c.update(width=_size(rng, 200, 8192))
            fits = c["tokens"] * c["k"] * c["width"] <= (1 << 28 if dtype == "f32" else 1 << 29)
        if fits:
            c.update(dtype=dtype, ragged=rng.random() < 0.4, drop=rng.choice([0.0, 0.0, 0.03, 0.2]))
            return c


# ------------------------------------------------------------------------------------ inputs ----

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32) * scale).to(dtype)


def _routing(case, g):
    """Row offsets, experts and gate weights of a router's decision: the k best of noisy scores, weights by a softmax over those."""
    T, E, k = case["tokens"], case["experts"], case["k"]
    popularity = torch.randn(E, generator=g, device=DEVICE) * 0.5
    scores = torch.randn(T, E, generator=g, device=DEVICE) + popularity
    best, expert = torch.topk(scores, k, dim=1)
    weight = torch.softmax(best, dim=1)
    lengths = torch.full((T,), k, dtype=torch.int64, device=DEVICE)
    if case["ragged"]:
        lengths = (torch.arange(T, device=DEVICE) % (k + 1))[torch.randperm(T, generator=g, device=DEVICE)]
    if case["drop"]:
        expert = torch.where(torch.rand(T, k, generator=g, device=DEVICE) < case["drop"], torch.full_like(expert, -1), expert)
    there = torch.arange(k, device=DEVICE)[None, :] < lengths[:, None]
    offsets = torch.zeros(T + 1, dtype=torch.int64, device=DEVICE)
    offsets[1:] = torch.cumsum(lengths, 0)
    return offsets.to(torch.int32), expert[there].to(torch.int32), weight[there].contiguous()


def _codes(w):
    """8-bit weights (groups, n, inner) and a scale per 128 x 128, as a checkpoint holds them."""
    groups, n, inner = w.shape
    nb, kb = -(-n // BLOCK), -(-inner // BLOCK)
    wide = torch.zeros(groups, nb * BLOCK, kb * BLOCK, device=DEVICE)
    wide[:, :n, :inner] = w
    tiles = wide.view(groups, nb, BLOCK, kb, BLOCK)
    scales = tiles.abs().amax(dim=(2, 4)).clamp(min=1e-20) / 448
    q = (tiles / scales[:, :, None, :, None]).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
    return q.view(groups, nb * BLOCK, kb * BLOCK)[:, :n, :inner].contiguous(), scales


def prepare(case, seed):
    g, op, dtype = _generator(seed), case["op"], DTYPES[case["dtype"]]
    s = {"op": op, "dtype": dtype}
    if op != "product":
        s["offsets"], s["experts"], s["weights"] = _routing(case, g)
        s["shape"], s["k"] = (case["tokens"], case["experts"]), case["k"]
        n = s["experts"].numel()
    if op in ("sort", "experts"):
        s["x"] = _normal(g, (case["tokens"], case.get("width", case.get("inner"))), dtype)
    elif op == "sort_grad":
        s["dxs"] = _normal(g, (n, case["width"]), dtype)
    elif op in ("unsort", "unsort_grad"):
        s["z"] = _normal(g, (n, case["width"]), dtype)
    if op == "unsort_grad":
        s["dy"] = _normal(g, (case["tokens"], case["width"]), dtype)
    if op == "product":
        s["x"] = _normal(g, (case["rows"], case["inner"]), dtype)
    if op == "experts_grad":
        s["xs"] = _normal(g, (n, case["inner"]), dtype)
        s["dy"] = _normal(g, (n, case["n"]), dtype)
    if op in ("product", "experts", "experts_grad"):
        groups = 1 if op == "product" else case["experts"]
        s["codes"], s["scales"] = _codes(_normal(g, (groups, case["n"], case["inner"]), torch.float32, case["inner"] ** -0.5))
    # what else a program has in hand: the operands' objects, the order that the forward pass left, the experts' row counts on the host
    if own:
        from nacho_b200 import nacho
        if op != "product":
            s["r"] = nacho.CSR_gpu(s["offsets"], s["experts"], s["weights"], s["shape"])
            if op not in ("sort", "experts"):
                s["order"] = nacho.gpu_expert_order(s["r"])
        if "codes" in s:
            s["w"] = nacho.to_fp8_tiles(s["codes"], s["scales"])
    elif op != "product":
        s["order"] = _order(s)
        s["bounds"] = s["order"][0].tolist()
    return s


# --------------------------------------------------------------------------------- plain forms ----

def _order(s):
    """offsets (experts + 1), rows (token of every slot), slots (slot of every entry)."""
    T, E = s["shape"]
    n = s["experts"].numel()
    key = s["experts"].long()
    key = torch.where((key < 0) | (key >= E), torch.full_like(key, E), key)
    by_key = torch.argsort(key, stable=True)
    start = torch.zeros(E + 1, dtype=torch.int64, device=DEVICE)
    start[1:] = torch.cumsum(torch.bincount(key, minlength=E + 1)[:E], 0)
    token = torch.searchsorted(s["offsets"].long(), torch.arange(n, device=DEVICE), right=True) - 1
    slots = torch.empty_like(key)
    slots[by_key] = torch.arange(n, device=DEVICE)
    kept = key < E
    rows = torch.where(kept[by_key], token[by_key], torch.full_like(key, -1))
    slots = torch.where(kept, slots, torch.full_like(slots, -1))
    return start.to(torch.int32), rows.to(torch.int32), slots.to(torch.int32)


def _sorted(x, rows):
    xs = x[rows.clamp(min=0).long()]
    return torch.where((rows >= 0)[:, None], xs, torch.zeros_like(xs))


def _steps(s):
    """The j-th entry of every token, for j = 0 .. k - 1: which tokens have it and kept it, the entry, its slot."""
    first, last, slots = s["offsets"][:-1].long(), s["offsets"][1:].long(), s["order"][2].long()
    for j in range(s["k"]):
        entry = first + j
        has = entry < last
        entry = entry[has]
        slot = slots[entry]
        kept = slot >= 0
        yield torch.nonzero(has).squeeze(1)[kept], entry[kept], slot[kept]


def _gathered(s, z, weights, tokens):
    y = torch.zeros(tokens, z.shape[1], device=DEVICE)
    for token, entry, slot in _steps(s):
        part = z[slot].float()
        if weights is not None:
            part = part * weights[entry][:, None]
        y[token] += part
    return y


def _blocks(x):
    """x as the 8-bit rows stand for it: a scale for every 128 entries of a row."""
    rows, inner = x.shape
    kb = -(-inner // BLOCK)
    wide = torch.zeros(rows, kb * BLOCK, device=DEVICE)
    wide[:, :inner] = x
    wide = wide.view(rows, kb, BLOCK)
    m = wide.abs().amax(dim=2, keepdim=True).clamp(min=FLOOR)
    top = torch.full_like(m, TOP)
    return ((wide * (top / m)).to(torch.float8_e4m3fn).float() * (m / top)).view(rows, kb * BLOCK)[:, :inner]


def _weights(s):
    q = s["codes"]
    wide = s["scales"].repeat_interleave(BLOCK, 1).repeat_interleave(BLOCK, 2)
    return q.float() * wide[:, :q.shape[1], :q.shape[2]]


def _by_group(a, w, bounds):
    y = torch.zeros(a.shape[0], w.shape[1], device=DEVICE)
    for e in range(len(bounds) - 1):
        y[bounds[e]:bounds[e + 1]] = a[bounds[e]:bounds[e + 1]] @ w[e].t()
    return y


def _plain(s):
    op, dtype = s["op"], s["dtype"]
    if op == "sort":
        offsets, rows, slots = _order(s)
        return offsets, rows, slots, _sorted(s["x"], rows)
    if op == "sort_grad":
        return _gathered(s, s["dxs"], None, s["shape"][0]).to(dtype)
    if op == "unsort":
        return _gathered(s, s["z"], s["weights"], s["shape"][0]).to(dtype)
    if op == "unsort_grad":
        dz, dw = torch.zeros(s["z"].shape, dtype=dtype, device=DEVICE), torch.zeros_like(s["weights"])
        for token, entry, slot in _steps(s):
            dy = s["dy"][token].float()
            dz[slot] = (dy * s["weights"][entry][:, None]).to(dtype)
            dw[entry] = (dy * s["z"][slot].float()).sum(1)
        return dz, dw
    if op == "product":
        return (_blocks(s["x"]) @ _weights(s)[0].t()).to(dtype)
    if op == "experts":
        offsets, rows, slots = _order(s)
        return offsets, rows, slots, _by_group(_blocks(_sorted(s["x"], rows)), _weights(s), s["bounds"]).to(dtype)
    if op == "experts_grad":
        w, bounds = _weights(s), s["bounds"]
        dx = _by_group(_blocks(s["dy"]), w.transpose(1, 2), bounds).to(dtype)
        dw = torch.zeros(w.shape, device=DEVICE)
        for e in range(len(bounds) - 1):
            part = slice(bounds[e], bounds[e + 1])
            if part.start < part.stop:
                dw[e] = _blocks(s["dy"][part].t()) @ _blocks(s["xs"][part].t()).t()
        return dx, dw


# ---------------------------------------------------------------------------------- one pass ----

def run(s):
    if not own:
        return _plain(s)
    from nacho_b200 import nacho
    op, dtype = s["op"], s["dtype"]
    if op == "sort":
        order, xs = nacho.gpu_expert_sort(s["r"], s["x"])
        return order.offsets, order.rows, order.slots, xs
    if op == "sort_grad":
        return nacho.gpu_expert_sort_grad(s["order"], s["dxs"])
    if op == "unsort":
        return nacho.gpu_expert_unsort(s["r"], s["order"], s["z"])
    if op == "unsort_grad":
        return nacho.gpu_expert_unsort_grad(s["r"], s["order"], s["z"], s["dy"])
    if op == "product":
        return nacho.gpu_fp8_product(nacho.to_fp8_rows(s["x"]), s["w"], dtype=dtype)
    if op == "experts":
        order, xs = nacho.gpu_expert_sort_fp8(s["r"], s["x"])
        return order.offsets, order.rows, order.slots, nacho.gpu_fp8_product(xs, s["w"], order, dtype=dtype)
    if op == "experts_grad":
        return nacho.gpu_fp8_product_grad(s["dy"], s["xs"], s["w"], s["order"])


# ----------------------------------------------------------------------------- work and truth ----

def work(case):
    op, size = case["op"], {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
    if op == "product":
        m, n, k = case["rows"], case["n"], case["inner"]
        return {"bytes": size * (m * k + m * n) + n * k + 4 * -(-n // BLOCK) * -(-k // BLOCK), "flops": 2 * m * n * k}
    T, E = case["tokens"], case["experts"]
    n = sum(t % (case["k"] + 1) for t in range(T)) if case["ragged"] else T * case["k"]
    kept = n * (1.0 - case["drop"])
    if op == "sort":
        return {"bytes": int(4 * (T + 1) + 4 * n + size * T * case["width"] + size * n * case["width"] + 8 * n + 4 * (E + 1)), "flops": 0}
    if op == "sort_grad":
        return {"bytes": int(4 * (T + 1) + 4 * n + size * (kept + T) * case["width"]), "flops": int(kept * case["width"])}
    if op == "unsort":
        return {"bytes": int(4 * (T + 1) + 8 * n + size * (kept + T) * case["width"]), "flops": int(2 * kept * case["width"])}
    if op == "unsort_grad":
        return {"bytes": int(4 * (T + 1) + 12 * n + size * (kept + n + T) * case["width"]), "flops": int(3 * kept * case["width"])}
    k, m = case["inner"], case["n"]
    used = E * (1.0 - (1.0 - 1.0 / E) ** kept)  # experts that have rows at all
    weights = used * (m * k + 4 * -(-m // BLOCK) * -(-k // BLOCK))
    if op == "experts":
        return {"bytes": int(4 * (T + 1) + 12 * n + size * T * k + weights + size * n * m), "flops": int(2 * kept * m * k)}
    return {"bytes": int(size * kept * (m + k) + weights + size * n * k + 4 * E * m * k), "flops": int(4 * kept * m * k)}


def _e4m3(v):
    """The nearest e4m3 numbers (ties to even; |v| <= 448), by their definition: 3 bits behind the leading one, none below 2^-9."""
    power = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -20))).clamp(min=-6.0)
    power = torch.where(v.abs() >= torch.exp2(power + 1), power + 1, power)  # where log2 rounded down across a power of two
    step = torch.exp2(power - 3)
    return torch.clamp(torch.round(v / step) * step, -TOP, TOP)


def _stored(x, dim):
    """x in 64 bits as its 8-bit blocks along ``dim`` stand for it. The two factors of a block are 32-bit numbers by definition."""
    x = x.movedim(dim, -1).float()
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for b in range(0, x.shape[-1], BLOCK):
        part = x[..., b:b + BLOCK]
        m = part.abs().max(dim=-1, keepdim=True).values.double().clamp(min=FLOOR)
        out[..., b:b + BLOCK] = _e4m3((part * (TOP / m).float()).double()) * (m / TOP).float().double()
    return out.movedim(-1, dim)


def _tile_values(s):
    w = s["codes"].double()
    for a in range(s["scales"].shape[1]):
        for b in range(s["scales"].shape[2]):
            w[:, a * BLOCK:(a + 1) * BLOCK, b * BLOCK:(b + 1) * BLOCK] *= s["scales"][:, a, b, None, None].double()
    return w


def _host_order(s):
    """The order by counting on the host, entry by entry of every expert."""
    T, E = s["shape"]
    expert = s["experts"].cpu().numpy().astype(np.int64)
    token = np.repeat(np.arange(T), np.diff(s["offsets"].cpu().numpy()))
    slots, rows, offsets = np.full(len(expert), -1, np.int32), np.full(len(expert), -1, np.int32), np.zeros(E + 1, np.int32)
    at = 0
    for e in range(E):
        mine = np.flatnonzero(expert == e)
        slots[mine] = np.arange(at, at + len(mine))
        rows[at:at + len(mine)] = token[mine]
        at += len(mine)
        offsets[e + 1] = at
    put = lambda a: torch.from_numpy(a).to(DEVICE)
    return put(offsets), put(rows), put(slots), put(token)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "product":
        return _stored(s["x"], 1) @ _tile_values(s)[0].t()
    offsets, rows, slots, token = _host_order(s)
    T = s["shape"][0]
    kept = slots >= 0
    if op == "sort":
        xs = torch.zeros(rows.numel(), case["width"], dtype=torch.float64, device=DEVICE)
        xs[rows >= 0] = s["x"][rows[rows >= 0].long()].double()
        return offsets, rows, slots, xs
    at, to = slots[kept].long(), token[kept]
    if op in ("sort_grad", "unsort"):
        y = torch.zeros(T, case["width"], dtype=torch.float64, device=DEVICE)
        w = torch.ones(at.numel(), device=DEVICE) if op == "sort_grad" else s["weights"][kept]
        source = s["dxs"] if op == "sort_grad" else s["z"]
        for c in range(0, case["width"], 512):  # by columns, which bounds the memory
            y[:, c:c + 512].index_add_(0, to, source[:, c:c + 512][at].double() * w.double()[:, None])
        return y
    if op == "unsort_grad":
        dz, dw = torch.zeros(s["z"].shape, dtype=torch.float64, device=DEVICE), torch.zeros(kept.numel(), dtype=torch.float64, device=DEVICE)
        w, dots = s["weights"][kept].double(), torch.zeros(at.numel(), dtype=torch.float64, device=DEVICE)
        for c in range(0, case["width"], 512):
            dy = s["dy"][:, c:c + 512][to].double()
            dz[at, c:c + 512] = dy * w[:, None]
            dots += (dy * s["z"][:, c:c + 512][at].double()).sum(1)
        dw[kept] = dots
        return dz, dw
    bound, w = offsets.tolist(), _tile_values(s)
    if op == "experts":
        y = torch.zeros(rows.numel(), case["n"], dtype=torch.float64, device=DEVICE)
        x = _stored(s["x"], 1)
        for e in range(len(bound) - 1):
            y[bound[e]:bound[e + 1]] = x[rows[bound[e]:bound[e + 1]].long()] @ w[e].t()
        return offsets, rows, slots, y
    dx = torch.zeros(rows.numel(), case["inner"], dtype=torch.float64, device=DEVICE)
    dw = torch.zeros(w.shape, dtype=torch.float64, device=DEVICE)
    dy = _stored(s["dy"], 1)
    for e in range(len(bound) - 1):
        part = slice(bound[e], bound[e + 1])
        if part.start < part.stop:
            dx[part] = dy[part] @ w[e]
            dw[e] = _stored(s["dy"][part], 0).t() @ _stored(s["xs"][part], 0)
    return dx, dw
