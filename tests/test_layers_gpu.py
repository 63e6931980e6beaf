"""GPU suite: gated layers, products in 8-bit integers and clipped gradients against plain implementations in 64 bits, at the sizes, strides and masks where they
can go wrong. Tolerances follow from the roundings: u of a type is half its spacing at 1, a 32-bit sum of n terms on the tensor cores (which cut off) is off by at
most n * 2^-23 of the sum of the terms' magnitudes, an activation by 2^-18 of its value (two approximations of a few steps each), results are rounded once."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # where numbers have no more digits
HALVES = [torch.bfloat16, torch.float16]
ACT = 2.0 ** -18


def nacho():
    from nacho_b200 import nacho as n
    return n


def normal(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def strided(t, pad, offset):
    """The same values in rows `pad` elements further apart, `offset` elements into their storage, with NaNs around them."""
    rows, cols = t.shape
    store = torch.full((offset + rows * (cols + pad),), float("nan"), dtype=t.dtype, device=t.device)
    view = store[offset:].view(rows, cols + pad)[:, :cols]
    view.copy_(t)
    return view


def order_of(counts, lead=0, tail=0):
    """An order whose experts have so many rows each, `lead` rows in front of the first (which no sort makes, and the products allow) and `tail` behind the last."""
    n = nacho()
    rows = lead + sum(counts) + tail
    at = [lead]
    for c in counts:
        at.append(at[-1] + c)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    return n.ExpertOrder_gpu(ints(at), torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda"), ints([0, rows]), (1, len(counts))), at


def act64(g, name):
    """act(g) and its derivative."""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * torch.sigmoid(-g))
    p, slope = 1.5957691216057308 * (g + 0.044715 * g ** 3), 1.5957691216057308 * (1 + 3 * 0.044715 * g * g)
    s = torch.sigmoid(p)
    return g * s, s + g * s * torch.sigmoid(-p) * slope


def close(got, want, tol, what):
    assert got.shape == want.shape, what
    # what lies beyond the type's numbers is rounded to an infinity (eight float16 terms of 3e4 sum to 2.4e5, and 65504 is the largest)
    most = torch.finfo(got.dtype).max
    beyond = (want.abs() - tol > most * (1 + U[got.dtype])) & (got.double() == want.sign() * math.inf)
    off = torch.where(beyond, 0.0, (got.double() - want).abs())
    bad = ~(off <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}, worst {float((off / tol).nan_to_num(posinf=1e9).max()):.3g} of the tolerance"


def gated64(x, w, bounds, act, dtype):
    """h, both and their tolerances."""
    hidden, rows = w.shape[1] // 2, x.shape[0]
    both, size = (torch.zeros(rows, 2 * hidden, dtype=torch.float64, device="cuda") for _ in range(2))
    for e in range(len(bounds) - 1):
        part = slice(bounds[e], bounds[e + 1])
        both[part] = x[part].double() @ w[e].double().t()
        size[part] = x[part].double().abs() @ w[e].double().abs().t()
    off = (x.shape[1] + 1) * 2.0 ** -23 * size
    g, u = both[:, :hidden], both[:, hidden:]
    a, _ = act64(g, act)
    # |act'| is at most 1.13
    off_h = 1.2 * off[:, :hidden] * (u.abs() + off[:, hidden:]) + (a.abs() + off[:, :hidden]) * off[:, hidden:] + ACT * (a * u).abs()
    h = a * u
    return h, off_h + U[dtype] * (h.abs() + off_h) + TINY[dtype], both, off + U[dtype] * (both.abs() + off) + TINY[dtype]


def check_gated(x, w, order, bounds, act, dtype, keep=True):
    three = w if w.dim() == 3 else w[None]
    h, tol_h, both, tol_both = gated64(x, three, bounds, act, dtype)
    got = nacho().gpu_gated_product(x, w, order, activation=act, keep=keep)
    if keep:
        close(got[1], both, tol_both, "both")
        got = got[0]
    assert got.dtype == dtype
    close(got, h, tol_h, "h")


# (rows, hidden, width): single tokens, few rows, the first of the tiles, ragged ones, sums of nothing but a tail
DENSE = [(1, 16, 64), (1, 1, 1), (1, 1500, 1100), (7, 33, 77), (8, 100, 129), (9, 64, 128), (32, 257, 1000), (33, 1, 8), (33, 128, 64), (64, 130, 72), (65, 127, 63), (129, 64, 65), (200, 300, 520),
         (257, 513, 1024), (300, 136, 2048), (1000, 1101, 1100)]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rows,hidden,width", DENSE)
def test_gated(rows, hidden, width, dtype, act):
    x, w = normal((rows, width), dtype, 1), normal((2 * hidden, width), dtype, 2, 1.5 * width ** -0.5)
    check_gated(x, w, None, [0, rows], act, dtype)
    check_gated(x, w, None, [0, rows], act, dtype, keep=False)


# sums so long, of so few tiles, that pairs of CTAs share them by two or by four: along the width, along the hidden units, along the rows
LONG = [(64, 130, 2100), (200, 64, 1100), (40, 1100, 64), (300, 600, 200), (2500, 40, 72), (1100, 64, 136), (2055, 33, 65)]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rows,hidden,width", LONG)
def test_gated_long_sums(rows, hidden, width, dtype):
    x, w = normal((rows, width), dtype, 1), normal((2 * hidden, width), dtype, 2, width ** -0.5)
    check_gated(x, w, None, [0, rows], "gelu", dtype)
    check_grad(normal((rows, hidden), dtype, 5), normal((rows, 2 * hidden), dtype, 6, 2.0), x, w, None, [0, rows], "gelu", dtype)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("counts,hidden,width", [([40, 0, 33], 96, 2100), ([70, 1, 5], 1100, 40), ([2100, 0, 1500, 33], 40, 72)])
def test_gated_long_sums_by_expert(counts, hidden, width, dtype):
    order, bounds = order_of(counts, 2, 5)
    rows = 7 + sum(counts)
    x, w = normal((rows, width), dtype, 3), normal((len(counts), 2 * hidden, width), dtype, 4, width ** -0.5)
    dh, both = normal((rows, hidden), dtype, 5), normal((rows, 2 * hidden), dtype, 6, 2.0)
    for t in (x, dh, both):
        t[:2], t[bounds[-1]:] = float("nan"), float("nan")
    check_gated(x, w, order, bounds, "silu", dtype)
    check_grad(dh, both, x, w, order, bounds, "silu", dtype)


COUNTS = [([0, 3, 0, 1, 9, 0], 0, 0), ([17, 0, 33, 2], 0, 5), ([100, 0, 1, 257, 64, 63], 0, 3), ([0, 0], 0, 40), ([300], 3, 0), ([40, 500, 0], 2, 7), ([1] * 70, 0, 0), ([65] * 40, 1, 1)]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("hidden,width", [(72, 64), (201, 131)])
@pytest.mark.parametrize("counts,lead,tail", COUNTS)
def test_gated_by_expert(counts, lead, tail, hidden, width, dtype):
    order, bounds = order_of(counts, lead, tail)
    x, w = normal((lead + sum(counts) + tail, width), dtype, 3), normal((len(counts), 2 * hidden, width), dtype, 4, 1.5 * width ** -0.5)
    x[:lead], x[bounds[-1]:] = float("nan"), float("nan")
    check_gated(x, w, order, bounds, "silu", dtype)


def grad64(dh, both, x, w, bounds, act, dtype):
    hidden = w.shape[1] // 2
    g, u, d = both[:, :hidden].double(), both[:, hidden:].double(), dh.double()
    a, slope = act64(g, act)
    dboth = torch.cat([d * u * slope, d * a], dim=1)
    # the derivative's parts may cancel: their magnitudes count
    parts = torch.cat([(d * u).abs() * (slope.abs() + 1.2), (d * a).abs()], dim=1)
    off = ACT * parts + U[dtype] * dboth.abs() * (1 + ACT) + TINY[dtype]
    dx, tol_x = (torch.zeros(x.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    dw, tol_w = (torch.zeros(w.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    for e in range(len(bounds) - 1):
        p = slice(bounds[e], bounds[e + 1])
        if p.start == p.stop:
            continue
        m = off[p] + (2 * hidden + 1) * 2.0 ** -23 * (dboth[p].abs() + off[p])
        dx[p], tol_x[p] = dboth[p] @ w[e].double(), m @ w[e].double().abs()
        m = off[p] + (p.stop - p.start + 1) * 2.0 ** -23 * (dboth[p].abs() + off[p])
        dw[e], tol_w[e] = dboth[p].t() @ x[p].double(), m.t() @ x[p].double().abs()
    rounded = lambda v, t: t + U[dtype] * (v.abs() + t) + TINY[dtype]
    return dx, rounded(dx, tol_x), dw, rounded(dw, tol_w)


def check_grad(dh, both, x, w, order, bounds, act, dtype):
    three = w if w.dim() == 3 else w[None]
    dx, tol_x, dw, tol_w = grad64(dh, both, x, three, bounds, act, dtype)
    got_x, got_w = nacho().gpu_gated_product_grad(dh, both, x, w, order, activation=act)
    assert got_x.dtype == got_w.dtype == dtype and got_w.shape == w.shape
    close(got_x, dx, tol_x, "dx")
    close(got_w.view(dw.shape), dw, tol_w, "dw")


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rows,hidden,width", DENSE)
def test_gated_gradients(rows, hidden, width, dtype, act):
    x, w = normal((rows, width), dtype, 1), normal((2 * hidden, width), dtype, 2, width ** -0.5)
    check_grad(normal((rows, hidden), dtype, 5), normal((rows, 2 * hidden), dtype, 6, 2.0), x, w, None, [0, rows], act, dtype)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("hidden,width", [(72, 64), (201, 131)])
@pytest.mark.parametrize("counts,lead,tail", COUNTS)
def test_gated_gradients_by_expert(counts, lead, tail, hidden, width, dtype):
    """Rows of other experts and of nobody hold NaNs where they must not matter."""
    order, bounds = order_of(counts, lead, tail)
    rows = lead + sum(counts) + tail
    x, w = normal((rows, width), dtype, 3), normal((len(counts), 2 * hidden, width), dtype, 4, width ** -0.5)
    dh, both = normal((rows, hidden), dtype, 5), normal((rows, 2 * hidden), dtype, 6, 2.0)
    for t in (x, dh, both):
        t[:lead], t[bounds[-1]:] = float("nan"), float("nan")
    check_grad(dh, both, x, w, order, bounds, "silu", dtype)


def test_experts_do_not_reach_one_another():
    """An infinity in one expert's row, its weights or its gradient stays there, although the blocks of neighbouring experts overlap."""
    n, dtype = nacho(), torch.bfloat16
    order, bounds = order_of([70, 50, 90])
    x, w, dh, both = normal((210, 96), dtype, 1), normal((3, 160, 96), dtype, 2, 0.1), normal((210, 80), dtype, 3), normal((210, 160), dtype, 4)
    want = n.gpu_gated_product(x, w, order), *n.gpu_gated_product_grad(dh, both, x, w, order)
    x[75], w[1], dh[80], both[90] = float("inf"), float("nan"), float("-inf"), float("nan")
    got = n.gpu_gated_product(x, w, order), *n.gpu_gated_product_grad(dh, both, x, w, order)
    others = torch.ones(210, dtype=torch.bool, device="cuda")
    others[70:120] = False
    for a, b in zip(got[:2], want[:2]):
        assert torch.equal(a[others], b[others]) and bool(torch.isfinite(a[others]).all())
    assert torch.equal(got[2][::2], want[2][::2]) and not bool(torch.isfinite(got[2][1]).all())


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rows", [3, 150])
@pytest.mark.parametrize("pad,offset", [(8, 0), (8, 8), (2, 0), (1, 3), (24, 1)])
def test_gated_strides(rows, pad, offset, dtype):
    hidden, width = 88, 136
    x, w = normal((rows, width), dtype, 1), normal((2 * hidden, width), dtype, 2, width ** -0.5)
    dh, both = normal((rows, hidden), dtype, 3), normal((rows, 2 * hidden), dtype, 4)
    s = lambda t: strided(t, pad, offset)
    check_gated(s(x), s(w), None, [0, rows], "silu", dtype)
    check_grad(s(dh), s(both), s(x), s(w), None, [0, rows], "silu", dtype)
    same = s(x[:1]).expand(rows, width)  # one row for all
    check_gated(same, w, None, [0, rows], "silu", dtype)
    check_grad(dh, both, same, w, None, [0, rows], "silu", dtype)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated_far_values(act, dtype):
    """Gates far on both sides of zero, where the logistic function has run out of digits: the results are what 64 bits round to."""
    g = torch.tensor([0.0, -0.0, 1e-3, -1e-3, 4.0, -4.0, 20.0, -20.0, 60.0, -60.0, 85.0, -85.0, 200.0, -200.0, 3e4, -3e4], device="cuda").to(dtype)
    x = torch.zeros(16, 64, dtype=dtype, device="cuda")
    x[:, 0], x[:, 1] = g, 1.0
    w = torch.zeros(2 * 8, 64, dtype=dtype, device="cuda")
    w[:8, 0], w[8:, 1] = 1.0, 2.0
    for copies in (1, 4):  # few rows, tiles
        xs = x.repeat(copies, 1)
        check_gated(xs, w, None, [0, 16 * copies], act, dtype)
        both = torch.cat([g[:, None].expand(16, 8), torch.full((16, 8), 2.0, dtype=dtype, device="cuda")], dim=1).repeat(copies, 1)
        check_grad(torch.ones(16 * copies, 8, dtype=dtype, device="cuda"), both, xs, w, None, [0, 16 * copies], act, dtype)


def test_gated_gradients_by_differences():
    """The gradients against differences of the forward pass in 64 bits."""
    dtype, rows, hidden, width = torch.float16, 40, 24, 32
    x, w, c = normal((rows, width), dtype, 1), normal((2 * hidden, width), dtype, 2, 0.3), normal((rows, hidden), dtype, 3)
    _, both = nacho().gpu_gated_product(x, w, keep=True)
    dx, dw = nacho().gpu_gated_product_grad(c, both, x, w)

    def loss(x, w):
        p = x @ w.t()
        return (act64(p[:, :hidden], "silu")[0] * p[:, hidden:] * c.double()).sum()

    step = 2.0 ** -12
    for t, grad, at in ((x, dx, [(0, 0), (7, 31), (39, 5)]), (w, dw, [(0, 0), (23, 7), (24, 9), (47, 31)])):
        for i in at:
            up, down = t.double().clone(), t.double().clone()
            up[i] += step
            down[i] -= step
            slope = float(loss(up, w.double()) - loss(down, w.double()) if t is x else loss(x.double(), up) - loss(x.double(), down)) / (2 * step)
            # both and the gradient of both are rounded to 2^-11 and so is the result; up to 64 terms of size 4 that may cancel
            assert abs(float(grad[i]) - slope) <= 2.0 ** -11 * (abs(slope) + 3 * 64)


# ---- 8-bit integers -----------------------------------------------------------------------------


def codes64(x):
    """Codes and scales by their definition; the factors and the product that is rounded are 32-bit numbers."""
    m = x.float().abs().amax(dim=-1, keepdim=True).clamp(min=2.0 ** -110)
    return torch.round(x.float() * (127.0 / m.double()).float()).double(), (m.double() / 127).float().squeeze(-1)


@pytest.mark.parametrize("dtype", [torch.float32, *HALVES])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (5, 32), (17, 33), (9, 1000), (2, 1024), (3, 1025), (2, 4100), (3, 8195), (1, 20001), (300, 257)])
def test_int8_rows(rows, cols, dtype):
    x = normal((rows, cols), dtype, rows + cols)
    x[0, cols // 2] *= 100
    q, scale = codes64(x)
    for given in (x, strided(x, 3, 1), strided(x, 16, 0)):
        z = nacho().to_int8_rows(given)
        assert z.shape.tolist() == [1, rows, cols]
        assert torch.equal(z.scales, scale)
        assert torch.equal(z.to_dense(), (q.float() * scale[:, None]))


def test_int8_rows_at_the_edges():
    x = torch.zeros(6, 200, device="cuda")
    x[1, 3], x[2, 0], x[3, 199], x[4, 7] = 1e-38, float("inf"), float("nan"), 3.4e38
    x[5] = torch.arange(200, device="cuda") / 2 - 50  # ties
    z = nacho().to_int8_rows(x)
    q, scale = codes64(x[[0, 1, 4, 5]])
    assert torch.equal(z.scales[[0, 1, 4, 5]], scale) and torch.equal(z.to_dense()[[0, 1, 4, 5]], q.float() * scale[:, None])
    assert bool(torch.isnan(z.to_dense()[2:4]).all())
    y = nacho().gpu_int8_product(z, nacho().to_int8_rows(torch.ones(40, 200, device="cuda")), dtype=torch.float32)
    assert bool(torch.isnan(y[2:4]).all()) and bool(torch.isfinite(y[[0, 1, 4, 5]]).all())
    assert nacho().to_int8_rows(torch.zeros(0, 5, device="cuda")).to_dense().shape == (0, 5)
    assert nacho().to_int8_rows(torch.zeros(5, 0, device="cuda")).to_dense().shape == (5, 0)


def check_int8(a, w, order, bounds, dtype, codes_a, scales_a, codes_w, scales_w):
    want = torch.zeros(codes_a.shape[0], codes_w.shape[1], dtype=torch.float64, device="cuda")
    for e in range(len(bounds) - 1):
        p = slice(bounds[e], bounds[e + 1])
        want[p] = (codes_a[p] @ codes_w[e].t()) * scales_a[p, None].double() * scales_w[e].double()
    got = nacho().gpu_int8_product(a, w, order, dtype=dtype)
    assert got.dtype == dtype
    # the sum is whole and rounded to 32 bits, so are its products with both scales, then the result
    close(got, want, 3 * 2.0 ** -24 * 1.01 * want.abs() + U[dtype] * want.abs() * 1.01 + TINY[dtype], "y")


@pytest.mark.parametrize("dtype", [torch.float32, *HALVES])
@pytest.mark.parametrize("rows,n,inner", [(1, 1, 1), (1, 17, 4096), (7, 100, 33), (8, 16, 64), (13, 129, 300), (32, 40, 1000), (33, 40, 1000), (33, 8, 7), (64, 256, 128), (100, 300, 129),
                                          (257, 513, 640), (700, 1500, 1100), (50, 300, 4100), (130, 200, 2100)])
def test_int8_product(rows, n, inner, dtype):
    x, w = normal((rows, inner), torch.float32, 1), normal((n, inner), torch.float32, 2, 0.05)
    (qa, sa), (qw, sw) = codes64(x), codes64(w)
    check_int8(nacho().to_int8_rows(x), nacho().to_int8_rows(w), None, [0, rows], dtype, qa, sa, qw[None], sw[None])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,inner", [(72, 64), (201, 131)])
@pytest.mark.parametrize("counts,lead,tail", COUNTS)
def test_int8_by_expert(counts, lead, tail, n, inner, dtype):
    order, bounds = order_of(counts, lead, tail)
    x, w = normal((lead + sum(counts) + tail, inner), torch.bfloat16, 3), normal((len(counts), n, inner), torch.bfloat16, 4)
    x[:lead], x[bounds[-1]:] = float("nan"), float("nan")
    (qa, sa), (qw, sw) = codes64(x), codes64(w)
    check_int8(nacho().to_int8_rows(x), nacho().to_int8_rows(w), order, bounds, dtype, qa.nan_to_num(), sa, qw, sw)


@pytest.mark.parametrize("rows", [2, 40])
def test_int8_sums_that_fill_32_bits(rows):
    """Codes of a caller's, -128 among them, at the largest width: the sums need all 32 bits."""
    inner = 131071
    codes = torch.full((rows, inner), -128, dtype=torch.int8, device="cuda")
    ones = torch.ones(rows, device="cuda")
    a = nacho().to_int8_rows(codes, ones)
    y = nacho().gpu_int8_product(a, a, dtype=torch.float32)
    assert bool((y == float(torch.tensor(128.0 * 128 * inner))).all())
    with pytest.raises(RuntimeError):
        b = nacho().to_int8_rows(torch.zeros(1, inner + 1, dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"))
        nacho().gpu_int8_product(b, b)


# ---- the norm of gradients ------------------------------------------------------------------------


def clip64(tensors, limit):
    norm = math.sqrt(sum(float((t.double() ** 2).sum()) for t in tensors))
    return norm, min(1.0, limit / (norm + 1e-6))


def check_clip(tensors, limit, out=None):
    kept = [t.clone() for t in tensors]
    norm, factor = clip64(kept, limit)
    got = nacho().gpu_clip_gradients(tensors, limit, out)
    assert got.shape == () and got.dtype == torch.float32
    # squares and up to 16 of their sums in 32 bits, the root's rounding
    assert abs(float(got) - norm) <= norm * 20 * 2.0 ** -24 + 2.0 ** -149
    for t, k, z in zip(tensors, kept, tensors if out is None else out):
        if out is not None and t.data_ptr() != z.data_ptr():
            assert torch.equal(t, k)
        want = k.double() * factor
        # the factor (the norm's error, a sum and a quotient), the product, the result's type
        slack = 0.0 if factor == 1.0 and z.dtype == t.dtype else (24 * 2.0 ** -24 if factor < 1 else 0.0) * 1.01 + U[z.dtype] * 1.01
        close(z, want, slack * want.abs() + (TINY[z.dtype] if slack else 0.0), "clipped")


SHAPES = [[(1,)], [(0,), (3, 5), (1, 1, 7)], [(1000, 1000), (33,), (4097,), (0, 4)], [(128, i + 1) for i in range(31)], [(9,)] * 33, [(64, 3)] * 600, [(2000, 2049), (5, 4), (300, 8), (1,)]]


@pytest.mark.parametrize("limit", [0.0, 0.5, 1e9, math.inf])
@pytest.mark.parametrize("shapes", SHAPES, ids=len)
@pytest.mark.parametrize("dtype", [torch.float32, *HALVES])
def test_clip(dtype, shapes, limit):
    check_clip([normal(s, dtype, i) for i, s in enumerate(shapes)], limit)


@pytest.mark.parametrize("limit", [0.5, 1e9])
def test_clip_into_other_tensors(limit):
    types = [torch.float32, *HALVES]
    tensors = [normal((50 + i, 40 + i % 3), types[i % 3], i) for i in range(40)]
    out = [torch.full(t.shape, float("nan"), dtype=types[i // 3 % 3], device="cuda") for i, t in enumerate(tensors)]
    out[0] = tensors[0]
    check_clip(tensors, limit, out)


def test_clip_alignment():
    """Views that begin anywhere, in a long buffer, and transposed ones; the elements around them stay."""
    for dtype in (torch.float32, *HALVES):
        buffer = normal((5000,), dtype, 1)
        kept = buffer.clone()
        views = [buffer[1:100], buffer[103:1500], buffer[1503:1600].view(97, 1), buffer[1600:2600].view(50, 20).t(), buffer[2608:4600]]
        norm, factor = clip64([v.clone() for v in views], 1.0)
        got = nacho().gpu_clip_gradients(views, 1.0)
        assert abs(float(got) - norm) <= norm * 20 * 2.0 ** -24
        want, tol = kept.double(), torch.zeros(5000, dtype=torch.float64, device="cuda")
        for a, b in ((1, 100), (103, 1500), (1503, 2600), (2608, 4600)):
            want[a:b] *= factor
            tol[a:b] = want[a:b].abs() * (24 * 2.0 ** -24 + U[dtype]) * 1.01 + TINY[dtype]
        close(buffer, want, tol, "buffer")


def test_clip_of_large_and_small_numbers():
    """Squares that 32 bits do not hold."""
    for scale in (1e30, 1e-30):
        check_clip([normal((300, 70), torch.float32, 1, scale), normal((77,), torch.bfloat16, 2, scale)], 0.1 * scale)
    zeros = [torch.zeros(100, 9, device="cuda"), torch.zeros(5, dtype=torch.float16, device="cuda")]
    check_clip(zeros, 1.0)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_clip_without_a_norm(bad):
    tensors = [normal((100, 10), torch.float32, 1), normal((70,), torch.bfloat16, 2)]
    tensors[1][3] = bad
    kept = [t.clone() for t in tensors]
    assert not math.isfinite(float(nacho().gpu_clip_gradients(tensors, 0.1)))
    out = [torch.zeros_like(t) for t in tensors]
    nacho().gpu_clip_gradients(tensors, 0.1, out)
    for t, k, z in zip(tensors, kept, out):
        assert torch.equal(t.nan_to_num(7.0), k.nan_to_num(7.0)) and torch.equal(z.nan_to_num(7.0), k.nan_to_num(7.0))


# ---- all of them ------------------------------------------------------------------------------------


def some_operands(rows=300, hidden=96, width=200, dtype=torch.bfloat16, seed=0):
    return (normal((rows, width), dtype, seed), normal((2 * hidden, width), dtype, seed + 1, width ** -0.5), normal((rows, hidden), dtype, seed + 2),
            normal((rows, 2 * hidden), dtype, seed + 3))


def all_calls(x, w, dh, both, order=None):
    """Every operator once, on the current stream; new tensors."""
    n = nacho()
    h, kept = n.gpu_gated_product(x, w, order, keep=True)
    dx, dw = n.gpu_gated_product_grad(dh, both, x, w, order, activation="gelu")
    few = n.gpu_gated_product(x[:5], w) if order is None else h
    y = n.gpu_int8_product(n.to_int8_rows(x), n.to_int8_rows(w), order, dtype=torch.float32)
    y1 = n.gpu_int8_product(n.to_int8_rows(x[:3]), n.to_int8_rows(w), dtype=torch.float16) if order is None else y
    out = [torch.empty_like(dx), torch.empty(dw.shape, device="cuda")]
    norm = n.gpu_clip_gradients([dx, dw], 0.5, out)
    return [h, kept, dx, dw, few, y, y1, norm, *out]


def equal(a, b):
    return all(torch.equal(p.nan_to_num(3.0), q.nan_to_num(3.0)) for p, q in zip(a, b))


def test_the_same_call_gives_the_same_bits():
    operands = some_operands()
    want = all_calls(*operands)
    for _ in range(5):
        assert equal(all_calls(*operands), want)


def test_streams_of_their_own():
    """Operands made on one stream, calls on two others at once, memory given back in between."""
    operands = some_operands(rows=700)
    want = all_calls(*operands)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for turn in range(6):
        s = streams[turn % 2]
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            copies = [t.clone() for t in operands]
            got.append(all_calls(*copies))
            del copies
    torch.cuda.synchronize()
    assert all(equal(g, want) for g in got)


def test_captured_calls():
    """Two graphs, replayed beside one another and after other calls, on operands that have changed since."""
    operands, others = some_operands(seed=0), some_operands(seed=10)
    order, _ = order_of([100, 0, 150, 33], tail=17)
    grouped = [normal((300, 200), torch.float16, 20), normal((4, 192, 200), torch.float16, 21, 0.1), normal((300, 96), torch.float16, 22), normal((300, 192), torch.float16, 23)]
    held = [t.clone() for t in operands]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        all_calls(*held)
        all_calls(*grouped, order)
    torch.cuda.synchronize()
    graphs, results = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    with torch.cuda.graph(graphs[0], stream=stream):
        results.append(all_calls(*held))
    with torch.cuda.graph(graphs[1], stream=stream):
        results.append(all_calls(*grouped, order))
    want_grouped = all_calls(*grouped, order)
    for given in (others, operands):
        for h, t in zip(held, given):
            h.copy_(t)
        want = all_calls(*given)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        assert equal(results[0], want) and equal(results[1], want_grouped)


def test_a_layer_forwards_backwards_clipped_and_served():
    """Tokens to their experts, the gated layer and its way down, back, gradients clipped, a step; then the layer served in integers. Against the same in 64 bits."""
    n, dtype = nacho(), torch.bfloat16
    tokens, experts, k, width, hidden = 200, 6, 2, 96, 80
    g = torch.Generator(device="cuda").manual_seed(5)
    expert = torch.topk(torch.rand(tokens, experts, generator=g, device="cuda"), k, dim=1).indices.flatten().int()
    expert[::17] = -1
    weight = torch.rand(tokens * k, generator=g, device="cuda")
    r = n.CSR_gpu(torch.arange(0, tokens * k + 1, k, dtype=torch.int32, device="cuda"), expert, weight, (tokens, experts))
    x, w, target = normal((tokens, width), dtype, 1), normal((experts, 2 * hidden, width), dtype, 2, width ** -0.5), normal((tokens, hidden), torch.float32, 3)
    order, xs = n.gpu_expert_sort(r, x)
    h, both = n.gpu_gated_product(xs, w, order, keep=True)
    y = n.gpu_expert_unsort(r, order, h)
    dz, dgate = n.gpu_expert_unsort_grad(r, order, h, (y.float() - target).to(dtype))
    dxs, dw = n.gpu_gated_product_grad(dz, both, xs, w, order)
    dx = n.gpu_expert_sort_grad(order, dxs)
    master = torch.empty(w.shape, device="cuda")
    norm = n.gpu_clip_gradients([dw], 0.25, [master])
    # in 64 bits, entry by entry
    want_y, keep = torch.zeros(tokens, hidden, dtype=torch.float64, device="cuda"), expert >= 0
    token, e = torch.arange(tokens * k, device="cuda")[keep] // k, expert[keep].long()
    p = torch.einsum("ij,ikj->ik", x[token].double(), w[e].double())
    a, slope = act64(p[:, :hidden], "silu")
    want_h = a * p[:, hidden:]
    want_y.index_add_(0, token, want_h * weight[keep].double()[:, None])
    dy = want_y - target.double()
    dh = dy[token] * weight[keep].double()[:, None]
    dp = torch.cat([dh * p[:, hidden:] * slope, dh * a], dim=1)
    want_dw = torch.zeros(w.shape, dtype=torch.float64, device="cuda").index_add_(0, e, torch.einsum("ik,ij->ikj", dp, x[token].double()))
    want_dx = torch.zeros(tokens, width, dtype=torch.float64, device="cuda").index_add_(0, token, torch.einsum("ik,ikj->ij", dp, w[e].double()))
    want_gate = torch.zeros(tokens * k, dtype=torch.float64, device="cuda")
    want_gate[keep] = (dy[token] * want_h).sum(1)
    # the chain rounds to 2^-8 at each of six steps; sums of some 100 terms: within 6 * 2^-8 of the largest in the root of the squares' mean
    for got, want in ((y, want_y), (dx, want_dx), (dw, want_dw), (dgate, want_gate)):
        assert float((got.double() - want).square().mean().sqrt()) <= 6 * 2.0 ** -8 * float(want.square().mean().sqrt())
    assert abs(float(norm) - float(dw.double().norm())) <= 1e-5 * float(norm)
    assert torch.allclose(master, dw.float() * min(1.0, 0.25 / (float(norm) + 1e-6)), rtol=1e-5, atol=1e-12)
    served = n.gpu_int8_product(n.to_int8_rows(xs), n.to_int8_rows(w), order, dtype=torch.float32)
    q, s = codes64(xs)
    qw, sw = codes64(w)
    for c in range(experts):
        lo, hi = order.offsets[c:c + 2].tolist()
        want = (q[lo:hi] @ qw[c].t()) * s[lo:hi, None].double() * sw[c].double()
        assert float((served[lo:hi].double() - want).abs().max() if hi > lo else 0) <= 4 * 2.0 ** -24 * float(want.abs().max() if hi > lo else 0)


@pytest.mark.parametrize("dtype", HALVES)
def test_extents_of_zero(dtype):
    n = nacho()
    z = lambda *s: torch.zeros(*s, dtype=dtype, device="cuda")
    ones = lambda *s: torch.ones(*s, dtype=dtype, device="cuda")
    order, _ = order_of([], tail=4)
    for rows, hidden, width in ((0, 8, 8), (4, 0, 8), (4, 8, 0), (0, 0, 0), (40, 8, 0), (40, 0, 8)):
        h, both = n.gpu_gated_product(ones(rows, width), ones(2 * hidden, width), keep=True)
        assert h.shape == (rows, hidden) and both.shape == (rows, 2 * hidden) and not bool(h.any()) and not bool(both.any())
        dx, dw = n.gpu_gated_product_grad(ones(rows, hidden), ones(rows, 2 * hidden), ones(rows, width), ones(2 * hidden, width))
        assert dx.shape == (rows, width) and dw.shape == (2 * hidden, width)
        if rows == 0 or hidden == 0:
            assert not bool(dx.any()) and not bool(dw.any())
        y = n.gpu_int8_product(n.to_int8_rows(ones(rows, width)), n.to_int8_rows(ones(hidden, width)), dtype=dtype)
        assert y.shape == (rows, hidden) and (width or not bool(y.any()))
    # no experts: rows of nobody
    h, both = n.gpu_gated_product(ones(4, 8), z(0, 12, 8), order, keep=True)
    assert h.shape == (4, 6) and not bool(h.any()) and not bool(both.any())
    dx, dw = n.gpu_gated_product_grad(ones(4, 6), ones(4, 12), ones(4, 8), z(0, 12, 8), order)
    assert dx.shape == (4, 8) and not bool(dx.any()) and dw.shape == (0, 12, 8)
    assert not bool(n.gpu_int8_product(n.to_int8_rows(ones(4, 8)), n.to_int8_rows(z(0, 5, 8)), order).any())


def test_offsets_that_fall_end_too():
    """Offsets that rise and fall again and again stand for more tiles than there are rows: the calls end, and no row is written outside its matrix."""
    n, dtype = nacho(), torch.bfloat16
    rows, groups = 3000, 300
    zigzag = torch.arange(groups + 1, device="cuda", dtype=torch.int32) % 2 * rows
    nobody = torch.zeros(rows, dtype=torch.int32, device="cuda")
    order = n.ExpertOrder_gpu(zigzag, nobody, nobody, torch.tensor([0, rows], dtype=torch.int32, device="cuda"), (1, groups))
    x, w = normal((rows, 64), dtype, 1), normal((groups, 64, 64), dtype, 2)
    n.gpu_gated_product(x, w, order, keep=True)
    n.gpu_gated_product_grad(normal((rows, 32), dtype, 3), normal((rows, 64), dtype, 4), x, w, order)
    n.gpu_int8_product(n.to_int8_rows(x), n.to_int8_rows(w), order)
    torch.cuda.synchronize()
    check_gated(x, w[0], None, [0, rows], "silu", dtype)


def test_rows_farther_than_32_bits_reach():
    """Rows two million elements apart, in storage of five gigabytes."""
    n, dtype, stride = nacho(), torch.bfloat16, 1 << 21
    store = torch.empty(1200 * stride, dtype=dtype, device="cuda")
    far = lambda t, at: store.view(-1, stride)[:, at:at + t.shape[1]].copy_(t)
    x, w, dh, both = some_operands(rows=1200, hidden=72, width=136)
    fx, fd, fb = far(x, 0), far(dh, 1024), far(both, 2048)
    assert equal(n.gpu_gated_product(fx, w, keep=True), n.gpu_gated_product(x, w, keep=True))
    assert equal(n.gpu_gated_product_grad(fd, fb, fx, w), n.gpu_gated_product_grad(dh, both, x, w))
    assert equal(n.gpu_gated_product_grad(fd, fb, far(x, 4097), w), n.gpu_gated_product_grad(dh, both, x, w))
    fw = far(normal((1200, 136), dtype, 9, 0.1), 8192)
    assert equal([n.gpu_gated_product(x[:3], fw)], [n.gpu_gated_product(x[:3], fw.contiguous())])
    assert equal([n.gpu_gated_product(x, fw)], [n.gpu_gated_product(x, fw.contiguous())])
    a, b = n.to_int8_rows(fx), n.to_int8_rows(x)
    assert torch.equal(a.scales, b.scales) and torch.equal(a.to_dense(), b.to_dense())


def test_a_wait_that_gives_up_is_reported():
    import ctypes as C
    from nacho_b200 import _capi
    n = nacho()
    x = normal((300, 700), torch.float32, 1)
    a, w = n.to_int8_rows(x), n.to_int8_rows(normal((200, 700), torch.float32, 2))
    want = n.gpu_int8_product(a, w, dtype=torch.float32)
    y = torch.full((300, 200), 7.0, device="cuda")
    struct = lambda m: _capi.Int8Struct(*m._dims, m._values.data_ptr(), m._scales.data_ptr())
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    for call in (lambda: n.gpu_int8_product(a, w), lambda: n.gpu_gated_product(x[:2].half(), x[:8].half()), lambda: n.gpu_gated_product(x.half(), x[:8].half())):
        status = _capi.lib.nb200_selftest_tiles_timeout(C.byref(struct(a)), C.byref(struct(w)), C.byref(_capi.DenseStruct(300, 200, 200, 0, y.data_ptr())), stream)
        assert status == _capi.OK
        torch.cuda.synchronize()
        assert torch.all(y == 7.0)
        with pytest.raises(RuntimeError, match="earlier gated or integer product: matrix product pipeline gave up"):
            call()
        assert torch.equal(n.gpu_int8_product(a, w, dtype=torch.float32), want)


def test_refusals():
    n = nacho()
    x, w, dh, both = some_operands()
    order, _ = order_of([100, 200])
    three = torch.stack([w, w])
    grad = lambda *a, **k: n.gpu_gated_product_grad(*a, **k)
    for error, call in [
            (TypeError, lambda: n.gpu_gated_product(x.float(), w.float())), (TypeError, lambda: n.gpu_gated_product(x, w.half())), (TypeError, lambda: n.gpu_gated_product(x.cpu(), w)),
            (TypeError, lambda: n.gpu_gated_product(x, w.t().contiguous().t())), (TypeError, lambda: n.gpu_gated_product(None, w)), (ValueError, lambda: n.gpu_gated_product(x, w[:-1])),
            (ValueError, lambda: n.gpu_gated_product(x[:, :-1], w)), (ValueError, lambda: n.gpu_gated_product(x, w, activation="relu")), (ValueError, lambda: n.gpu_gated_product(x, three)),
            (ValueError, lambda: n.gpu_gated_product(x, w, order)), (ValueError, lambda: n.gpu_gated_product(x[:-1], three, order)), (TypeError, lambda: n.gpu_gated_product(x, three, "order")),
            (TypeError, lambda: n.gpu_gated_product(x, torch.stack([w] * 4)[::2], order)), (TypeError, lambda: n.gpu_gated_product(x[0], w)),
            (ValueError, lambda: grad(dh[:-1], both, x, w)), (ValueError, lambda: grad(dh, both[:, :-2], x, w)), (ValueError, lambda: grad(dh[:, 1:], both, x, w)),
            (TypeError, lambda: grad(dh.half(), both, x, w)), (TypeError, lambda: grad(dh, both.float(), x, w)), (ValueError, lambda: grad(dh, both, x, w, activation="")),
            (TypeError, lambda: n.INT8_gpu(1)), (TypeError, lambda: n.to_int8_rows(x.cpu())), (TypeError, lambda: n.to_int8_rows(x.int())), (TypeError, lambda: n.to_int8_rows(x, x)),
            (TypeError, lambda: n.to_int8_rows(x.char().t(), torch.ones(200, device="cuda"))), (ValueError, lambda: n.to_int8_rows(x.char(), torch.ones(299, device="cuda"))),
            (ValueError, lambda: n.to_int8_rows(x.char(), torch.ones(300, device="cuda").half())), (ValueError, lambda: n.to_int8_rows(x.char(), torch.ones(300))),
            (ValueError, lambda: n.gpu_int8_product(n.to_int8_rows(x), n.to_int8_rows(w[:, 1:]))), (ValueError, lambda: n.gpu_int8_product(n.to_int8_rows(x), n.to_int8_rows(three))),
            (ValueError, lambda: n.gpu_int8_product(n.to_int8_rows(three), n.to_int8_rows(w))), (TypeError, lambda: n.gpu_int8_product(x, n.to_int8_rows(w))),
            (TypeError, lambda: n.gpu_int8_product(n.to_int8_rows(x), n.to_int8_rows(w), dtype=torch.float64)),
            (TypeError, lambda: n.gpu_clip_gradients(x, 1.0)), (ValueError, lambda: n.gpu_clip_gradients([], 1.0)), (ValueError, lambda: n.gpu_clip_gradients([x], -1.0)),
            (ValueError, lambda: n.gpu_clip_gradients([x], float("nan"))), (TypeError, lambda: n.gpu_clip_gradients([x.cpu()], 1.0)), (TypeError, lambda: n.gpu_clip_gradients([x.double()], 1.0)),
            (TypeError, lambda: n.gpu_clip_gradients([x, 1.0], 1.0)), (ValueError, lambda: n.gpu_clip_gradients([x[:, ::2]], 1.0)), (ValueError, lambda: n.gpu_clip_gradients([x, x], 1.0)),
            (ValueError, lambda: n.gpu_clip_gradients([x[:100], x[99:]], 1.0)), (ValueError, lambda: n.gpu_clip_gradients([x], 1.0, [])), (ValueError, lambda: n.gpu_clip_gradients([x], 1.0, [w])),
            (ValueError, lambda: n.gpu_clip_gradients([x, w], 1.0, [torch.empty_like(x)] * 2)), (ValueError, lambda: n.gpu_clip_gradients([x[:100], x[100:200]], 1.0, [x[100:200], x[200:]])),
            (ValueError, lambda: n.gpu_clip_gradients([x[:100]], 1.0, [x.view(torch.float16)[:100]])), (ValueError, lambda: n.gpu_clip_gradients([x[:200]], 1.0, [x[:200].t().contiguous().t()])),
            (TypeError, lambda: n.gpu_clip_gradients([x.to_sparse()], 1.0))]:
        kept = x.clone()
        with pytest.raises(error):
            call()
        assert torch.equal(x, kept)


def test_the_example_runs_with_the_layer_in_16_bits():
    from examples import routed_experts as example
    losses, dx = example.descend(tokens=130, experts=5, best=2, width=72, hidden=56, steps=2, halves=True, clip=0.5)
    assert len(losses) == 2 and all(math.isfinite(v) for v in losses) and dx.shape == (130, 72) and bool(torch.isfinite(dx).all())
    r, x = None, normal((40, 72), torch.bfloat16, 1)
    up, down = normal((1, 112, 72), torch.bfloat16, 2, 0.1), nacho().to_fp8_tiles(normal((1, 64, 56), torch.float32, 3, 0.1))
    r = nacho().CSR_gpu(torch.arange(41, dtype=torch.int32, device="cuda"), torch.zeros(40, dtype=torch.int32, device="cuda"), torch.ones(40, device="cuda"), (40, 1))
    y, kept = example.forward_halves(r, x, up, down)
    dx, dgate, dup, ddown = example.backward_halves(r, up, down, kept, normal((40, 64), torch.bfloat16, 4))
    # its gated half against the operator's own gradient, whose result it is
    order, xs, both, hidden, z = kept
    dz, _ = nacho().gpu_expert_unsort_grad(r, order, z, normal((40, 64), torch.bfloat16, 4))
    want = nacho().gpu_gated_product_grad(nacho().gpu_fp8_product_grad(dz, hidden, down, order)[0], both, xs, up, order)
    assert torch.equal(dup, want[1]) and torch.equal(dx, want[0])


def test_clipping_counts_as_a_change_in_place():
    t = torch.ones(10, device="cuda")
    version = t._version
    nacho().gpu_clip_gradients([t], 0.1)
    assert t._version > version
    with torch.inference_mode():
        frozen = torch.ones(10, device="cuda")
        assert abs(float(nacho().gpu_clip_gradients([frozen], 1e9)) - math.sqrt(10)) <= 1e-5
    with pytest.raises(RuntimeError):  # as any change in place of such a tensor out there
        nacho().gpu_clip_gradients([frozen], 0.1)
    assert bool((frozen == 1).all())


# rows that a tile's narrow side divides, with sums so long that pairs share them
@pytest.mark.parametrize("rows,hidden,width", [(64, 1024, 2048), (128, 512, 2100), (256, 640, 2048), (512, 256, 1100), (256, 72, 64)])
def test_whole_tiles_of_long_sums(rows, hidden, width):
    dtype = torch.bfloat16
    x, w = normal((rows, width), dtype, 1), normal((2 * hidden, width), dtype, 2, width ** -0.5)
    check_gated(x, w, None, [0, rows], "silu", dtype)
    check_grad(normal((rows, hidden), dtype, 5), normal((rows, 2 * hidden), dtype, 6, 2.0), x, w, None, [0, rows], "silu", dtype)
    order, bounds = order_of([rows // 2, 0, rows // 2])
    check_gated(x, torch.stack([w, w, w.flip(0)]), order, bounds, "silu", dtype)
    (qa, sa), (qw, sw) = codes64(x), codes64(w)
    check_int8(nacho().to_int8_rows(x), nacho().to_int8_rows(w), None, [0, rows], torch.float32, qa, sa, qw[None], sw[None])


@pytest.mark.parametrize("out", [False, True])
def test_a_refused_clip_changes_nothing(out):
    """The last tensor must not be written here: those in front do not count as changed."""
    with torch.inference_mode():
        frozen = torch.full((9,), 2.0, device="cuda")
    given = [normal((30, 7), torch.float32, 1), normal((11,), torch.float32, 2)]
    kept, versions = [t.clone() for t in given], [t._version for t in given]
    with pytest.raises(RuntimeError, match="inference"):
        if out:
            nacho().gpu_clip_gradients([torch.ones_like(t) for t in (*given, frozen)], 0.1, [*given, frozen])
        else:
            nacho().gpu_clip_gradients([*given, frozen], 0.1)
    assert [t._version for t in given] == versions and all(torch.equal(t, k) for t, k in zip(given, kept)) and bool((frozen == 2).all())


def test_a_norm_holds_nothing_else():
    """Norms that are kept for a log hold four bytes each, however many tensors there were."""
    for n in (1, 600):
        norm = nacho().gpu_clip_gradients([normal((5, 3), torch.float32, i) for i in range(n)], 1.0)
        assert norm.untyped_storage().nbytes() == 4 and norm.storage_offset() == 0


@pytest.mark.parametrize("shape", [(40, 200), (1, 33), (3, 5, 64)])
def test_scales_hold_no_codes(shape):
    for z in (nacho().to_int8_rows(normal(shape, torch.float32, 1)), nacho().to_int8_rows(torch.ones(shape, dtype=torch.int8, device="cuda"), torch.ones(shape[:-1], device="cuda"))):
        assert z.scales.untyped_storage().nbytes() == 4 * math.prod(shape[:-1]) and z.scales.storage_offset() == 0


# ---- many tiles, guards, launches beside one another ---------------------------------------------------

# more tiles for each pair of CTAs than it knows ahead, several times over
@pytest.mark.parametrize("rows,hidden,width", [(5000, 5120, 72), (4900, 5001, 65), (1200, 20000, 136)])
def test_many_tiles_of_gated_products(rows, hidden, width):
    dtype = torch.bfloat16
    check_gated(normal((rows, width), dtype, 1), normal((2 * hidden, width), dtype, 2, width ** -0.5), None, [0, rows], "gelu", dtype)


@pytest.mark.parametrize("rows,hidden,width", [(7000, 24, 7040), (7001, 21, 6999), (100, 3600, 7040), (77, 3601, 6999)])
def test_many_tiles_of_gradients(rows, hidden, width):
    """Of the rows' gradient, then of the weights'."""
    dtype = torch.float16
    x, w = normal((rows, width), dtype, 1), normal((2 * hidden, width), dtype, 2, hidden ** -0.5)
    check_grad(normal((rows, hidden), dtype, 5), normal((rows, 2 * hidden), dtype, 6, 2.0), x, w, None, [0, rows], "silu", dtype)


@pytest.mark.parametrize("rows,n,inner,dtype", [(7000, 7040, 100, torch.bfloat16), (6999, 7001, 33, torch.float16), (7000, 7040, 160, torch.float32)])
def test_many_tiles_of_integers(rows, n, inner, dtype):
    x, w = normal((rows, inner), torch.float32, 1), normal((n, inner), torch.float32, 2, 0.05)
    (qa, sa), (qw, sw) = codes64(x), codes64(w)
    check_int8(nacho().to_int8_rows(x), nacho().to_int8_rows(w), None, [0, rows], dtype, qa, sa, qw[None], sw[None])


@pytest.mark.parametrize("hidden,width", [(1320, 72), (1301, 67)])
def test_many_tiles_by_expert(hidden, width):
    dtype = torch.bfloat16
    counts = [(i * i * 37 + 11 * i) % 400 * (i % 5 > 0) for i in range(60)]
    order, bounds = order_of(counts, 0, 9)
    rows = sum(counts) + 9
    x, w = normal((rows, width), dtype, 3), normal((60, 2 * hidden, width), dtype, 4, width ** -0.5)
    dh, both = normal((rows, hidden), dtype, 5), normal((rows, 2 * hidden), dtype, 6, 2.0)
    for t in (x, dh, both):
        t[bounds[-1]:] = float("nan")
    check_gated(x, w, order, bounds, "silu", dtype)
    check_grad(dh, both, x, w, order, bounds, "silu", dtype)


def guarded(rows, cols, dtype, pad=0, fill=7.0):
    """A matrix within a larger array of one value: the array, the matrix, which elements are its own."""
    stride, lead = cols + pad, 512
    store = torch.full((lead + rows * stride + 512,), fill, dtype=dtype, device="cuda")
    view = store[lead:lead + rows * stride].view(rows, stride)[:, :cols]
    own = torch.zeros(store.shape, dtype=torch.bool, device="cuda")
    own[lead:lead + rows * stride].view(rows, stride)[:, :cols] = True
    return store, view, own


@pytest.mark.parametrize("rows,groups", [(3000, 300), (500, 300), (900, 7)])
@pytest.mark.parametrize("hidden,width,pad", [(32, 64, 16), (33, 65, 3)])
def test_nothing_is_written_around_results(rows, groups, hidden, width, pad):
    """Offsets that rise and fall, or lie outside the rows: what is written lies in the results' own elements all the same."""
    import ctypes as C
    from nacho_b200 import _capi
    dtype, n = torch.bfloat16, nacho()
    x, w = normal((rows, width), dtype, 1), normal((groups * 2 * hidden, width), dtype, 2)
    dh, kept = normal((rows, hidden), dtype, 3), normal((rows, 2 * hidden), dtype, 4)
    a, b = n.to_int8_rows(x), n.to_int8_rows(w.view(groups, 2 * hidden, width))
    struct = lambda t: C.byref(_capi.DenseStruct(t.shape[0], t.shape[1], t.stride(0), {torch.float32: 0, torch.bfloat16: 2}[t.dtype], t.data_ptr()))
    int8 = lambda m: C.byref(_capi.Int8Struct(*m._dims, m._values.data_ptr(), m._scales.data_ptr()))
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    room = lambda bytes_: torch.empty(max(1, bytes_), dtype=torch.uint8, device="cuda")
    lib, at = _capi.lib, torch.arange(groups + 1, device="cuda", dtype=torch.int32)
    even = (at * rows // groups).int()
    for offsets in (even, at % 2 * rows, even.flip(0).contiguous(), ((at * 7919) % (rows + 100) - 50).int()):
        results = {name: guarded(r, c, t, p) for name, r, c, t, p in (("h", rows, hidden, dtype, pad), ("both", rows, 2 * hidden, dtype, 0), ("dx", rows, width, dtype, pad),
                                                                        ("dw", groups * 2 * hidden, width, dtype, pad), ("y", rows, 2 * hidden, dtype, pad),
                                                                        ("y32", rows, 2 * hidden, torch.float32, pad))}
        r, o = {name: struct(v[1]) for name, v in results.items()}, C.c_void_p(offsets.data_ptr())
        need = lib.nb200_gated_product_scratch(struct(x), struct(w), groups)
        some = room(need)
        assert lib.nb200_gated_product(struct(x), struct(w), groups, o, 0, r["h"], r["both"], some.data_ptr(), need, stream) == _capi.OK
        need = lib.nb200_gated_product_grad_scratch(struct(x), struct(w), groups)
        more = room(need)
        assert lib.nb200_gated_product_grad(struct(dh), struct(kept), struct(x), struct(w), groups, o, 0, r["dx"], r["dw"], more.data_ptr(), need, stream) == _capi.OK
        assert lib.nb200_int8_product(int8(a), int8(b), o, r["y"], stream) == _capi.OK
        assert lib.nb200_int8_product(int8(a), int8(b), o, r["y32"], stream) == _capi.OK
        torch.cuda.synchronize()
        for name, (store, view, own) in results.items():
            assert bool((store[~own] == 7.0).all()), name
        if offsets is even:  # and all of it is written
            order = n.ExpertOrder_gpu(offsets, torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda"),
                                      torch.tensor([0, rows], dtype=torch.int32, device="cuda"), (1, groups))
            three = w.view(groups, 2 * hidden, width)
            want = dict(zip(("h", "both", "dx", "dw"), (*n.gpu_gated_product(x, three, order, keep=True), *n.gpu_gated_product_grad(dh, kept, x, three, order))))
            want["y"], want["y32"] = n.gpu_int8_product(a, b, order), n.gpu_int8_product(a, b, order, dtype=torch.float32)
            assert all(torch.equal(results[name][1], t.view(results[name][1].shape)) for name, t in want.items())


@pytest.mark.parametrize("rows,hidden,width,pad", [(300, 96, 200, 0), (1003, 301, 260, 1), (2048, 512, 1024, 0), (128, 1024, 2048, 3), (4000, 1100, 520, 5)])
def test_gradients_beside_one_another(rows, hidden, width, pad):
    """Calls that follow at once, on operands that change, in memory that the ones in front have given back: the bits of calls whose kernels run one by one."""
    from nacho_b200 import _capi
    n, dtype = nacho(), torch.bfloat16
    order, _ = order_of([rows // 3, 0, rows - rows // 3 - 5], tail=5)
    sets = []
    for i in range(4):
        x, w, dh, both = some_operands(rows, hidden, width, dtype, 10 * i)
        if pad:
            x, w, dh, both = (strided(t, pad, pad) for t in (x, w, dh, both))
        sets.append(((dh, both, x, w, None), (dh, both, x, torch.stack([w, w.flip(0), w]), order)))
    want = []
    _capi.lib.nb200_profile_enable(2)  # an event between any two kernels
    for pair in sets:
        for given in pair:
            want.append(n.gpu_gated_product_grad(*given))
            torch.cuda.synchronize()
    _capi.lib.nb200_profile_enable(0)
    off = torch.zeros((), dtype=torch.int64, device="cuda")
    for turn in range(25):
        k = (turn * 5 + turn // 8) % 8
        got = n.gpu_gated_product_grad(*sets[k // 2][k % 2])
        for g, t in zip(got, want[k]):
            off += (g != t).sum()
        del got
    assert int(off) == 0
