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
                                          (257, 513, 640), (700, 1500, 1100)])
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
