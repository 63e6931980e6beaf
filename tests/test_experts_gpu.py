"""GPU suite: the operators around a router against plain implementations in 64 bits, at the sizes, strides and masks where they can go
wrong. Tolerances follow from the roundings: u of a type is half its spacing at 1, a 32-bit sum of n terms is off by at most n * 2^-24 (where
the tensor cores cut off instead of rounding, n * 2^-23) of the sum of the terms' magnitudes, a result is rounded once to its type."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # where numbers have no more digits
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def nacho():
    from nacho_b200 import nacho as n
    return n


def routing(tokens, experts, k, seed=0, ragged=False, drop=0.0, lead=0, tail=0):
    """A CSR_gpu with entries in any order of experts, and (token, expert, weight) of all entries; `lead` and `tail` entries belong to no row."""
    rng = np.random.default_rng(seed)
    lengths = rng.integers(0, k + 1, tokens) if ragged else np.full(tokens, k)
    row_ptr = lead + np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
    n = int(row_ptr[-1]) + tail
    expert = rng.integers(0, max(experts, 1), n).astype(np.int32)
    expert[rng.random(n) < drop] = rng.choice([-1, experts, 1 << 30, -(1 << 31)])
    weight = rng.uniform(0.05, 1, n).astype(np.float32)
    token = np.full(n, -1)
    token[lead:n - tail] = np.repeat(np.arange(tokens), lengths)
    put = lambda a, t: torch.from_numpy(np.ascontiguousarray(a, t)).cuda()
    r = nacho().CSR_gpu(put(row_ptr, np.int32), put(expert, np.int32), put(weight, np.float32), (tokens, experts))
    return r, token, expert, weight


def plain_order(token, expert, experts):
    keep = (expert >= 0) & (expert < experts) & (token >= 0)
    n = len(expert)
    by = np.flatnonzero(keep)[np.argsort(expert[keep], kind="stable")]
    slots, rows = np.full(n, -1, np.int32), np.full(n, -1, np.int32)
    slots[by] = np.arange(len(by))
    rows[:len(by)] = token[by]
    offsets = np.concatenate([[0], np.cumsum(np.bincount(expert[by], minlength=max(experts, 1))[:experts])]).astype(np.int32)
    return offsets, rows, slots


def normal(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def assert_order(order, token, expert, experts):
    for got, want, what in zip((order.offsets, order.rows, order.slots), plain_order(token, expert, experts), ("offsets", "rows", "slots")):
        assert got.dtype == torch.int32 and np.array_equal(got.cpu().numpy(), want), what


def near(got, want, spread, roundings, what=""):
    """|got - want| <= u |want| (the last rounding) + roundings * 2^-23 * spread (the sum's)."""
    bound = U[got.dtype] * want.abs() + TINY[got.dtype] + roundings * 2.0 ** -23 * spread * (1 + U[got.dtype])
    off = (got.double() - want).abs()
    assert torch.all(off <= bound), f"{what}: {float((off - bound).max())} beyond the bound, {float(off.max())} off"


# ---- the order and the rows ------------------------------------------------------------

ROUTINGS = {
    "one": dict(tokens=1, experts=1, k=1), "no_tokens": dict(tokens=0, experts=5, k=2), "no_entries": dict(tokens=9, experts=5, k=0),
    "no_experts": dict(tokens=3, experts=0, k=2), "ragged": dict(tokens=777, experts=13, k=5, ragged=True),
    "dropped": dict(tokens=300, experts=8, k=3, drop=0.3), "all_dropped": dict(tokens=40, experts=8, k=3, drop=1.0),
    "one_expert": dict(tokens=500, experts=1, k=2), "most_experts": dict(tokens=700, experts=4096, k=8, ragged=True, drop=0.1),
    "part": dict(tokens=60, experts=7, k=4, ragged=True, drop=0.1, lead=37, tail=1030), "long_row": dict(tokens=2, experts=6, k=5000, drop=0.05),
    "tiles": dict(tokens=30011, experts=61, k=7, ragged=True, drop=0.02), "many_tiles": dict(tokens=200003, experts=300, k=6, ragged=True, drop=0.1, lead=5, tail=9),
    "edge_2559": dict(tokens=2559, experts=64, k=1), "edge_2560": dict(tokens=512, experts=300, k=5), "edge_2561": dict(tokens=2561, experts=64, k=1),
    "edge_8191": dict(tokens=8191, experts=64, k=1), "edge_8192": dict(tokens=1024, experts=64, k=8), "edge_8193": dict(tokens=8193, experts=64, k=1),
}


@pytest.mark.parametrize("name", ROUTINGS)
def test_order(name):
    case = ROUTINGS[name]
    r, token, expert, _ = routing(seed=len(name), **case)
    assert_order(nacho().gpu_expert_order(r), token, expert, case["experts"])
    x = normal((case["tokens"], 24), torch.bfloat16, 1)
    order, xs = nacho().gpu_expert_sort(r, x)
    assert_order(order, token, expert, case["experts"])
    rows = order.rows.long()
    want = torch.where((rows >= 0)[:, None], x[rows.clamp(min=0)] if len(x) else torch.zeros(len(rows), 24, dtype=x.dtype, device="cuda"), torch.zeros((), dtype=x.dtype, device="cuda"))
    assert torch.equal(xs, want)


def strided(x, how):
    """The same values at another place: rows apart, rows that start at an odd element, one row for all."""
    if how == "apart":
        wide = torch.zeros(len(x), x.shape[1] + 16, dtype=x.dtype, device=x.device)
        wide[:, 8:8 + x.shape[1]] = x
        return wide[:, 8:8 + x.shape[1]]
    if how == "odd":
        wide = torch.zeros(len(x), x.shape[1] + 5, dtype=x.dtype, device=x.device)
        wide[:, 1:1 + x.shape[1]] = x
        return wide[:, 1:1 + x.shape[1]]
    if how == "one":
        return x[:1].expand(len(x), -1)
    return x


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("width,how", [(1, "plain"), (7, "plain"), (64, "odd"), (128, "one"), (130, "apart"), (1001, "plain"), (2048, "apart"), (5000, "plain"), (0, "plain")])
def test_rows_there_and_back(dtype, width, how):
    r, token, expert, weight = routing(211, 9, 6, seed=width, ragged=True, drop=0.1)
    n = len(expert)
    x, dy = strided(normal((211, width), dtype, 2), how), strided(normal((211, width), dtype, 3), how)
    z = strided(normal((n, width), dtype, 4), how)
    order, xs = nacho().gpu_expert_sort(r, x)
    _, rows, slots = plain_order(token, expert, 9)
    rows, slots = torch.from_numpy(rows).cuda().long(), torch.from_numpy(slots).cuda().long()
    assert torch.equal(xs, torch.where((rows >= 0)[:, None], x[rows.clamp(min=0)], torch.zeros((), dtype=dtype, device="cuda")))
    kept = slots >= 0
    to, at = torch.from_numpy(token).cuda()[kept], slots[kept]
    w64, z64, dy64 = r.values.double()[kept][:, None], z.double(), dy.double()

    def summed(terms):
        return torch.zeros(211, width, dtype=torch.float64, device="cuda").index_add_(0, to, terms)

    # a sum of up to 6 terms: a rounding each where products are fused
    near(nacho().gpu_expert_unsort(r, order, z), summed(w64 * z64[at]), summed((w64 * z64[at]).abs()), 6, "unsort")
    near(nacho().gpu_expert_sort_grad(order, z), summed(z64[at]), summed(z64[at].abs()), 6, "sort_grad")
    dz, dw = nacho().gpu_expert_unsort_grad(r, order, z, dy)
    want = torch.zeros(n, width, dtype=torch.float64, device="cuda")
    want[at] = w64 * dy64[to]
    near(dz, want, want.abs(), 1, "dz")
    assert not dz[rows < 0].any()
    want, spread = torch.zeros(n, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda")
    want[kept], spread[kept] = (dy64[to] * z64[at]).sum(1), (dy64[to] * z64[at]).abs().sum(1)
    near(dw, want, spread, width, "dw")


def test_rows_of_nobody_are_not_read():
    """Slots behind the last expert's may hold anything: NaNs there, and in rows of other tokens, reach nobody."""
    r, token, expert, _ = routing(50, 4, 3, seed=5, drop=0.4)
    order = nacho().gpu_expert_order(r)
    z = normal((150, 40), torch.float32, 1)
    clean = nacho().gpu_expert_unsort(r, order, z)
    dirty = z.clone()
    dirty[order.rows < 0] = float("nan")
    assert torch.equal(nacho().gpu_expert_unsort(r, order, dirty), clean)
    dy = normal((50, 40), torch.float32, 2)
    dz, dw = nacho().gpu_expert_unsort_grad(r, order, dirty, dy)
    assert not torch.isnan(dz).any() and not torch.isnan(dw).any()
    bad = int(torch.nonzero(order.rows == 7)[0])
    dirty[bad] = float("inf")
    y = nacho().gpu_expert_unsort(r, order, dirty)
    others = torch.arange(50, device="cuda") != 7
    assert torch.equal(y[others], clean[others]) and torch.isinf(y[7]).all()


def test_gradients_against_differences():
    """Both directions are linear: differences of any length give the gradient. Steps are powers of two of whole numbers, so that the sums of 32 bits are exact."""
    r, token, expert, _ = routing(37, 5, 4, seed=8, ragged=True, drop=0.1)
    n = len(expert)
    whole = lambda shape, seed: torch.randint(-8, 9, shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").float()
    r = nacho().CSR_gpu(r.dim_j_offsets, r.dim_j_indices, whole((n,), 1), r.shape)
    order = nacho().gpu_expert_order(r)
    z, dy, x = whole((n, 33), 2), whole((37, 33), 3), whole((37, 33), 4)
    loss = lambda r, z: float((nacho().gpu_expert_unsort(r, order, z).double() * dy.double()).sum())
    dz, dw = nacho().gpu_expert_unsort_grad(r, order, z, dy)
    kept = order.rows >= 0
    step = whole((n, 33), 5) * kept[:, None]
    assert loss(r, z + step) - loss(r, z) == float((dz.double() * step.double()).sum())
    wstep = whole((n,), 6)
    moved = nacho().CSR_gpu(r.dim_j_offsets, r.dim_j_indices, r.values + wstep, r.shape)
    assert loss(moved, z) - loss(r, z) == float((dw.double() * wstep.double()).sum())
    dx = nacho().gpu_expert_sort_grad(order, z)
    xstep = whole((37, 33), 7)
    first, second = nacho().gpu_expert_sort(r, x)[1], nacho().gpu_expert_sort(r, x + xstep)[1]
    assert float(((second - first).double() * z.double()).sum()) == float((dx.double() * xstep.double()).sum())


# ---- 8-bit blocks ----------------------------------------------------------------------

def plain_factors(m):
    m = np.maximum(np.float32(m), np.float32(2.0 ** -110))
    return np.float32(m / np.float32(448)), np.float32(np.float32(448) / m)


def plain_blocks(x, rows_per_scale):
    """What x stands for, block by block, with the roundings to 8 bits of the CPU's conversion."""
    x = x.float().cpu().numpy()
    out = np.zeros_like(x)
    with np.errstate(all="ignore"):
        for r in range(0, x.shape[0], rows_per_scale):
            for c in range(0, x.shape[1], 128):
                part = x[r:r + rows_per_scale, c:c + 128]
                m = np.abs(part).max()
                scale, inverse = plain_factors(m) if not np.isnan(m) else (np.float32("nan"), np.float32("nan"))
                q = torch.from_numpy(part * inverse).to(torch.float8_e4m3fn).float().numpy()
                out[r:r + rows_per_scale, c:c + 128] = q * scale
    return torch.from_numpy(out).cuda()


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=7e30), torch.nan_to_num(b, nan=7e30)) and torch.equal(torch.isnan(a), torch.isnan(b))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols,how", [(1, 1, "plain"), (3, 128, "plain"), (5, 127, "plain"), (8, 129, "odd"), (130, 256, "apart"), (257, 1001, "plain"), (64, 640, "one"), (0, 128, "plain"), (4, 0, "plain")])
def test_quantised(dtype, rows, cols, how):
    x = strided(normal((rows, cols), dtype, rows + cols), how)
    a = nacho().to_fp8_rows(x)
    assert tuple(a.shape.tolist()) == (1, rows, cols) and not a.tiled
    assert same(a.to_dense(), plain_blocks(x, 1) if rows else x.float())
    w = nacho().to_fp8_tiles(x)
    assert w.tiled and same(w.to_dense()[0], plain_blocks(x, 128) if rows else x.float())
    if rows:
        assert same(w.transposed().to_dense()[0], w.to_dense()[0].t())


def test_blocks_with_extreme_values():
    x = torch.zeros(12, 200, device="cuda")
    x[1, 3], x[2, 5], x[3, 190] = float("nan"), float("inf"), float("-inf")
    x[4] = 3e38
    x[5] = 1e-45
    x[6, 0], x[6, 1] = 2.0 ** -111, -2.0 ** -118
    x[7, :3] = torch.tensor([448.0, 2.0 ** -9, 2.0 ** -10])
    x[8, :4] = torch.tensor([448.0, 17.0, 19.0, -25.0])  # halfway between two codes: to the even one
    x[9, 0], x[9, 1] = -3e38, 1.0
    x[10, :2] = torch.tensor([-0.0, 0.0])
    x[11] = torch.finfo(torch.float32).min
    a = nacho().to_fp8_rows(x).to_dense()
    assert same(a, plain_blocks(x, 1))
    assert torch.isnan(a[1, :128]).all() and not a[1, 128:].any() and torch.isnan(a[2, :128]).all() and torch.isnan(a[3, 128:]).all()
    assert a[8, :4].tolist() == [448.0, 16.0, 20.0, -24.0] and a[7, :3].tolist() == [448.0, 2.0 ** -9, 0.0]


@pytest.mark.parametrize("shape", [(1, 1, 1), (3, 130, 257), (2, 128, 128), (4, 20, 500), (1, 0, 128), (0, 5, 128)])
def test_tiles_of_groups_and_given_codes(shape):
    w = normal(shape, torch.float32, 3)
    t = nacho().to_fp8_tiles(w)
    dense = t.to_dense()
    assert dense.shape == shape
    for g in range(shape[0] if shape[1] else 0):
        assert same(dense[g], plain_blocks(w[g], 128))
    if w.numel():
        assert same(t.transposed().to_dense(), dense.transpose(1, 2)) and same(t.transposed().transposed().to_dense(), dense)
    codes = torch.randint(0, 256, shape, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda", dtype=torch.uint8)
    scales = torch.rand(shape[0], -(-shape[1] // 128), -(-shape[2] // 128), device="cuda") + 0.5
    wide = scales.repeat_interleave(128, 1).repeat_interleave(128, 2)[:, :shape[1], :shape[2]]
    want = codes.view(torch.float8_e4m3fn).float() * wide
    assert same(nacho().to_fp8_tiles(codes.view(torch.float8_e4m3fn), scales).to_dense(), want)
    if shape[0]:
        rows = torch.rand(shape[1], -(-shape[2] // 128), device="cuda") + 0.5
        want = codes[0].view(torch.float8_e4m3fn).float() * rows.repeat_interleave(128, 1)[:, :shape[2]]
        assert same(nacho().to_fp8_rows(codes[0].contiguous(), rows).to_dense(), want)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("width,how", [(1, "plain"), (200, "odd"), (1024, "apart"), (1001, "plain"), (4224, "plain")])
def test_sorted_and_quantised_in_one_pass(dtype, width, how):
    r, token, expert, _ = routing(301, 11, 4, seed=width, ragged=True, drop=0.1)
    x = strided(normal((301, width), dtype, 6), how)
    order, a = nacho().gpu_expert_sort_fp8(r, x)
    assert_order(order, token, expert, 11)
    _, xs = nacho().gpu_expert_sort(r, x)
    assert same(a.to_dense(), nacho().to_fp8_rows(xs).to_dense())


# ---- products --------------------------------------------------------------------------

def product_bound(inner):
    """Additions inside a block of 128 and of the blocks, two products of scales."""
    return min(inner, 128) + -(-inner // 128) + 2


@pytest.mark.parametrize("rows,n,inner", [(1, 1, 1), (1, 128, 128), (1, 4096, 2048), (2, 300, 1000), (3, 17, 4100), (16, 256, 128), (17, 255, 129), (33, 1000, 640), (64, 128, 7168),
                                          (65, 520, 96), (100, 100, 100), (127, 257, 384), (128, 256, 256), (129, 512, 1280), (300, 77, 333), (700, 1030, 520), (2049, 640, 1024),
                                          (0, 5, 128), (4, 0, 128), (4, 5, 0)])
def test_product(rows, n, inner):
    a, w = nacho().to_fp8_rows(normal((rows, inner), torch.float32, 1)), nacho().to_fp8_tiles(normal((n, inner), torch.float32, 2))
    da, dw = a.to_dense().double(), w.to_dense()[0].double()
    want, spread = da @ dw.t(), da.abs() @ dw.abs().t()
    for dtype in TYPES:
        y = nacho().gpu_fp8_product(a, w, dtype=dtype)
        assert y.shape == (rows, n) and y.dtype == dtype and y.is_contiguous()
        near(y, want, spread, product_bound(inner), str(dtype))


EXPERTS = [dict(tokens=1, experts=8, k=2), dict(tokens=16, experts=64, k=4), dict(tokens=64, experts=5, k=3, ragged=True, drop=0.2), dict(tokens=300, experts=7, k=2, drop=0.05),
           dict(tokens=1000, experts=3, k=1), dict(tokens=513, experts=40, k=8, ragged=True), dict(tokens=50, experts=6, k=3, drop=1.0), dict(tokens=0, experts=4, k=2),
           dict(tokens=2000, experts=2, k=2, drop=0.01, lead=3, tail=5), dict(tokens=90, experts=300, k=1)]


@pytest.mark.parametrize("case", range(len(EXPERTS)))
@pytest.mark.parametrize("n,inner", [(256, 512), (130, 200), (515, 1024), (8, 40)])
def test_product_by_expert(case, n, inner):
    case = EXPERTS[case]
    r, token, expert, _ = routing(seed=n + inner, **case)
    x, w = normal((case["tokens"], inner), torch.bfloat16, 3), nacho().to_fp8_tiles(normal((case["experts"], n, inner), torch.bfloat16, 4))
    order, a = nacho().gpu_expert_sort_fp8(r, x)
    da, dw = a.to_dense().double(), w.to_dense().double()
    offsets = order.offsets.tolist()
    want, spread = (torch.zeros(len(expert), n, dtype=torch.float64, device="cuda") for _ in range(2))
    for e in range(case["experts"]):
        part = slice(offsets[e], offsets[e + 1])
        want[part], spread[part] = da[part] @ dw[e].t(), da[part].abs() @ dw[e].abs().t()
    for dtype in (torch.float32, torch.bfloat16):
        y = nacho().gpu_fp8_product(a, w, order, dtype=dtype)
        near(y, want, spread, product_bound(inner), str(dtype))
        assert not y[offsets[-1]:].any()


@pytest.mark.parametrize("rows", [40, 700])
def test_nothing_leaks_between_rows_and_experts(rows):
    """NaNs in one expert's rows, in another's weights, in a column of weights: everything else is as without them."""
    expert = torch.arange(rows, device="cuda", dtype=torch.int32) * 7 // rows
    r = nacho().CSR_gpu(torch.arange(rows + 1, device="cuda", dtype=torch.int32), expert, torch.ones(rows, device="cuda"), (rows, 7))
    x, weights = normal((rows, 300), torch.float32, 1), normal((7, 200, 300), torch.float32, 2)
    order, a = nacho().gpu_expert_sort_fp8(r, x)
    clean = nacho().gpu_fp8_product(a, nacho().to_fp8_tiles(weights), order, dtype=torch.float32)
    assert not torch.isnan(clean).any()
    x[expert == 2] = float("nan")
    weights[4] = float("nan")
    weights[5, 190:, :] = float("inf")
    order, a = nacho().gpu_expert_sort_fp8(r, x)
    y = nacho().gpu_fp8_product(a, nacho().to_fp8_tiles(weights), order, dtype=torch.float32)
    bad = ((expert == 2) | (expert == 4))[:, None] | ((expert == 5)[:, None] & (torch.arange(200, device="cuda") >= 128)[None, :])
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], clean[~bad])


def column_blocks(x, offsets):
    """What x stands for with a scale per column and 128 rows of a group."""
    out = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    for e in range(len(offsets) - 1):
        if offsets[e] < offsets[e + 1]:
            out[offsets[e]:offsets[e + 1]] = plain_blocks(x[offsets[e]:offsets[e + 1]].t().contiguous(), 1).t().double()
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("case,n,inner", [(2, 130, 200), (3, 256, 384), (4, 64, 128), (5, 40, 136), (6, 8, 16), (7, 16, 24), (8, 515, 257), (0, 300, 129)])
def test_gradients_of_the_product(dtype, case, n, inner):
    case = EXPERTS[case]
    r, token, expert, _ = routing(seed=n, **case)
    order = nacho().gpu_expert_order(r)
    x, dy = strided(normal((len(expert), inner), dtype, 5), "apart"), strided(normal((len(expert), n), dtype, 6), "apart")
    w = nacho().to_fp8_tiles(normal((case["experts"], n, inner), torch.float32, 7))
    dx, dw = nacho().gpu_fp8_product_grad(dy, x, w, order)
    offsets = order.offsets.tolist()
    q, wide = nacho().to_fp8_rows(dy).to_dense().double(), w.to_dense().double()
    dcols, xcols = column_blocks(dy, offsets), column_blocks(x, offsets)
    want, spread = (torch.zeros(len(expert), inner, dtype=torch.float64, device="cuda") for _ in range(2))
    wantw, spreadw = torch.zeros_like(wide), torch.zeros_like(wide)
    for e in range(case["experts"]):
        part = slice(offsets[e], offsets[e + 1])
        want[part], spread[part] = q[part] @ wide[e], q[part].abs() @ wide[e].abs()
        wantw[e], spreadw[e] = dcols[part].t() @ xcols[part], dcols[part].abs().t() @ xcols[part].abs()
    assert dx.dtype == dtype and dw.dtype == torch.float32 and dw.shape == wide.shape
    near(dx, want, spread, product_bound(n), "dx")
    near(dw, wantw, spreadw, product_bound(max(max(np.diff(offsets)), 1)), "dw")
    if case["experts"] == 1:
        return
    dx1, dw1 = nacho().gpu_fp8_product_grad(dy[offsets[0]:offsets[1]], x[offsets[0]:offsets[1]], nacho().to_fp8_tiles(wide[0].float().contiguous()))
    assert torch.equal(dw1[0], dw[0]) and dx1.shape == (offsets[1], inner)


def test_gradients_of_the_product_against_differences():
    """With whole numbers up to 16 and a 448 in every block all codes and sums are exact, so the product is bilinear as it stands."""
    g = torch.Generator(device="cuda").manual_seed(1)
    whole = lambda *shape: torch.randint(-8, 9, shape, generator=g, device="cuda").float()
    r, token, expert, _ = routing(60, 3, 2, seed=1)
    order = nacho().gpu_expert_order(r)
    offsets = order.offsets.tolist()
    x, dy, w = whole(120, 128), whole(120, 128), whole(3, 128, 128)
    for t in (x, dy):  # a 448 in every row, and in every column of every expert's rows
        t[torch.arange(120), torch.arange(120)] = 448
        for e in range(3):
            t[offsets[e]] = 448
    w[:, 0, 0] = 448
    other = whole(3, 128, 128)
    other[:, 0, 0] = 448
    moved = x.clone()
    moved[:, 120:] = whole(120, 8)
    for e in range(3):
        moved[offsets[e]] = 448
    tiles = nacho().to_fp8_tiles
    loss = lambda x, w: float((nacho().gpu_fp8_product(nacho().to_fp8_rows(x), tiles(w), order, dtype=torch.float32).double() * dy.double()).sum())
    dx, dw = nacho().gpu_fp8_product_grad(dy, x, tiles(w), order)
    assert loss(x, other) - loss(x, w) == float((dw.double() * (other - w).double()).sum())
    assert loss(moved, w) - loss(x, w) == float((dx.double() * (moved - x).double()).sum())


# ---- how they are called ---------------------------------------------------------------

def test_refusals():
    n = nacho()
    r, _, _, _ = routing(10, 4, 2)
    x = normal((10, 32), torch.bfloat16, 1)
    order, xs = n.gpu_expert_sort(r, x)
    a, w = n.to_fp8_rows(xs), n.to_fp8_tiles(normal((4, 16, 32), torch.bfloat16, 2))
    for bad in (x.cpu(), x.to(torch.float64), x[0], None, x.t()):
        with pytest.raises(TypeError):
            n.gpu_expert_sort(r, bad)
        with pytest.raises(TypeError):
            n.to_fp8_rows(bad)
    for call in (lambda: n.gpu_expert_sort(r, x[:9]), lambda: n.gpu_expert_sort_fp8(r, x[:9]), lambda: n.gpu_expert_unsort(r, order, xs[:19]), lambda: n.gpu_expert_sort_grad(order, x),
                 lambda: n.gpu_expert_unsort_grad(r, order, xs, x[:, :31]), lambda: n.gpu_expert_unsort_grad(r, order, xs, x[:9]), lambda: n.gpu_fp8_product(a, w),
                 lambda: n.gpu_fp8_product(w, w, order), lambda: n.gpu_fp8_product(a, a), lambda: n.gpu_fp8_product(n.to_fp8_rows(x), w, order),
                 lambda: n.gpu_fp8_product(n.to_fp8_rows(xs[:, :31]), w, order), lambda: n.gpu_fp8_product(a, n.to_fp8_tiles(normal((3, 16, 32), torch.float32, 1)), order),
                 lambda: a.transposed(), lambda: n.to_fp8_tiles(torch.zeros(4, 4, dtype=torch.uint8, device="cuda"), torch.zeros(2, 1, device="cuda")),
                 lambda: n.gpu_fp8_product_grad(xs, xs, w, order), lambda: n.gpu_expert_unsort(routing(10, 4, 1)[0], order, xs)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: n.gpu_expert_sort(order, x), lambda: n.gpu_expert_unsort(order, r, xs), lambda: n.gpu_fp8_product(xs, w, order), lambda: n.gpu_fp8_product(a, w, r),
                 lambda: n.gpu_fp8_product(a, w, order, dtype=torch.int32), lambda: n.gpu_expert_unsort_grad(r, order, xs, x.float()), lambda: n.FP8_gpu(),
                 lambda: n.to_fp8_tiles(normal((4, 16, 32), torch.float32, 1)[:, :8]), lambda: n.to_fp8_rows(x, 1.0), lambda: n.gpu_fp8_product_grad(xs, xs, a, order)):
        with pytest.raises(TypeError):
            call()
    wide = n.CSR_gpu(r.dim_j_offsets, r.dim_j_indices, r.values, (10, 4097))
    with pytest.raises(RuntimeError, match="beyond the limit"):
        n.gpu_expert_order(wide)
    n.gpu_expert_sort(r, x)  # the context is as it was


def test_offsets_that_point_nowhere():
    """Row offsets that fall, or lie outside the entries, reach no memory outside the arrays."""
    entries = 40
    expert = (torch.arange(entries, device="cuda") % 5).to(torch.int32)
    for offsets in ([0, 20, 10, 40], [-100, 5, 1 << 30, 40], [40, 30, 20, -(1 << 31)]):
        r = nacho().CSR_gpu(torch.tensor(offsets, dtype=torch.int32, device="cuda"), expert, torch.ones(entries, device="cuda"), (3, 5))
        x = normal((3, 130), torch.float32, 1)
        order, xs = nacho().gpu_expert_sort(r, x)
        nacho().gpu_expert_unsort_grad(r, order, xs, x)
        w = nacho().to_fp8_tiles(normal((5, 40, 130), torch.float32, 2))
        order, a = nacho().gpu_expert_sort_fp8(r, x)
        nacho().gpu_fp8_product(a, w, order)
        torch.cuda.synchronize()
        wild = nacho().ExpertOrder_gpu(torch.tensor([-5, 70, 3, 1 << 30, 2, 1000], dtype=torch.int32, device="cuda"), torch.full((entries,), 1 << 30, dtype=torch.int32, device="cuda"),
                                       torch.full((entries,), 1 << 30, dtype=torch.int32, device="cuda"), r.dim_j_offsets, (3, 5))
        nacho().gpu_fp8_product(a, w, wild)
        nacho().gpu_fp8_product_grad(normal((entries, 40), torch.float32, 1), xs, w, wild)
        assert not nacho().gpu_expert_unsort(r, wild, xs).any()
        torch.cuda.synchronize()


def layer(r, x, w, dy):
    n = nacho()
    order, xs = n.gpu_expert_sort_fp8(r, x)
    z = n.gpu_fp8_product(xs, w, order)
    y = n.gpu_expert_unsort(r, order, z)
    dz, dg = n.gpu_expert_unsort_grad(r, order, z, dy)
    dxs, dw = n.gpu_fp8_product_grad(dz, n.gpu_expert_sort(r, x)[1], w, order)
    return y, dg, dw, n.gpu_expert_sort_grad(order, dxs)


@pytest.mark.parametrize("tokens", [20, 4000])
def test_streams_graphs_and_repeats(tokens):
    """The same bits from call to call, on another stream than the operands', and from a captured graph."""
    r, _, _, _ = routing(tokens, 16, 4, seed=2, drop=0.05)
    x, w, dy = normal((tokens, 512), torch.bfloat16, 1), nacho().to_fp8_tiles(normal((16, 384, 512), torch.bfloat16, 2)), normal((tokens, 384), torch.bfloat16, 3)
    want = layer(r, x, w, dy)
    equal = lambda got: all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(equal(layer(r, x, w, dy)) for _ in range(5))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer(r, x, w, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert equal(got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        layer(r, x, w, dy)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            held = layer(r, x, w, dy)
    for _ in range(3):
        for t in held:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert equal(held)


def test_more_elements_than_32_bits_count():
    tokens, width, k = 70001, 8192, 4
    r, token, expert, weight = routing(tokens, 30, k, seed=3)
    x = normal((tokens, width), torch.bfloat16, 1)
    order, xs = nacho().gpu_expert_sort(r, x)
    assert xs.numel() > 1 << 31
    _, rows, slots = plain_order(token, expert, 30)
    some = torch.tensor([0, 1, len(rows) // 2, len(rows) - 2, len(rows) - 1], device="cuda")
    assert torch.equal(xs[some], x[torch.from_numpy(rows).cuda().long()[some]])
    y = nacho().gpu_expert_unsort(r, order, xs)
    total = torch.from_numpy(weight.reshape(tokens, k)).cuda().double().sum(1)
    at = torch.tensor([0, 5, tokens // 2, tokens - 1], device="cuda")
    near(y[at], x[at].double() * total[at, None], x[at].double().abs() * total[at, None], k)
    dz, dw = nacho().gpu_expert_unsort_grad(r, order, xs, x)
    entry = torch.from_numpy(np.argsort(slots)).cuda()[some]
    near(dz[some], r.values[entry].double()[:, None] * xs[some].double(), xs[some].double().abs(), 1)
    near(dw[entry], (xs[some].double() ** 2).sum(1), (xs[some].double() ** 2).sum(1), width)
    del y, dz, dw, xs
    order, a = nacho().gpu_expert_sort_fp8(r, x)
    w = nacho().to_fp8_tiles(normal((30, 24, width), torch.bfloat16, 2))
    z = nacho().gpu_fp8_product(a, w, order, dtype=torch.float32)
    q = nacho().to_fp8_rows(x[torch.from_numpy(rows).cuda().long()[some]].contiguous()).to_dense().double()
    of = torch.bucketize(some.int(), order.offsets, right=True) - 1
    wide = w.to_dense().double()[of]
    near(z[some], torch.einsum("rk,rnk->rn", q, wide), torch.einsum("rk,rnk->rn", q.abs(), wide.abs()), product_bound(width))


def test_example_learns():
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "routed_experts.py")
    spec = importlib.util.spec_from_file_location("routed_experts", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, dx = example.descend(tokens=257, experts=6, best=2, width=130, hidden=200)
    assert all(b < a for a, b in zip(losses, losses[1:])) and dx.shape == (257, 130) and not torch.isnan(dx).any()


def test_a_wait_that_gives_up_is_reported_by_the_next_product():
    import ctypes as C
    from nacho_b200 import _capi
    n = nacho()
    a, w = n.to_fp8_rows(normal((300, 700), torch.float32, 1)), n.to_fp8_tiles(normal((200, 700), torch.float32, 2))
    want = n.gpu_fp8_product(a, w, dtype=torch.float32)
    y = torch.full((300, 200), 7.0, device="cuda")
    struct = lambda m: _capi.Fp8Struct(*m._dims, int(m.tiled), m._values.data_ptr(), m._scales.data_ptr())
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    status = _capi.lib.nb200_selftest_product_timeout(C.byref(struct(a)), C.byref(struct(w)), C.byref(_capi.DenseStruct(300, 200, 200, 0, y.data_ptr())), stream)
    assert status == _capi.OK
    torch.cuda.synchronize()
    assert torch.all(y == 7.0)
    with pytest.raises(RuntimeError, match="earlier 8-bit product: matrix product pipeline gave up"):
        n.gpu_fp8_product(a, w)
    assert torch.equal(n.gpu_fp8_product(a, w, dtype=torch.float32), want)


def test_offsets_that_fall_end():
    """Offsets that rise and fall again and again stand for more tiles than a matrix has: the product ends after as many as rising ones have."""
    n = nacho()
    rows, groups = 60000, 400
    zigzag = torch.arange(groups + 1, device="cuda", dtype=torch.int32) % 2 * rows
    nobody = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    order = n.ExpertOrder_gpu(zigzag, nobody, nobody, torch.zeros(1, dtype=torch.int32, device="cuda"), (0, groups))
    a, w = n.to_fp8_rows(normal((rows, 128), torch.bfloat16, 1)), n.to_fp8_tiles(normal((groups, 256, 128), torch.bfloat16, 2))
    start, stop = torch.cuda.Event(True), torch.cuda.Event(True)
    n.gpu_fp8_product(a, w, order)
    start.record()
    n.gpu_fp8_product(a, w, order)
    stop.record()
    torch.cuda.synchronize()
    assert start.elapsed_time(stop) < 20  # ms; all of its tiles would be 200 products of the matrix
