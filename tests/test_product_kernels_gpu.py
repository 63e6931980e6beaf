"""GPU suite: every kernel and launch shape that the 8-bit products choose between, against products in 64 bits of what the codes stand for. Which one a
shape takes follows from the rules at nb200_fp8_product for 148 SMs. Tolerances are those of test_experts_gpu.py; a cluster that shares a sum
adds up to eight parts more."""
import numpy as np
import pytest
import torch

from test_experts_gpu import TYPES, column_blocks, nacho, near, normal, product_bound, routing

pytestmark = pytest.mark.gpu

CLUSTER = 8


def with_offsets(offsets, rows):
    """An order of which only the offsets matter."""
    nobody = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    return nacho().ExpertOrder_gpu(torch.tensor(offsets, dtype=torch.int32, device="cuda"), nobody, nobody, torch.zeros(1, dtype=torch.int32, device="cuda"), (0, len(offsets) - 1))


def by_group(a, w, offsets):
    """Products in 64 bits and the sums of their terms' magnitudes; rows of no group are zeros."""
    da, dw = a.to_dense().double(), w.to_dense().double()
    want, spread = (torch.zeros(da.shape[0], dw.shape[1], dtype=torch.float64, device="cuda") for _ in range(2))
    for g in range(len(dw)):
        part = slice(offsets[g], offsets[g + 1])
        want[part], spread[part] = da[part] @ dw[g].t(), da[part].abs() @ dw[g].abs().t()
    return want, spread


def check(a, w, order, offsets, types=TYPES):
    inner = int(a.shape[2])
    want, spread = by_group(a, w, offsets)
    for dtype in types:
        y = nacho().gpu_fp8_product(a, w, order, dtype=dtype)
        near(y, want, spread, product_bound(inner) + CLUSTER, str(dtype))
        assert not y[:offsets[0]].any() and not y[offsets[-1]:].any()
        assert torch.equal(nacho().gpu_fp8_product(a, w, order, dtype=dtype), y)


ONE_GROUP = [
    (65, 200, 6200), (128, 1024, 8192), (100, 130, 6145),                 # 128 rows on the other side, shared by a cluster
    (129, 130, 6200), (300, 260, 6272), (1000, 129, 6145),                # the same in several turns, CTAs of their own
    (33, 300, 3000), (64, 4096, 3100), (50, 9344, 2950), (64, 1, 20000),  # 64 rows; as many tiles as the rule allows; the longest sums
    (64, 9472, 3000), (128, 9472, 6200),                                  # one tile more: the tiles' kernel
    (17, 40, 1025), (32, 18944, 300), (32, 20000, 130), (16, 300000, 60),  # 16 and 32 rows, shared, not shared, several tiles of columns each
]


@pytest.mark.parametrize("rows,n,inner", ONE_GROUP)
def test_few_rows_of_one_group(rows, n, inner):
    a, w = nacho().to_fp8_rows(normal((rows, inner), torch.float32, 1)), nacho().to_fp8_tiles(normal((n, inner), torch.float32, 2))
    check(a, w, None, [0, rows])


@pytest.mark.parametrize("inner", [100, 500, 2048, 4200])
@pytest.mark.parametrize("experts,rows,hot", [(40, 200, 180), (40, 700, 650), (7, 140, 140), (150, 150, 100), (300, 4000, 3000), (64, 64, 1)])
def test_a_hot_expert_takes_turns(experts, rows, hot, inner):
    """Most rows go to one expert: more than all turns of the launch together hold."""
    lengths = np.full(experts, 0)
    lengths[experts // 2] = hot
    for i in range(rows - hot):
        lengths[i * 7 % experts] += 1
    offsets = np.concatenate([[0], np.cumsum(lengths)]).tolist()
    a, w = nacho().to_fp8_rows(normal((rows, inner), torch.float32, 3)), nacho().to_fp8_tiles(normal((experts, 130, inner), torch.float32, 4))
    check(a, w, with_offsets(offsets, rows), offsets, [torch.float32, torch.bfloat16])


@pytest.mark.parametrize("experts,n,inner,each", [(300, 1100, 300, 2), (300, 1100, 300, 15), (1100, 1100, 128, 3), (600, 1030, 200, 8)])
def test_short_sums_take_several_tiles_of_columns(experts, n, inner, each):
    lengths = np.random.default_rng(experts).integers(0, 2 * each + 1, experts)
    offsets = np.concatenate([[0], np.cumsum(lengths)]).tolist()
    rows = offsets[-1] + 3
    a, w = nacho().to_fp8_rows(normal((rows, inner), torch.float32, 5)), nacho().to_fp8_tiles(normal((experts, n, inner), torch.bfloat16, 6))
    check(a, w, with_offsets(offsets, rows), offsets, [torch.float32, torch.bfloat16])


# results whose rows 16, 8, 4 and 2 bytes divide (with 16-bit types), and with a second tile of one column
@pytest.mark.parametrize("rows,n,inner", [(2000, 1304, 300), (2049, 1300, 260), (2050, 1302, 140), (2001, 1301, 1000), (1025, 2305, 128), (5000, 640, 520), (3000, 1280, 2048)])
def test_pairs_on_one_group(rows, n, inner):
    a, w = nacho().to_fp8_rows(normal((rows, inner), torch.float32, 7)), nacho().to_fp8_tiles(normal((n, inner), torch.float32, 8))
    check(a, w, None, [0, rows])


GROUPS = [
    [0, 1200, 2400, 2400, 3001, 3700, 6000], [5, 700, 1500, 2303, 4000], [13, 13, 1000, 3000], [0, 31, 63, 96, 2000, 2033, 4100],  # pairs
    [0, 40, 81, 150, 150, 260, 300], [3, 64, 130, 133, 390], [0, 1, 2, 130, 300], [129, 200, 329, 512],                                # single CTAs
    [2, 10, 22, 30], [9, 9, 20, 39, 44, 44], [1, 17], [7, 40],                                                                         # few rows
]


@pytest.mark.parametrize("n", [1304, 1301, 1302])
@pytest.mark.parametrize("case", range(len(GROUPS)))
def test_rows_in_front_of_and_behind_the_groups(case, n):
    offsets = GROUPS[case]
    rows = offsets[-1] + (0, 1, 5, 200)[case % 4]
    a, w = nacho().to_fp8_rows(normal((rows, 390), torch.float32, 9)), nacho().to_fp8_tiles(normal((len(offsets) - 1, n, 390), torch.float32, 10))
    check(a, w, with_offsets(offsets, rows), offsets)


@pytest.mark.parametrize("case", [dict(tokens=3000, experts=5, k=2, drop=0.05), dict(tokens=1000, experts=40, k=2), dict(tokens=4000, experts=16, k=4, ragged=True, drop=0.1)])
@pytest.mark.parametrize("n,inner", [(1304, 300), (643, 2100)])
def test_by_expert(case, n, inner):
    r, *_ = routing(seed=n, **case)
    x, w = normal((case["tokens"], inner), torch.bfloat16, 11), nacho().to_fp8_tiles(normal((case["experts"], n, inner), torch.bfloat16, 12))
    order, a = nacho().gpu_expert_sort_fp8(r, x)
    check(a, w, order, order.offsets.tolist())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,n,inner", [(1, 8, 16), (300, 200, 136), (1000, 520, 264), (2300, 129, 1301), (77, 1304, 130), (4099, 300, 300)])
def test_gradients_of_a_dense_product(dtype, rows, n, inner):
    dy, x = normal((rows, n), dtype, 13), normal((rows, inner), dtype, 14)
    w = nacho().to_fp8_tiles(normal((n, inner), torch.float32, 15))
    dx, dw = nacho().gpu_fp8_product_grad(dy, x, w)
    q, wide = nacho().to_fp8_rows(dy).to_dense().double(), w.to_dense().double()[0]
    assert dx.dtype == dtype and dw.shape == (1, n, inner)
    near(dx, q @ wide, q.abs() @ wide.abs(), product_bound(n) + CLUSTER, "dx")
    dcols, xcols = column_blocks(dy, [0, rows]), column_blocks(x, [0, rows])
    near(dw[0], dcols.t() @ xcols, dcols.abs().t() @ xcols.abs(), product_bound(rows), "dw")


@pytest.mark.parametrize("experts,rows", [(3, 2000), (20, 9000)])
def test_gradients_of_large_tiles(experts, rows):
    """Several tiles of every expert by pairs of CTAs, and more blocks than places for scales."""
    n, inner = 520, 777
    offsets = np.sort(np.random.default_rng(experts).integers(0, rows, experts + 1))
    offsets[0], offsets[-1] = 0, rows - 5
    dy, x, w = normal((rows, n), torch.bfloat16, 16), normal((rows, inner), torch.bfloat16, 17), nacho().to_fp8_tiles(normal((experts, n, inner), torch.float32, 18))
    offsets = offsets.tolist()
    dx, dw = nacho().gpu_fp8_product_grad(dy, x, w, with_offsets(offsets, rows))
    q, wide = nacho().to_fp8_rows(dy).to_dense().double(), w.to_dense().double()
    dcols, xcols = column_blocks(dy, offsets), column_blocks(x, offsets)
    assert not dx[offsets[-1]:].any()
    for e in range(experts):
        part = slice(offsets[e], offsets[e + 1])
        near(dx[part], q[part] @ wide[e], q[part].abs() @ wide[e].abs(), product_bound(n) + CLUSTER, "dx")
        near(dw[e], dcols[part].t() @ xcols[part], dcols[part].abs().t() @ xcols[part].abs(), product_bound(max(part.stop - part.start, 1)), "dw")


def test_offsets_that_fall_end_after_a_matrix_worth_of_tiles():
    """Every other group has all rows. The tiles of rising offsets, (rows / 256 + 2 groups) at most, are less than those of five such groups: nobody writes a later one's."""
    n = nacho()
    rows, groups = 60000, 401  # an odd number of them, so that the last offset is all rows and none is cleared
    order = with_offsets((np.arange(groups + 1) % 2 * rows).tolist(), rows)
    weights = torch.arange(1, groups + 1, device="cuda", dtype=torch.float32)[:, None, None].expand(groups, 200, 8).contiguous()
    a, w = n.to_fp8_rows(torch.ones(rows, 8, device="cuda")), n.to_fp8_tiles(weights)
    y = n.gpu_fp8_product(a, w, order, dtype=torch.float32)
    of_group = torch.round(y / 8).int() - 1
    assert int(of_group.max()) <= 8 and int(of_group.min()) >= 0 and not torch.any(of_group % 2)
