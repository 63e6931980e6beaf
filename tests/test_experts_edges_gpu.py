"""GPU suite: the operators around a router where their extents end: no experts, no columns, as many entries as there can be, calls in
graphs, and every kernel that the dispatch can choose. Tolerances are those of test_experts_gpu.py."""
import numpy as np
import pytest
import torch

from test_experts_gpu import assert_order, nacho, near, normal, product_bound, routing

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("tokens,k,n", [(1, 1, 16), (30, 2, 130), (900, 4, 256)])
def test_no_experts(dtype, tokens, k, n):
    """A rank without experts of its own: every entry is dropped, products and gradients are zeros."""
    r, token, expert, _ = routing(tokens, 0, k, seed=1)
    x = normal((tokens, 200), dtype, 2)
    order, a = nacho().gpu_expert_sort_fp8(r, x)
    assert_order(order, token, expert, 0)
    w = nacho().to_fp8_tiles(torch.zeros(0, n, 200, device="cuda"))
    torch.full((tokens * k, n), 7.0, dtype=dtype, device="cuda")  # what the next result may find in its memory
    y = nacho().gpu_fp8_product(a, w, order, dtype=dtype)
    assert y.shape == (tokens * k, n) and y.dtype == dtype and not y.any()
    z = nacho().gpu_expert_unsort(r, order, y)
    assert z.shape == (tokens, n) and not z.any()
    dx, dw = nacho().gpu_fp8_product_grad(normal((tokens * k, n), dtype, 3), normal((tokens * k, 200), dtype, 4), w, order)
    assert dx.shape == (tokens * k, 200) and not dx.any() and dw.shape == (0, n, 200)


@pytest.mark.parametrize("tokens", [0, 7, 3000])
def test_no_columns(tokens):
    """Rows without columns still have an order, and nothing is summed over them."""
    r, token, expert, _ = routing(tokens, 6, 3, seed=tokens, ragged=True, drop=0.1)
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.zeros(tokens, 0, dtype=dtype, device="cuda")
        order, a = nacho().gpu_expert_sort_fp8(r, x)
        assert_order(order, token, expert, 6)
        assert tuple(a.shape.tolist()) == (1, len(expert), 0)
        assert_order(nacho().gpu_expert_sort(r, x)[0], token, expert, 6)
        y = nacho().gpu_fp8_product(a, nacho().to_fp8_tiles(torch.zeros(6, 40, 0, device="cuda")), order, dtype=dtype)
        assert y.shape == (len(expert), 40) and not y.any()
        dx, dw = nacho().gpu_fp8_product_grad(normal((len(expert), 40), dtype, 1), torch.zeros(len(expert), 0, dtype=dtype, device="cuda"),
                                              nacho().to_fp8_tiles(torch.zeros(6, 40, 0, device="cuda")), order)
        assert dx.shape == (len(expert), 0) and dw.shape == (6, 40, 0)
        dx, dw = nacho().gpu_fp8_product_grad(torch.zeros(len(expert), 0, dtype=dtype, device="cuda"), normal((len(expert), 40), dtype, 1),
                                              nacho().to_fp8_tiles(torch.zeros(6, 0, 40, device="cuda")), order)
        assert dx.shape == (len(expert), 40) and not dx.any() and dw.shape == (6, 0, 40)


@pytest.mark.parametrize("shape", [(3, 0, 128), (2, 0, 1), (3, 5, 0), (0, 0, 0), (4, 0, 0)])
def test_tiles_of_groups_without_elements(shape):
    w = nacho().to_fp8_tiles(torch.zeros(shape, device="cuda"))
    assert tuple(w.shape.tolist()) == shape and w.to_dense().shape == shape
    assert tuple(w.transposed().shape.tolist()) == (shape[0], shape[2], shape[1])
    wide = torch.zeros(shape[0], shape[1] + 3, shape[2] + 3, device="cuda")
    assert tuple(nacho().to_fp8_tiles(wide[:, 3:, 3:]).shape.tolist()) == shape


def test_graphs_outlive_larger_calls_and_one_another():
    """Two graphs captured on one stream, a larger call there afterwards, and both replayed at once on two other streams: each one's order is its own."""
    cases = [routing(3000, 64, 4, seed=1), routing(2500, 300, 7, seed=2, ragged=True, drop=0.1)]
    tokens = [normal((len(c[0].dim_j_offsets) - 1, 96), torch.bfloat16, 3) for c in cases]
    stream, graphs, held = torch.cuda.Stream(), [], []
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for (r, *_), x in zip(cases, tokens):
            nacho().gpu_expert_sort(r, x)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                held.append(nacho().gpu_expert_sort(r, x))
            graphs.append(graph)
        nacho().gpu_expert_order(routing(200000, 300, 5, seed=3)[0])
    torch.cuda.synchronize()
    others = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for (order, xs), _ in zip(held, graphs):
            for t in (order.offsets, order.rows, order.slots, xs):
                t.zero_()
        torch.cuda.synchronize()
        for graph, other in zip(graphs, others):
            with torch.cuda.stream(other):
                graph.replay()
        torch.cuda.synchronize()
        for (r, token, expert, _), x, (order, xs) in zip(cases, tokens, held):
            assert_order(order, token, expert, int(r.shape[1]))
            rows = order.rows.long()
            assert torch.equal(xs, torch.where((rows >= 0)[:, None], x[rows.clamp(min=0)], torch.zeros((), dtype=x.dtype, device="cuda")))


def test_a_report_finds_its_word_after_a_release():
    """A product that gives up while the scratch pools are released still has a place to say so."""
    import ctypes as C
    from nacho_b200 import _capi
    n = nacho()
    a, w = n.to_fp8_rows(normal((300, 700), torch.float32, 1)), n.to_fp8_tiles(normal((200, 700), torch.float32, 2))
    want = n.gpu_fp8_product(a, w, dtype=torch.float32)
    y = torch.full((300, 200), 7.0, device="cuda")
    struct = lambda m: _capi.Fp8Struct(*m._dims, int(m.tiled), m._values.data_ptr(), m._scales.data_ptr())
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()  # without scratch of its own, for which a release would wait
    status = _capi.lib.nb200_selftest_product_timeout(C.byref(struct(a)), C.byref(struct(w)), C.byref(_capi.DenseStruct(300, 200, 200, 0, y.data_ptr())),
                                                      C.c_void_p(stream.cuda_stream))
    assert status == _capi.OK and _capi.lib.nb200_release_workspaces() == _capi.OK
    torch.cuda.synchronize()
    assert torch.all(y == 7.0)
    with torch.cuda.stream(stream):
        with pytest.raises(RuntimeError, match="earlier 8-bit product: matrix product pipeline gave up"):
            n.gpu_fp8_product(a, w)
        got = n.gpu_fp8_product(a, w, dtype=torch.float32)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("experts", [1280, 2560, 2561, 4096])
@pytest.mark.parametrize("tokens,k", [(2561, 1), (1025, 4), (8193, 1), (70001, 3)])
def test_many_experts(experts, tokens, k):
    """Tables of counts as large as the place where they lie."""
    r, token, expert, _ = routing(tokens, experts, k, seed=experts, drop=0.02)
    assert_order(nacho().gpu_expert_order(r), token, expert, experts)


@pytest.mark.parametrize("experts", range(1224, 1231))
def test_experts_whose_counters_take_48_kb(experts):
    """With a kernel's other shared memory that is more than it has without asking."""
    r, token, expert, _ = routing(3000, experts, 1, seed=experts)
    assert_order(nacho().gpu_expert_order(r), token, expert, experts)


def test_tiles_whose_entries_16_bits_do_not_count():
    """More than 2^15 entries a tile, all of them of one expert."""
    entries = (1 << 23) + 12345
    r = nacho().CSR_gpu(torch.arange(0, entries + 1, 5, dtype=torch.int32, device="cuda"), torch.ones(entries, dtype=torch.int32, device="cuda"),
                        torch.ones(entries, device="cuda"), (entries // 5, 3))
    entries = entries // 5 * 5
    order = nacho().gpu_expert_order(r)
    assert order.offsets.tolist() == [0, 0, entries, entries]
    assert torch.equal(order.slots[:entries], torch.arange(entries, dtype=torch.int32, device="cuda")) and torch.all(order.slots[entries:] == -1)
    assert torch.equal(order.rows[:entries], torch.arange(entries, dtype=torch.int32, device="cuda") // 5)


MOST = (1 << 31) - 1 - 1024  # tokens and entries that an order takes
CHUNK = 1 << 26


def filled(n, values):
    """n 32-bit numbers on the GPU, from a function of a chunk of their places (64-bit)."""
    out = torch.empty(n, dtype=torch.int32, device="cuda")
    for at in range(0, n, CHUNK):
        out[at:at + CHUNK] = values(torch.arange(at, min(at + CHUNK, n), device="cuda"))
    return out


@pytest.fixture
def room():
    """The memory of a large test goes back to the device."""
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("entries", [(1 << 31) - (1 << 22), MOST])
def test_as_many_entries_as_there_can_be(entries, room):
    """Entry e goes to expert e % 6, every sixth one is dropped, so its slot is known."""
    tokens = (1 << 20) + 77
    row_ptr = filled(tokens + 1, lambda t: t * entries // tokens)
    expert = filled(entries, lambda e: e % 6)
    weight = torch.ones(entries, device="cuda")
    weight[1::2] = 2
    r = nacho().CSR_gpu(row_ptr, expert, weight, (tokens, 5))
    order = nacho().gpu_expert_order(r)
    first = [0]
    for c in range(5):
        first.append(first[-1] + (entries - c + 5) // 6)
    assert order.offsets.tolist() == first
    base = torch.tensor(first, device="cuda")
    for at in range(0, entries, CHUNK):
        e = torch.arange(at, min(at + CHUNK, entries), device="cuda")
        want = torch.where(e % 6 < 5, base[e % 6] + e // 6, -1)
        assert torch.equal(order.slots[at:at + CHUNK], want.int())
        kept = want >= 0
        token = torch.searchsorted(row_ptr, e[kept].int(), right=True) - 1
        assert torch.equal(order.rows[want[kept]], token.int())
    assert torch.all(order.rows[first[-1]:] == -1)
    z, dy = torch.ones(entries, 1, dtype=torch.bfloat16, device="cuda"), torch.full((tokens, 1), 3.0, dtype=torch.bfloat16, device="cuda")
    y = nacho().gpu_expert_sort_grad(order, z)
    some = [0, 1, tokens // 2, tokens - 1]
    want = [sum(e % 6 < 5 for e in range(t * entries // tokens, (t + 1) * entries // tokens)) for t in some]
    assert torch.equal(y[some].flatten(), torch.tensor(want, device="cuda").to(torch.bfloat16))
    dz, dw = nacho().gpu_expert_unsort_grad(r, order, z, dy)
    for at in range(0, entries, CHUNK):
        e = torch.arange(at, min(at + CHUNK, entries), device="cuda")
        assert torch.equal(dw[at:at + CHUNK], torch.where(e % 6 < 5, 3.0, 0.0))
        kept = e[e % 6 < 5]
        assert torch.equal(dz[base[kept % 6] + kept // 6, 0], (3.0 * weight[kept]).to(torch.bfloat16))
    assert not dz[first[-1]:].any()


def test_offsets_that_fall_stand_for_more_blocks_than_32_bits_count(room):
    """Every other group has all rows: the first one's gradient is whole, the next one gets what blocks are left, the others none."""
    rows, groups = 140_000_000, 4096
    zigzag = torch.arange(groups + 1, device="cuda", dtype=torch.int32) % 2 * rows
    nobody = torch.zeros(rows, dtype=torch.int32, device="cuda")
    order = nacho().ExpertOrder_gpu(zigzag, nobody, nobody, torch.zeros(1, dtype=torch.int32, device="cuda"), (0, groups))
    ones = torch.ones(rows, 1, dtype=torch.bfloat16, device="cuda")
    dx, dw = nacho().gpu_fp8_product_grad(ones, ones, nacho().to_fp8_tiles(torch.ones(groups, 1, 1, device="cuda")), order)
    assert dx.shape == (rows, 1)
    want = torch.zeros(groups, device="cuda")
    want[0], want[2] = rows, groups * 128  # there is room for a block per group more than the rows have
    # every block stands for 128 within two roundings of its scales; a million of them are added in 32 bits
    assert torch.all((dw.flatten() - want).abs() <= want * (2 ** -22 + rows / 128 * 2 ** -24))
    assert not dw[1].any() and not dw[3:].any()


def test_as_many_tokens_as_there_can_be(room):
    """A thousand entries over the rows of all numbers of tokens that 32 bits count."""
    row_ptr = filled(MOST + 1, lambda t: t * 1000 // MOST)
    expert = torch.arange(1000, dtype=torch.int32, device="cuda") % 7
    r = nacho().CSR_gpu(row_ptr, expert, torch.ones(1000, device="cuda"), (MOST, 7))
    order = nacho().gpu_expert_order(r)
    token = torch.searchsorted(row_ptr, torch.arange(1000, dtype=torch.int32, device="cuda"), right=True) - 1
    assert_order(order, token.cpu().numpy(), expert.cpu().numpy(), 7)
    y = nacho().gpu_expert_sort_grad(order, torch.ones(1000, 1, dtype=torch.bfloat16, device="cuda"))
    assert y.shape == (MOST, 1) and torch.equal(torch.nonzero(y.view(torch.int16).flatten()).flatten(), token)


def test_extents_that_leave_no_room_to_count():
    """The last 1024 numbers in front of 2^31 are refused before anything runs."""
    one = torch.zeros(2, dtype=torch.int32, device="cuda")
    import ctypes as C
    from nacho_b200 import _capi
    for tokens, entries in ((MOST + 1, 0), (0, MOST + 1), (1, (1 << 31) - 1)):
        r = _capi.CsrStruct(tokens, 3, entries, one.data_ptr(), one.data_ptr(), None)
        order = _capi.ExpertOrderStruct(0, 0, 0, None, one.data_ptr(), one.data_ptr(), one.data_ptr())
        assert _capi.lib.nb200_expert_sort(C.byref(r), None, C.byref(order), None, None) == _capi.E_UNSUPPORTED
