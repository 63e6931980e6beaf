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
