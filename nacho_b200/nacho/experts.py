"""Operators around a router. A router's decision is a ``CSR_gpu`` of tokens x experts whose values are the gate weights:
rows may be empty, entries may stand in any order of experts, and an entry whose column lies outside the
matrix (-1, say) is dropped. The tokens' rows are brought into the order of the experts, multiplied with every expert's
weights in 8-bit floating point, and brought back:

    order, xs = gpu_expert_sort_fp8(r, x)              # or gpu_expert_sort, which does not quantise
    z = gpu_fp8_product(xs, w, order)                  # w = to_fp8_tiles(weights), (experts, n, inner)
    y = gpu_expert_unsort(r, order, z)

Dense operands are 2-D CUDA tensors of float32, float16 or bfloat16 with contiguous rows at any distance; results are new
contiguous tensors without an autograd graph: gradients are calls of their own. No call waits for the device, and all of them can be captured in graphs, products once one
has been called on the stream. Sums are 32-bit in a fixed order and rounded once.
"""
from __future__ import annotations

import torch

from .nacho_ext import CSR_gpu, _dev_array, _dims, _host_shape, _native, _shape_array

__all__ = ["ExpertOrder_gpu", "FP8_gpu", "to_fp8_rows", "to_fp8_tiles", "gpu_expert_order", "gpu_expert_sort", "gpu_expert_sort_fp8", "gpu_expert_sort_grad",
           "gpu_expert_unsort", "gpu_expert_unsort_grad", "gpu_fp8_product", "gpu_fp8_product_grad"]

BLOCK = 128
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


class ExpertOrder_gpu:
    """Entries of a routing sorted by expert, those of one expert in storage order. Expert ``c`` has the slots ``offsets[c]`` to
    ``offsets[c + 1] - 1``; ``rows`` is the token of every slot (-1 for the slots behind the last expert's, as many as entries were
    dropped), ``slots`` the slot of every entry (-1 for a dropped one), ``token_offsets`` the routing's row offsets."""

    __slots__ = ("_offsets", "_rows", "_slots", "_token_offsets", "_shape", "_dims")

    def __init__(self, offsets, rows, slots, token_offsets, shape):
        self._offsets = _dev_array(offsets, torch.int32, "offsets")
        self._rows = _dev_array(rows, torch.int32, "rows")
        self._slots = _dev_array(slots, torch.int32, "slots")
        self._token_offsets = _dev_array(token_offsets, torch.int32, "token_offsets")
        self._shape = _shape_array(shape, 2)
        self._dims = _dims(self._shape)
        if self._rows.numel() != self._slots.numel():
            raise ValueError("rows and slots differ in length")
        if self._token_offsets.numel() != self._dims[0] + 1 or self._offsets.numel() != self._dims[1] + 1:
            raise ValueError("token_offsets and offsets must hold tokens + 1 and experts + 1 entries")
        if not (self._offsets.device == self._rows.device == self._slots.device == self._token_offsets.device):
            raise ValueError("all buffers of an order must live on one device")

    offsets = property(lambda self: self._offsets)
    rows = property(lambda self: self._rows)
    slots = property(lambda self: self._slots)
    token_offsets = property(lambda self: self._token_offsets)
    shape = property(_host_shape)

    @property
    def device(self):
        return self._slots.device

    def __repr__(self):
        return f"ExpertOrder_gpu(shape={self._dims}, entries={self._slots.numel()})"


class FP8_gpu:
    """Matrices in 8-bit floating point (e4m3), made by ``to_fp8_rows`` (a 32-bit scale for every 128 columns of a row) or ``to_fp8_tiles`` (for
    every 128 x 128). The codes lie in the order in which the tensor cores take them; ``to_dense`` gives the values."""

    __slots__ = ("_values", "_scales", "_tiled", "_shape", "_dims")

    def __init__(self, *args, **kwargs):
        raise TypeError("FP8_gpu is made by to_fp8_rows, to_fp8_tiles or gpu_expert_sort_fp8")

    tiled = property(lambda self: self._tiled)

    @property
    def shape(self):
        """(groups, rows, columns); one group where there is a scale per row."""
        return _host_shape(self)

    @property
    def device(self):
        return self._values.device

    def to_dense(self) -> torch.Tensor:
        """The float32 values that the codes and scales stand for."""
        groups, rows, cols = self._dims
        z = _native.fp8_unpack(self)
        return z.view(groups, rows, cols) if self._tiled else z

    def transposed(self) -> FP8_gpu:
        """Every group's transpose, for matrices with a scale per tile: the same codes in another order."""
        if not self._tiled:
            raise ValueError("transposed: only matrices with a scale per tile have a transpose")
        return _native.fp8_transpose(self)

    def __repr__(self):
        return f"FP8_gpu(shape={self._dims}, scales per {'tile' if self._tiled else 'row'})"


def _packed(codes, scales, tiled, where):
    if not isinstance(scales, torch.Tensor) or codes.dtype not in (torch.float8_e4m3fn, torch.uint8):
        raise TypeError(f"{where}: codes must be float8_e4m3fn (or their bytes) and come with a tensor of scales")
    if not codes.is_cuda or codes.dim() not in ((2, 3) if tiled else (2,)) or not codes.is_contiguous():
        raise TypeError(f"{where}: expected a contiguous CUDA tensor of {'2 or 3' if tiled else '2'} dimensions")
    if max(codes.shape) >= 1 << 31:
        raise ValueError(f"{where}: an extent beyond int32")
    blocks = [-(-n // BLOCK) for n in codes.shape[-2:]]
    want = (*codes.shape[:-2], *blocks) if tiled else (codes.shape[0], blocks[1])
    if scales.dtype != torch.float32 or scales.device != codes.device or tuple(scales.shape) != want:
        raise ValueError(f"{where}: expected float32 scales of shape {want} on the codes' device")
    return _native.fp8_pack(codes.view(torch.uint8), scales.contiguous(), tiled)


def to_fp8_rows(x, scales=None) -> FP8_gpu:
    """Rows in 8 bits with a scale for every 128 columns: with m the largest magnitude there (at least 2^-110) the scale is m / 448 and a code
    e4m3(x * (448 / m)). A NaN or infinity makes NaNs of its block. With ``scales`` (rows, blocks), ``x`` already holds codes (float8_e4m3fn)."""
    if scales is not None:
        return _packed(x, scales, False, "to_fp8_rows")
    return _native.fp8_rows(x)


def to_fp8_tiles(w, scales=None) -> FP8_gpu:
    """The same with a scale for every 128 x 128, of one matrix (n, inner) or of one per expert (experts, n, inner). With ``scales``
    ([experts,] row blocks, column blocks), ``w`` already holds codes, as a checkpoint does."""
    if scales is not None:
        return _packed(w, scales, True, "to_fp8_tiles")
    return _native.fp8_tiles(w)


def gpu_expert_order(r: CSR_gpu) -> ExpertOrder_gpu:
    """The order of the experts, for rows that are moved later. At most 4096 experts, and 2^31 - 1025 tokens and entries."""
    return _native.expert_order(r)


def gpu_expert_sort(r: CSR_gpu, x: torch.Tensor) -> tuple[ExpertOrder_gpu, torch.Tensor]:
    """The order and ``xs`` with ``xs[slot] = x[token]``, a row per entry of ``r``; zeros in the slots behind the last expert's."""
    return _native.expert_sort(r, x)


def gpu_expert_sort_fp8(r: CSR_gpu, x: torch.Tensor) -> tuple[ExpertOrder_gpu, FP8_gpu]:
    """The same with the rows quantised on the way, as ``to_fp8_rows(xs)`` has them."""
    return _native.expert_sort_fp8(r, x)


def gpu_expert_sort_grad(order: ExpertOrder_gpu, dxs: torch.Tensor) -> torch.Tensor:
    """Gradient of the sort: every token's sum of the rows at its entries' slots."""
    return _native.expert_sort_grad(order, dxs)


def gpu_expert_unsort(r: CSR_gpu, order: ExpertOrder_gpu, z: torch.Tensor) -> torch.Tensor:
    """``y[t]`` = sum of ``r.values[e] * z[slot(e)]`` over the kept entries of token ``t``, zeros for a token without any."""
    return _native.expert_unsort(r, order, z)


def gpu_expert_unsort_grad(r: CSR_gpu, order: ExpertOrder_gpu, z: torch.Tensor, dy: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Gradients ``(dz, dvalues)`` of the way back: ``dz[slot(e)] = r.values[e] * dy[t]`` and ``dvalues[e] = <dy[t], z[slot(e)]>`` (float32); zeros for
    what nothing depends on."""
    return _native.expert_unsort_grad(r, order, z, dy)


def gpu_fp8_product(a: FP8_gpu, w: FP8_gpu, order: ExpertOrder_gpu | None = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a @ w.T`` for rows ``a`` and tiles ``w``; with an order, the rows of expert ``c`` are multiplied with ``w[c]``, and slots of nobody get
    zeros (all of them where there are no experts)."""
    if dtype not in _TYPES:
        raise TypeError("gpu_fp8_product: dtype must be float32, float16 or bfloat16")
    return _native.fp8_product(a, w, order, _TYPES[dtype])


def gpu_fp8_product_grad(dy: torch.Tensor, x: torch.Tensor, w: FP8_gpu, order: ExpertOrder_gpu | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Gradients ``(dx, dw)`` of ``y = x @ w.T`` in 8 bits: ``dx`` is the product of ``dy``, quantised by rows, with the transposed tiles, in the type of
    ``dy``; ``dw`` (float32, the shape of ``w``) sums over every expert's rows, both operands quantised along those, a scale for every
    column and 128 rows. Rounding to 8 bits counts as the identity."""
    if not isinstance(w, FP8_gpu) or not w.tiled:
        raise TypeError("gpu_fp8_product_grad: w must be an FP8_gpu with a scale per tile")
    dx_type = _TYPES.get(getattr(dy, "dtype", None))
    if dx_type is None or not isinstance(x, torch.Tensor):
        raise TypeError("gpu_fp8_product_grad: dy and x must be CUDA tensors of rows of float32, float16 or bfloat16")
    groups, n, inner = w._dims
    if dy.dim() != 2 or dy.shape[1] != n or x.dim() != 2 or x.shape[1] != inner:
        raise ValueError(f"gpu_fp8_product_grad: dy and x must have {n} and {inner} columns")
    dw, rows = _native.fp8_grad_w(dy, x, order, groups)
    return _native.fp8_product(rows, w.transposed(), order, dx_type), dw


_native.bind_experts((ExpertOrder_gpu, FP8_gpu))
