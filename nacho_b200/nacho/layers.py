"""Layers around the routed experts, and what training and serving them takes: the gated half of a feed-forward layer with its gradients in 16 bits, linear
layers in 8-bit integers, and the norm by which gradients are clipped:

    h, both = gpu_gated_product(xs, w, order, keep=True)          # act(xs @ w[:hidden].T) * (xs @ w[hidden:].T), every expert with its own w
    dxs, dw = gpu_gated_product_grad(dh, both, xs, w, order)
    norm = gpu_clip_gradients([dw, ddown], 1.0)                   # in place
    y = gpu_int8_product(to_int8_rows(x), weights)                # weights = to_int8_rows(w), once

Operands and results are as in ``experts``: 2-D CUDA tensors with contiguous rows at any distance, new contiguous results without an autograd graph, no call
waits for the device, and all of them can be captured in graphs, products once one has been called on the stream. Sums are 32-bit (or exact) in a fixed
order and rounded once.
"""
from __future__ import annotations

import torch

from .experts import _TYPES, ExpertOrder_gpu
from .nacho_ext import _host_shape, _native

__all__ = ["INT8_gpu", "to_int8_rows", "gpu_gated_product", "gpu_gated_product_grad", "gpu_int8_product", "gpu_clip_gradients"]

_ACTIVATIONS = {"silu": 0, "gelu": 1}


class INT8_gpu:
    """Matrices in 8-bit integers with a 32-bit scale for every row, made by ``to_int8_rows``; ``to_dense`` gives the values."""

    __slots__ = ("_values", "_scales", "_shape", "_dims")

    def __init__(self, *args, **kwargs):
        raise TypeError("INT8_gpu is made by to_int8_rows")

    @property
    def shape(self):
        """(groups, rows, columns)."""
        return _host_shape(self)

    scales = property(lambda self: self._scales)

    @property
    def device(self):
        return self._values.device

    def to_dense(self) -> torch.Tensor:
        """The float32 values that the codes and scales stand for, (rows, columns), or (groups, rows, columns) of several groups."""
        z = _native.int8_unpack(self)
        return z if self._dims[0] == 1 else z.view(self._dims)

    def __repr__(self):
        return f"INT8_gpu(shape={self._dims})"


def to_int8_rows(x, scales=None) -> INT8_gpu:
    """Rows, of tokens (rows, inner), of a layer's channels (n, inner) or of every expert's (experts, n, inner), in 8-bit integers with a scale each: with m the
    row's largest magnitude (at least 2^-110) the scale is m / 127 and a code round(x * (127 / m)), ties to even. A row with a NaN or an infinity stands for
    NaNs. With ``scales`` ([experts,] rows), ``x`` already holds codes (int8), as a checkpoint does."""
    if scales is None:
        return _native.int8_rows(x)
    if not isinstance(x, torch.Tensor) or not isinstance(scales, torch.Tensor) or x.dtype != torch.int8:
        raise TypeError("to_int8_rows: codes must be int8 and come with a tensor of scales")
    if not x.is_cuda or x.dim() not in (2, 3) or not x.is_contiguous():
        raise TypeError("to_int8_rows: expected a contiguous CUDA tensor of 2 or 3 dimensions")
    if max(x.shape) >= 1 << 31:
        raise ValueError("to_int8_rows: an extent beyond int32")
    if scales.dtype != torch.float32 or scales.device != x.device or scales.shape != x.shape[:-1]:
        raise ValueError(f"to_int8_rows: expected float32 scales of shape {tuple(x.shape[:-1])} on the codes' device")
    return _native.int8_pack(x, scales.contiguous())


def _activation(name, where):
    if name not in _ACTIVATIONS:
        raise ValueError(f"{where}: activation must be one of {', '.join(_ACTIVATIONS)}")
    return _ACTIVATIONS[name]


def gpu_gated_product(x: torch.Tensor, w: torch.Tensor, order: ExpertOrder_gpu | None = None, activation: str = "silu", keep: bool = False):
    """``act(x @ w[:hidden].T) * (x @ w[hidden:].T)`` for float16 or bfloat16 ``x`` (rows, width) and ``w`` (2 hidden, width); with an order, ``w`` is
    (experts, 2 hidden, width), the rows of expert ``c`` take ``w[c]``, and slots of nobody get zeros. ``activation``: "silu", or "gelu" in its tanh form.
    ``keep``: also both products (rows, 2 hidden), as the gradients take them."""
    return _native.gated_product(x, w, order, _activation(activation, "gpu_gated_product"), bool(keep))


def gpu_gated_product_grad(dh: torch.Tensor, both: torch.Tensor, x: torch.Tensor, w: torch.Tensor, order: ExpertOrder_gpu | None = None,
                           activation: str = "silu") -> tuple[torch.Tensor, torch.Tensor]:
    """Gradients ``(dx, dw)`` of ``gpu_gated_product``, from the gradient of its result and the products it kept, all of one type. The gradient of both
    products is rounded to that type before it is multiplied, beside the rounding of the results (together 1.4 times as far from exact ones); zeros for
    what nothing depends on."""
    return _native.gated_product_grad(dh, both, x, w, order, _activation(activation, "gpu_gated_product_grad"))


def gpu_int8_product(a: INT8_gpu, w: INT8_gpu, order: ExpertOrder_gpu | None = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a @ w.T`` for rows ``a`` and channels ``w``, summed in whole numbers (at most 131071 columns); with an order, the rows of expert ``c`` are multiplied
    with ``w[c]``, and slots of nobody get zeros."""
    if dtype not in _TYPES:
        raise TypeError("gpu_int8_product: dtype must be float32, float16 or bfloat16")
    return _native.int8_product(a, w, order, _TYPES[dtype])


def gpu_clip_gradients(gradients, max_norm: float, out=None) -> torch.Tensor:
    """The root of the sum of all elements' squares of a list or tuple of tensors (a float32 tensor without dimensions), and every element times
    ``max_norm / (norm + 1e-6)`` where that is below 1: in place, or into the tensors ``out`` of the same shapes, which may be of other types (32-bit ones
    that an optimiser reads, say). A norm that is no finite number changes nothing, so that a caller who sees it can leave the step out. The tensors must not
    overlap in memory."""
    limit = float(max_norm)
    if not limit >= 0:
        raise ValueError("gpu_clip_gradients: max_norm must not be negative")
    return _native.clip(gradients, out, limit)


_native.bind_layers(INT8_gpu)
