"""Microscaled 4-bit matrices (OCP MX: E2M1 elements, a power-of-two scale for each 32 along a row) and their product: a
quarter of bf16's bytes for a head, a table or a projection, on tensor cores that take them at four times bf16's rate.
No counterpart in the reference.

* ``quantize`` / ``dequantize``: rows of float32 or bfloat16 to an ``MXTensor`` and back;
* ``linear``: ``projection.linear`` with both operands in 4 bits, ``act(x^ w^T + bias) + residual``: the weight is quantised
  once, x within the call (or before it);
* ``embedding.lookup`` reads rows of an ``MXTensor``.

A block's scale is 2^e with e = floor(log2 max|x|) - 2 (at least -127); an element is x 2^-e rounded to the nearest of 0, 0.5,
1, 1.5, 2, 3, 4, 6 and their negatives, ties to even, beyond 6 to 6.  A block that holds NaN or an infinity comes back as NaN
throughout.  ``quantize`` and ``dequantize`` have no gradient; ``linear``'s goes straight through x's rounding: dz =
dy act'(z), dx = dz w^, and so on for bias and residual; the weight is frozen.

CUDA tensors only; on the current stream, without synchronising, keeping no state between calls; can be captured in a CUDA
graph.  A device wait that gives up makes the unfinished outputs NaN and sets 4 in ``status``.
"""

from __future__ import annotations

from typing import Optional, Union

import torch

from . import _native
from . import talker_sampler as ts
from .projection import ACTIVATIONS

BLOCK = 32


class MXTensor:
    """A matrix of ``shape`` [..., k] in microscaled 4 bits, its leading dimensions taken as rows.

    ``codes``: uint8 [rows, 16 * ceil(k / 32)], two elements a byte, the first in the low half, zeros past a row's end.
    ``scales``: uint8 [ceil(rows / 128), ceil(k / 256), 1024], exponents plus 127 in tiles of 128 rows x 8 blocks; the scale
    of (row, block) of a tile is at ``block // 4 * 512 + row % 32 * 16 + row // 32 * 4 + block % 4``; zeros past the matrix.
    """

    __slots__ = ("codes", "scales", "shape")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape):
        shape = torch.Size(shape)
        if not shape or shape[-1] < 1 or min(shape) < 0:
            raise ValueError(f"shape must be [..., k] with k at least 1, got {tuple(shape)}")
        k, rows = shape[-1], shape[:-1].numel()
        for name, t, want in (("codes", codes, (rows, 16 * -(-k // BLOCK))),
                              ("scales", scales, (-(-rows // 128), -(-k // 256), 1024))):
            if not t.is_cuda:
                ts._need_cuda(t)
            if t.dtype is not torch.uint8 or t.shape != want or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"{name} must be contiguous 16-byte aligned uint8 {list(want)}, got {t.dtype} {list(t.shape)}")
        if codes.device != scales.device:
            raise ValueError("codes and scales must be on one device")
        self.codes, self.scales, self.shape = codes, scales, shape

    @classmethod
    def _made(cls, codes: torch.Tensor, scales: torch.Tensor, shape: torch.Size) -> "MXTensor":
        q = cls.__new__(cls)
        q.codes, q.scales, q.shape = codes, scales, shape
        return q

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def is_cuda(self) -> bool:
        return self.codes.is_cuda


def quantize(x: torch.Tensor) -> MXTensor:
    """x [..., k], float32 or bfloat16, rows any stride apart, as an ``MXTensor``."""
    ts._need_cuda(x)
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"x must be float32 or bfloat16, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be [..., k] with k at least 1, got {tuple(x.shape)}")
    x2 = x.detach() if x.requires_grad else x
    x2 = x2 if x2.dim() == 2 else x2.reshape(x.shape[:-1].numel(), x.shape[-1])
    return MXTensor._made(*_native.ops().mx_quantize(x2), x.shape)


def dequantize(q: MXTensor, *, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of an ``MXTensor``, float32 or bfloat16 (exact but for values below bfloat16's range)."""
    if not isinstance(q, MXTensor):
        raise ValueError(f"q must be an MXTensor, got {type(q).__name__}")
    if dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"dtype must be float32 or bfloat16, got {dtype}")
    x = _native.ops().mx_dequantize(q.codes, q.scales, q.shape[-1], dtype)
    return x if len(q.shape) == 2 else x.reshape(q.shape)


def linear(x: Union[torch.Tensor, MXTensor], weight: MXTensor, bias: Optional[torch.Tensor] = None, *,
           activation: Optional[str] = None, residual: Optional[torch.Tensor] = None,
           status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x^ weight^T + bias) + residual``: x [..., in] bfloat16 (rounded to 4 bits within the call) or an ``MXTensor``,
    weight an ``MXTensor`` [out, in], bias [out] and residual [..., out] bfloat16; any in and out.  ``activation``: None,
    "relu", "gelu" or "silu" (0 at -infinity).  Differentiable once, in x, bias and residual; the gradient of x takes
    the weight in bfloat16, out * in * 2 bytes of workspace."""
    ts._need_cuda(x, bias, residual, status)
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation: {activation!r}")
    if not isinstance(weight, MXTensor) or len(weight.shape) != 2 or weight.shape[0] < 1:
        raise ValueError("weight must be an MXTensor [out, in]")
    n, k = weight.shape
    quantised = isinstance(x, MXTensor)
    if not quantised and x.dtype != torch.bfloat16:
        raise ValueError(f"x must be bfloat16 or an MXTensor, got {x.dtype}")
    if len(x.shape) < 1 or x.shape[-1] != k:
        raise ValueError(f"x [..., in] and weight [out, in] do not fit: {tuple(x.shape)}, {tuple(weight.shape)}")
    for name, t in (("bias", bias), ("residual", residual)):
        if t is not None and t.dtype != torch.bfloat16:
            raise ValueError(f"{name} must be bfloat16, got {t.dtype}")
    if bias is not None and tuple(bias.shape) != (n,):
        raise ValueError(f"bias must be [{n}], got {tuple(bias.shape)}")
    shape = (*x.shape[:-1], n)
    if residual is not None and tuple(residual.shape) != shape:
        raise ValueError(f"residual must be {shape}, got {tuple(residual.shape)}")
    if quantised:
        x2, xs = x.codes, x.scales
    else:
        x2, xs = x if x.dim() == 2 else x.reshape(x.shape[:-1].numel(), k), None
    r2 = residual if residual is None or residual.dim() == 2 else residual.reshape(x2.shape[0], n)
    out, _ = _native.ops().mx_linear(x2, xs, weight.codes, weight.scales, k, bias, r2, ACTIVATIONS[activation], False, status)
    return out if len(shape) == 2 else out.reshape(shape)
