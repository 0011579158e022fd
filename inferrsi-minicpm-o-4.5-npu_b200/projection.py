"""The projections around the heads -- Thinker rows to the Talker's width (``engine/models/talker.py``, ``condition``),
the layers that feed a head -- as one tensor-core product with everything in its epilogue:

    linear(x, weight, bias, activation, residual) = act(x weight^T + bias) + residual

``checkpoint="e4m3"`` keeps what the backward pass needs, x and the pre-activation, in microscaled 8 bits (OCP MX: blocks of
32 along a row, each with a power-of-two scale, elements rounded to E4M3): about 2 bytes for each pair of input and output
elements instead of 4, at 3 fraction bits, so that the weight's gradient is 2 to 3 % off and slopes are those of the rounded
pre-activation; a block that holds NaN or an infinity comes back as NaN.  The output, and the gradients of x (but for its
slopes) and residual, are as without.

bf16 in and out, fp32 in between, rounded once.  Differentiable in x, weight, bias and residual (once).  Like the head
products of this engine it takes CUDA tensors only, runs on the current stream, never synchronises, keeps no state
between calls and can be captured in a CUDA graph.  A device wait that gives up makes the unfinished outputs NaN and sets
4 in ``status``.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _native
from . import talker_sampler as ts

# the activations' C-ABI codes; "gelu" is the exact form, 0.5 z (1 + erf(z / sqrt 2))
ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "silu": 3}


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
           activation: Optional[str] = None, residual: Optional[torch.Tensor] = None,
           status: Optional[torch.Tensor] = None, checkpoint: Optional[str] = None) -> torch.Tensor:
    """``act(x weight^T + bias) + residual``: x [..., in], weight [out, in], bias [out], residual [..., out], all bf16;
    in a multiple of 8, any out.  ``activation``: None, "relu", "gelu" or "silu" (0 at -infinity).  ``checkpoint``: None, or
    "e4m3" to keep 8 bits of x and of the pre-activation for the backward pass."""
    ts._need_cuda(x, weight, bias, residual, status)
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation: {activation!r}")
    if checkpoint not in (None, "e4m3"):
        raise ValueError(f"unknown checkpoint format: {checkpoint!r}")
    for name, t in (("x", x), ("weight", weight), ("bias", bias), ("residual", residual)):
        if t is not None and t.dtype != torch.bfloat16:
            raise ValueError(f"{name} must be bfloat16, got {t.dtype}")
    if weight.dim() != 2 or weight.shape[0] < 1 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x [..., in] and weight [out, in] do not fit: {tuple(x.shape)}, {tuple(weight.shape)}")
    n, k = weight.shape
    if k < 8 or k % 8:
        raise ValueError(f"in must be a multiple of 8, got {k}")
    if bias is not None and tuple(bias.shape) != (n,):
        raise ValueError(f"bias must be [{n}], got {tuple(bias.shape)}")
    shape = (*x.shape[:-1], n)
    if residual is not None and tuple(residual.shape) != shape:
        raise ValueError(f"residual must be {shape}, got {tuple(residual.shape)}")
    act = ACTIVATIONS[activation]
    x2 = x if x.dim() == 2 else x.reshape(-1, k)
    r2 = residual if residual is None or x.dim() == 2 else residual.reshape(-1, n)
    if checkpoint is None:
        out, _ = _native.ops().linear(x2, weight, bias, r2, act, False, status)
    else:
        out = _native.ops().linear_kept(x2, weight, bias, r2, act, False, False, status)[0]
    return out if x.dim() == 2 else out.reshape(shape)
