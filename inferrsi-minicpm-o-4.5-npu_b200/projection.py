"""The projections around the heads -- Thinker rows to the Talker's width (``engine/models/talker.py``, ``condition``),
the layers that feed a head -- as one tensor-core product with everything in its epilogue:

    linear(x, weight, bias, activation, residual) = act(x weight^T + bias) + residual

bf16 in and out, fp32 in between, rounded once.  Differentiable in x, weight, bias and residual (once).  Like the head
products of this engine it takes CUDA tensors only, runs on the current stream, never synchronises, keeps no state
between calls and can be captured in a CUDA graph.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _native
from . import talker_sampler as ts

# the activations' C-ABI codes; "gelu" is the exact form, 0.5 z (1 + erf(z / sqrt 2))
ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "silu": 3}


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, status):
        out, preact = _native.ops().linear(x, weight, bias, residual, act, act != 0, status)
        ctx.save_for_backward(x, weight, preact if act else None)
        ctx.act, ctx.status = act, status
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, weight, preact = ctx.saved_tensors
        want_x, want_w, want_b, want_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if want_x or want_w or want_b:
            dx, dw, db = _native.ops().linear_grad(g, x, weight, preact, ctx.act, want_x, want_w, want_b, ctx.status)
        return (dx if want_x else None, dw if want_w else None, db if want_b else None, g if want_r else None, None,
                None)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
           activation: Optional[str] = None, residual: Optional[torch.Tensor] = None,
           status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x weight^T + bias) + residual``: x [..., in], weight [out, in], bias [out], residual [..., out], all bf16;
    in a multiple of 8, any out.  ``activation``: None, "relu", "gelu" or "silu"."""
    ts._need_cuda(x, weight, bias, residual, status)
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation: {activation!r}")
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
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x2, weight, bias, r2)):
        out = _Linear.apply(x2, weight, bias, r2, act, status)
    else:
        out, _ = _native.ops().linear(x2, weight, bias, r2, act, False, status)
    return out if x.dim() == 2 else out.reshape(shape)
