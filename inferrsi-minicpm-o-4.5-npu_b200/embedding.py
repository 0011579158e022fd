"""The embedding lookup: what turns a sampled token back into the next step's input, and -- differentiable -- the other end
of training a head.  No counterpart in the reference, whose models call torch's own embedding.

    lookup(tokens, table, scale) = scale * table[tokens]

A token of ``PAD`` (any id below 0: what inactive rows sample) gives zeros and has no part in the gradient; an id past the
table is taken the same way and sets 32 in ``status``.  The table is float32, bfloat16 or a microscaled 4-bit matrix
(``mx.MXTensor``, no gradient; bfloat16 rows).  The gradient is the whole table's, in its type: every id's rows summed in
fp32 and rounded once.  The sums are of pieces of 8 to 32 positions, cut at fixed places of the list of all positions ordered by
id, in ascending order within a piece; an id's pieces are joined in a fixed tree.  The same call gives the same bits; where an id's
pieces are cut, and with that its last bits, depends on the other tokens of the call.

CUDA tensors only; on the current stream, without synchronising, keeping no state between calls; can be captured in a CUDA
graph.  Differentiable once, in the table.
"""

from __future__ import annotations

from typing import Optional, Union

import torch

from . import _native
from . import mx
from . import talker_sampler as ts

_F32_MAX = torch.finfo(torch.float32).max


def lookup(tokens: torch.Tensor, table: Union[torch.Tensor, "mx.MXTensor"], *, scale: float = 1.0,
           status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``scale * table[tokens]``: tokens int64 or int32 of any shape, table [vocab, width] with rows any stride apart;
    [*tokens.shape, width] in the table's type (bfloat16 from a 4-bit table)."""
    ts._need_cuda(tokens, table, status)
    scale = float(scale)
    if not abs(scale) <= _F32_MAX:
        raise ValueError(f"scale must be finite in float32, got {scale!r}")
    if tokens.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"tokens must be int64 or int32, got {tokens.dtype}")
    t = tokens if tokens.dim() == 1 else tokens.reshape(-1)
    if t.dtype != torch.int64 or not t.is_contiguous():
        t = t.to(torch.int64).contiguous()
    if isinstance(table, mx.MXTensor):
        if len(table.shape) != 2 or table.shape[0] < 1:
            raise ValueError(f"table must be [vocab, width], got {tuple(table.shape)}")
        width = table.shape[1]
        out = _native.ops().embedding_mx(t, table.codes, table.scales, width, scale, status)
    else:
        if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1:
            raise ValueError(f"table must be [vocab, width], got {tuple(table.shape)}")
        if table.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"table must be float32 or bfloat16, got {table.dtype}")
        width = table.shape[1]
        out = _native.ops().embedding(t, table, scale, status)
    return out if tokens.dim() == 1 else out.reshape(*tokens.shape, width)
