"""Log probabilities of given tokens, with entropy, rank and top alternatives: what a sampled step returns beside its
token, what scoring a prompt needs, and -- differentiable -- what a policy-gradient or distillation loss is made of.
No counterpart in the reference, whose call sites stop at the token (``engine/runtime/thinker_decode.py:83,107``,
``engine/talker_sampler.py:234-249``).

* ``token_logprobs``: from logits rows (raw, or the processed rows of ``talker_sampler.processed_logits``, whose
  masked ids are -inf);
* ``LMHeadLogprobs``: straight from hidden rows and a language-model or codec head on the tensor cores, the [B, V]
  logits never written.

With z = logits / temperature: ``logprob = z[token] - logsumexp(z)`` and ``entropy = -sum p log p`` (natural logarithm,
fp32).  A token of ``PAD`` (any id below 0, or one >= V) is no token: logprob 0, rank -1, no gradient through logprob.
A row that is -inf throughout has logprob -inf, entropy 0 and gradient 0; NaN or +inf in a row makes it NaN.

Both are differentiable through ``logprob`` and ``entropy`` (not through rank or alternatives, and once: there is no
second derivative, and tangents are refused).  All calls are asynchronous, run on the current stream and can be captured
in a CUDA graph; they keep no state between calls, so calls on several streams may overlap.  Waits inside the kernels are
bounded (``b2s_wait_limit``): one that gives up, which a sound GPU never sees, makes what it left unfinished NaN, ranks
and ids of alternatives -1, and sets 4 in ``status`` where there is one.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _native
from . import talker_sampler as ts

MAX_TOP = 32


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor                 # [B] float32
    entropy: torch.Tensor                 # [B] float32
    rank: torch.Tensor                    # [B] int64: ids before the token (value descending, id ascending); -1: none
    top_ids: Optional[torch.Tensor]       # [B, top] int64 in that order, or None
    top_logprobs: Optional[torch.Tensor]  # [B, top] float32, or None


class HeadLogprobs(NamedTuple):
    logprob: torch.Tensor  # [B] float32
    entropy: torch.Tensor  # [B] float32


def _check_temperature(t) -> float:
    t = ts._temperature(t)
    if not 1e-6 <= t <= 1e6:
        raise ValueError(f"temperature must be within [1e-6, 1e6], got {t!r}")
    return t


def _check_tokens(tokens: torch.Tensor, rows: int) -> torch.Tensor:
    if tokens.dim() != 1 or tokens.shape[0] != rows or tokens.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"tokens must be int64 [{rows}], got {tokens.dtype} {tuple(tokens.shape)}")
    return tokens if tokens.dtype == torch.int64 and tokens.is_contiguous() else tokens.to(torch.int64).contiguous()


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0, temperature: float = 1.0,
                   status: Optional[torch.Tensor] = None) -> TokenLogprobs:
    """Log probability, entropy and rank of ``tokens`` [B] under ``logits`` [B, V] (float32 or bfloat16, rows any
    stride apart), with the ``top`` most probable ids and their log probabilities (equal values: lowest id first)."""
    ts._need_cuda(logits, tokens, status)
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16) or logits.shape[1] < 1:
        raise ValueError("logits must be a float32 or bfloat16 [rows, vocab] tensor")
    if not 0 <= int(top) <= min(MAX_TOP, logits.shape[1]):
        raise ValueError(f"top must be within [0, {min(MAX_TOP, logits.shape[1])}], got {top}")
    temperature, top = _check_temperature(temperature), int(top)
    tokens = _check_tokens(tokens, logits.shape[0])
    lp, ent, rank, ids, vals, _ = _native.ops().token_logprobs(logits, tokens, temperature, top, False, status)
    return TokenLogprobs(lp, ent, rank, ids if top else None, vals if top else None)


class LMHeadLogprobs:
    """Log probability and entropy of given tokens straight from a head ([V, H] bf16, H a multiple of 8; the Thinker's
    LM head or the Talker's codec head): the logits are fp32 tensor-core sums that never leave the chip.  Any number
    of rows.  Differentiable in ``hidden`` and, where it requires a gradient, in the head; the gradient's workspace is
    rows x V x 2 bytes."""

    def __init__(self, head: torch.Tensor):
        ts._need_cuda(head)
        if head.dtype != torch.bfloat16 or head.dim() != 2 or head.shape[0] < 1:
            raise ValueError("head must be a bf16 [vocab, hidden] tensor")
        if head.shape[1] < 8 or head.shape[1] % 8:
            raise ValueError(f"hidden must be a multiple of 8, got {head.shape[1]}")
        self.head = head

    def __call__(self, hidden: torch.Tensor, tokens: torch.Tensor, *, temperature: float = 1.0,
                 status: Optional[torch.Tensor] = None) -> HeadLogprobs:
        ts._need_cuda(hidden, tokens, status)
        if hidden.dim() != 2 or hidden.shape[1] != self.head.shape[1] or hidden.dtype != torch.bfloat16:
            raise ValueError(f"hidden must be bf16 [rows, {self.head.shape[1]}]")
        temperature = _check_temperature(temperature)
        tokens = _check_tokens(tokens, hidden.shape[0])
        lp, ent, _ = _native.ops().lmhead_logprobs(hidden, self.head, tokens, temperature, False, status)
        return HeadLogprobs(lp, ent)
