"""Log probabilities of given tokens, with entropy and top alternatives, from logits rows.

    token_logprobs(logits, ids, top=0) -> (logprob, entropy, top_logprob, top_id)

The full-vocabulary readout beside int8_kernels.option_logits (which reads only gathered label
rows): what scoring answers of several tokens needs (mica_b200.answers). The reference has no
counterpart: it never looks past its label rows (v0.5/serving/lib/release_runtime.py:298-306).

Errors follow fused_kernels: ValueError for arguments that fit no call, RuntimeError for what the
kernels do not serve (a CPU tensor, another dtype). There is no CPU branch.
"""
from __future__ import annotations

import torch

from . import _native as N
from .int8_kernels import _launched

MAX_TOP = 32


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, top: int = 0):
    """logits [N, V] (bf16, fp16 or fp32; unit column stride, any row stride), ids int64 [N] or [N, M].

    Returns fp32 logprob (the shape of ids), fp32 entropy [N] in nats, fp32 top_logprob [N, top] and
    int64 top_id [N, top] (largest first, ties by the lowest id; top <= 32). -inf logits are tokens
    that are not allowed; a row with nothing else has log probability -inf everywhere and entropy 0.
    A negative id is padding and gives 0, one past the end NaN; a NaN or +inf logit makes its row NaN."""
    r = N.calls().token_logprobs(logits, ids, top)
    _launched()
    return r
