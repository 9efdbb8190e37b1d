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

from . import ops
from .int8_kernels import _launched
from .paged import _served

MAX_TOP = 32


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, top: int = 0):
    """logits [N, V] (bf16, fp16 or fp32; unit column stride, any row stride), ids int64 [N] or [N, M].

    Returns fp32 logprob (the shape of ids), fp32 entropy [N] in nats, fp32 top_logprob [N, top] and
    int64 top_id [N, top] (largest first, ties by the lowest id; top <= 32). -inf logits are tokens
    that are not allowed; a row with nothing else has log probability -inf everywhere and entropy 0.
    A negative id is padding and gives 0, one past the end NaN; a NaN or +inf logit makes its row NaN."""
    if logits.dim() != 2 or ids.dim() not in (1, 2) or ids.shape[0] != logits.shape[0]:
        raise ValueError(f'token_logprobs: logits {tuple(logits.shape)} with ids {tuple(ids.shape)}')
    if ids.dtype != torch.int64:
        raise ValueError(f'token_logprobs: ids are int64, not {ids.dtype}')
    if not 0 <= top <= min(MAX_TOP, logits.shape[1]):
        raise ValueError(f'token_logprobs: top {top} of {logits.shape[1]} tokens (at most {MAX_TOP})')
    if logits.shape[1] == 0 or logits.shape[1] >= 2**31 or logits.shape[0] >= 2**31:
        raise ValueError(f'token_logprobs: logits {tuple(logits.shape)}')
    if logits.device.type != 'cuda' or ids.device != logits.device:
        raise RuntimeError(f'token_logprobs: CUDA tensors of one device only, not {logits.device} and {ids.device}')
    if logits.dtype not in ops.DTYPE_CODE:
        raise RuntimeError(f'token_logprobs: {logits.dtype} is not served (bf16, fp16 or fp32)')
    if not _served(logits.device):
        raise RuntimeError('token_logprobs: not a B200 (sm_100)')
    if logits.requires_grad and torch.is_grad_enabled():
        raise RuntimeError('token_logprobs: no backward pass (call it under torch.no_grad())')
    if logits.stride(1) != 1 and logits.shape[1] > 1 or logits.stride(0) < logits.shape[1] and logits.shape[0] > 1:
        logits = logits.contiguous()
    two = ids[:, None] if ids.dim() == 1 else ids
    if two.shape[1] > 1 and two.stride(1) != 1 or two.stride(0) < two.shape[1] and two.shape[0] > 1:
        two = two.contiguous()
    lp, ent, top_lp, top_id = ops.token_logprobs_do(logits, two, top)
    _launched()
    return lp.view(ids.shape), ent, top_lp, top_id
