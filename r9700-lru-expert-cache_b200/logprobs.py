"""Log probabilities of given tokens: ``token_logprobs`` from logits, with the entropy, the token's
rank and the top alternatives of every row (csrc/logprobs.cu), ``fp8_head_logprobs`` from the FP8
head's operands without its logits (csrc/fp8_gemm.cu), and ``score_prompt``, a prompt's hidden
states to its tokens' log probabilities with the two and ``fp8_block_gemm``.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .fp8_block_gemm import _operands, fp8_block_gemm

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_TOP_K = 64


class TokenLogprobs(NamedTuple):
    """Per row: the token's log probability, the entropy and the logsumexp (fp32 [M]), the token's
    rank (int64 [M], 1 = no logit is larger) and the top alternatives (int64 and fp32 [M, top_k])."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    logsumexp: torch.Tensor
    rank: torch.Tensor
    top_ids: torch.Tensor
    top_logprobs: torch.Tensor


class HeadLogprobs(NamedTuple):
    """Per row, fp32 [M]: the token's log probability, the entropy, the logsumexp."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    logsumexp: torch.Tensor


def _ids(what: str, token_ids: torch.Tensor, M: int, device: torch.device) -> torch.Tensor:
    if token_ids.device != device or token_ids.shape != (M,) or token_ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{what}: token_ids must be int64 or int32 [{M}] on {device}, got {token_ids.dtype} "
                         f"{tuple(token_ids.shape)} on {token_ids.device}")
    if token_ids.dtype is not torch.int64 or not token_ids.is_contiguous():
        token_ids = token_ids.to(torch.int64).contiguous()
    return token_ids


def token_logprobs(logits: torch.Tensor, token_ids: torch.Tensor, top_k: int = 0) -> TokenLogprobs:
    """The log probability of ``token_ids`` [M] under softmax(logits [M, V]) (bf16, f16 or f32, unit
    column stride), with each row's entropy, logsumexp, the token's rank and the ``top_k`` (up to 64)
    most likely tokens, the lower id first among equal logits.

    A -inf logit has probability 0. A row of nothing but -inf has logsumexp and log probabilities
    -inf and entropy 0; a row with a NaN or +inf has NaN for all three. A token id outside [0, V)
    has log probability NaN and rank 0."""
    dev, code = logits.device, _DTYPES.get(logits.dtype)
    if not logits.is_cuda or code is None or logits.ndim != 2:
        _lib.require_cuda("token_logprobs", logits)
        raise ValueError("token_logprobs: logits must be bf16, f16 or f32 [M, V]")
    M, V = logits.shape
    ld, col = logits.stride()
    if V < 1 or (V > 1 and col != 1):
        raise ValueError("token_logprobs: logits must have columns, of unit stride")
    if not 0 <= top_k <= MAX_TOP_K or top_k > V:
        raise ValueError(f"token_logprobs: top_k must be between 0 and min(V, {MAX_TOP_K}), got {top_k}")
    if M <= 1:
        ld = V
    elif ld < V:
        raise ValueError("token_logprobs: rows of logits must not overlap")
    ids = _ids("token_logprobs", token_ids, M, dev)
    lp, ent, lse = torch.empty(3, M, dtype=torch.float32, device=dev).unbind(0)
    rank = torch.empty(M, dtype=torch.int64, device=dev)
    top_ids = torch.empty(M, top_k, dtype=torch.int64, device=dev)
    top_lp = torch.empty(M, top_k, dtype=torch.float32, device=dev)
    if M:
        _lib.launch("b200_token_logprobs", _lib.score().b200_token_logprobs, dev, logits.data_ptr(), code, ld, M, V,
                    ids.data_ptr(), top_k, lp.data_ptr(), rank.data_ptr(), ent.data_ptr(), lse.data_ptr(),
                    top_ids.data_ptr(), top_lp.data_ptr())
    return TokenLogprobs(lp, ent, lse, rank, top_ids, top_lp)


def fp8_head_logprobs(qx: torch.Tensor, wq: torch.Tensor, xs: torch.Tensor, ws: torch.Tensor,
                      token_ids: torch.Tensor, packed: bool = False) -> HeadLogprobs:
    """``token_logprobs`` of the logits (qx * xs) @ (wq * ws).T, kept in fp32 and never written to
    memory: operands as for ``fp8_block_gemm``, outputs without rank and alternatives."""
    args, M, N, K = _operands("fp8_head_logprobs", qx, wq, xs, ws, packed)
    ids = _ids("fp8_head_logprobs", token_ids, M, qx.device)
    dev = qx.device
    lp, ent, lse = torch.empty(3, M, dtype=torch.float32, device=dev).unbind(0)
    if M:
        lib = _lib.score()
        scratch = torch.empty(lib.b200_fp8_head_logprobs_workspace_bytes(M, N), dtype=torch.uint8, device=dev)
        _lib.launch("b200_fp8_head_logprobs", lib.b200_fp8_head_logprobs, dev, *args, ids.data_ptr(), M, N, K,
                    lp.data_ptr(), ent.data_ptr(), lse.data_ptr(), scratch.data_ptr(), scratch.numel())
    return HeadLogprobs(lp, ent, lse)


def score_prompt(hidden: torch.Tensor, wq: torch.Tensor, ws: torch.Tensor, token_ids: torch.Tensor,
                 top_k: int = 0, packed: bool = True, rows_at_once: int = 1024) -> TokenLogprobs | HeadLogprobs:
    """The log probabilities of a prompt's tokens: hidden bf16 or f16 [M, K] (row i predicts
    token_ids[i]) quantized per group of 128, through the FP8 head (wq, ws), the strip pack of
    ``pack_fp8_block`` by default. Without alternatives (top_k 0) the logits are never written;
    with them they are, in 32 bits like the head's own, for ``rows_at_once`` rows at a time (4 bytes a
    row and token of the vocabulary)."""
    if rows_at_once < 1:
        raise ValueError("score_prompt: rows_at_once must be at least 1")
    _lib.require_cuda("score_prompt", hidden)
    with torch.cuda.device(hidden.device):           # (the quantiser launches on the current device)
        return _score_prompt(hidden, wq, ws, token_ids, top_k, packed, rows_at_once)


def _score_prompt(hidden, wq, ws, token_ids, top_k, packed, rows_at_once):
    from .fused_silu_mul_quant import per_token_group_quant_fp8
    qx, xs = per_token_group_quant_fp8(hidden)
    if top_k == 0:
        return fp8_head_logprobs(qx, wq, xs, ws, token_ids, packed=packed)
    M = hidden.shape[0]
    ids = _ids("score_prompt", token_ids, M, hidden.device)
    parts = []
    logits = torch.empty(min(M, rows_at_once), wq.shape[0], dtype=torch.float32, device=hidden.device)
    for r0 in range(0, max(M, 1), rows_at_once):
        r1 = min(M, r0 + rows_at_once)
        y = fp8_block_gemm(qx[r0:r1], wq, xs[r0:r1], ws, out=logits[:r1 - r0], packed=packed)
        parts.append(token_logprobs(y, ids[r0:r1], top_k))
    return parts[0] if len(parts) == 1 else TokenLogprobs(*(torch.cat(t) for t in zip(*parts)))
