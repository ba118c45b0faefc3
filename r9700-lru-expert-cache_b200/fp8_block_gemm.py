"""``fp8_block_gemm``: the FP8 128x128 block-scaled matrix product for any number of tokens, backed
by the sm_100a kernels of csrc/fp8_gemm.cu (``b200_fp8_block_gemm``).

The FP8 target head (``fp8_target_lmhead``) passes over its weight once for 64 tokens; a prompt's
hundreds or thousands of rows go through this product instead, with the same operands: activations
e4m3 with an fp32 scale for each row's group of 128 (``per_token_group_quant_fp8``,
``silu_mul_quant_group``) and weights e4m3 with an fp32 scale for each block of 128 x 128, row-major
as a checkpoint holds them or in the head's strip pack (``pack_fp8_block``).
"""
from __future__ import annotations

import torch

from . import _lib

_BLK = 128
FP8 = torch.float8_e4m3fn
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _operands(what: str, qx: torch.Tensor, wq: torch.Tensor, xs: torch.Tensor, ws: torch.Tensor,
              packed: bool) -> tuple:
    """Checks the four operands and returns the C entries' leading arguments with M, N and K."""
    dev = qx.device
    if not qx.is_cuda or wq.device != dev or xs.device != dev or ws.device != dev:
        _lib.require_cuda(what, qx, wq, xs, ws)
        raise ValueError(f"{what}: operands are on different devices")
    if qx.dtype is not FP8 or wq.dtype is not FP8 or qx.ndim != 2 or wq.ndim != 2:
        raise ValueError(f"{what}: qx and wq must be 2-D e4m3 tensors")
    M, K = qx.shape
    N, wk = wq.shape
    if wk != K:
        raise ValueError(f"{what}: weight {tuple(wq.shape)} does not match activations {tuple(qx.shape)}")
    if N < 1 or K < 16 or K % 16:
        raise ValueError(f"{what}: N must be at least 1 and K a positive multiple of 16 (N={N}, K={K})")
    kb, nb = (K + 127) // _BLK, (N + 127) // _BLK
    if xs.dtype is not torch.float32 or xs.shape != (M, kb):
        raise ValueError(f"{what}: xs must be fp32 [{M}, {kb}], got {xs.dtype} {tuple(xs.shape)}")
    xs_row, xs_col = xs.stride()
    ws_row, ws_col = ws.stride() if ws.ndim == 2 else (0, 0)
    if ws.dtype is not torch.float32 or ws.shape != (nb, kb) or (kb > 1 and ws_col != 1):
        raise ValueError(f"{what}: ws must be fp32 [{nb}, {kb}] with unit column stride, got {ws.dtype} "
                         f"{tuple(ws.shape)}")
    ldx, x_col = qx.stride()
    ldw, w_col = wq.stride()
    if M <= 1:
        ldx = K
    if packed:
        if N % 16 or K % _BLK or not wq.is_contiguous():
            raise ValueError(f"{what}: a strip pack is contiguous with N % 16 == 0 and K % 128 == 0")
        ldw, w_col = K, 1
    elif N == 1:
        ldw = K
    if x_col != 1 or w_col != 1 or ldx < K or ldw < K or ldx % 16 or ldw % 16:
        raise ValueError(f"{what}: rows of qx and wq must be contiguous, their strides multiples of 16")
    x_ptr, w_ptr = qx.data_ptr(), wq.data_ptr()
    if (M and x_ptr % 16) or w_ptr % 16:
        raise ValueError(f"{what}: qx and wq must be 16-byte aligned")
    return (x_ptr, ldx, xs.data_ptr(), xs_row, xs_col, w_ptr, ldw, int(packed), ws.data_ptr(), ws_row), M, N, K


def fp8_block_gemm(qx: torch.Tensor, wq: torch.Tensor, xs: torch.Tensor, ws: torch.Tensor,
                   out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None,
                   packed: bool = False) -> torch.Tensor:
    """(qx * xs) @ (wq * ws).T -> [M, N] in ``out_dtype`` (bf16, f16 or f32) or into ``out``.

    qx e4m3 [M, K], xs fp32 [M, ceil(K/128)] (any strides, so a group-major scale tensor may be
    passed transposed), wq e4m3 [N, K] row-major (or, with ``packed``, the strip pack of
    ``pack_fp8_block``), ws fp32 [ceil(N/128), ceil(K/128)]. K is a multiple of 16; rows of qx and
    wq may be strided by multiples of 16. Each 128-K block's sum is scaled and added in fp32 and
    the result rounded once."""
    args, M, N, K = _operands("fp8_block_gemm", qx, wq, xs, ws, packed)
    ldy = N
    if out is None:
        code = _DTYPES.get(out_dtype)
        if code is None:
            raise ValueError(f"fp8_block_gemm: unsupported output dtype {out_dtype}")
        out = torch.empty(M, N, dtype=out_dtype, device=qx.device)
    else:
        _lib.require_cuda("fp8_block_gemm", out)
        code = _DTYPES.get(out.dtype)
        if out.shape != (M, N) or code is None or out.device != qx.device or \
                (N > 1 and out.stride(1) != 1) or (M > 1 and out.stride(0) < N):
            raise ValueError(f"fp8_block_gemm: out must be bf16, f16 or f32 [{M}, {N}] on {qx.device} with unit "
                             "column stride and rows that do not overlap")
        if M > 1:
            ldy = out.stride(0)
    if M:
        _lib.launch("b200_fp8_block_gemm", _lib.score().b200_fp8_block_gemm, qx.device, *args, out.data_ptr(), ldy,
                    code, M, N, K)
    return out
