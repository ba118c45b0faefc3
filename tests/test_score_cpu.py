"""CPU-only checks of the scoring entries' boundary (include/b200_score.h): every declared symbol is
exported and bound, the argument codes come back before any launch, and the Python entry points
refuse what the kernels do not take."""
from __future__ import annotations

import ctypes
import os
import re

import pytest
import torch

from conftest import ROOT, load_pkg

P = load_pkg()
L = P._lib
FP8 = torch.float8_e4m3fn


def test_every_declared_symbol_is_exported():
    src = open(os.path.join(ROOT, "include", "b200_score.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    names = re.findall(r"\b([A-Za-z_][A-Za-z0-9_]*)\s*\([^;{]*\)\s*;", src)
    lib = L.score()
    assert len(names) == 5
    for n in names:
        assert hasattr(lib, n), n
    assert set(names) == set(L.SCORE_PROTOS)


def _gemm(M=4, N=128, K=128, ldx=None, ldw=None, ldy=None, packed=0, dtype=0, x=16, w=16, y=16):
    p = ctypes.c_void_p
    return L.score().b200_fp8_block_gemm(p(x), K if ldx is None else ldx, p(16), 1, 1, p(w), K if ldw is None else ldw,
                                         packed, p(16), 1, p(y), N if ldy is None else ldy, dtype, M, N, K, None)


@pytest.mark.parametrize("args,code", [
    (dict(M=-1), -1), (dict(M=(1 << 30) + 1), -1), (dict(N=0), -2), (dict(N=(1 << 30) + 1, ldy=1 << 31), -2), (dict(N=130, packed=1), -2), (dict(K=0), -3), (dict(K=24), -3),
    (dict(K=144, packed=1), -3), (dict(ldx=112), -4), (dict(ldx=136), -4), (dict(ldw=112), -4), (dict(ldw=130), -4),
    (dict(ldy=127), -4), (dict(dtype=3), -5), (dict(dtype=-1), -5), (dict(x=8), -10), (dict(w=17), -10),
    (dict(y=17), -10), (dict(y=18, dtype=2), -10), (dict(M=0), 0)])
def test_gemm_codes(args, code):
    assert _gemm(**args) == code


def _logprobs(dtype=0, ld=100, M=4, V=100, top_k=0, x=16):
    p = ctypes.c_void_p
    return L.score().b200_token_logprobs(p(x), dtype, ld, M, V, p(16), top_k, *[p(16)] * 6, None)


@pytest.mark.parametrize("args,code", [
    (dict(M=-1), -1), (dict(M=(1 << 27) + 1), -1), (dict(V=0), -2), (dict(V=(1 << 30) + 1, ld=1 << 31), -2), (dict(ld=99), -4), (dict(dtype=3), -5), (dict(top_k=-1), -6),
    (dict(top_k=65), -6), (dict(V=10, top_k=11), -6), (dict(x=17), -10), (dict(x=18, dtype=2), -10), (dict(M=0), 0)])
def test_logprobs_codes(args, code):
    assert _logprobs(**args) == code


def _head(M=4, N=128, K=128, ws_ptr=16, ws_bytes=None):
    p = ctypes.c_void_p
    lib = L.score()
    need = lib.b200_fp8_head_logprobs_workspace_bytes(M, N) if ws_bytes is None else ws_bytes
    return lib.b200_fp8_head_logprobs(p(16), K, p(16), 1, 1, p(16), K, 0, p(16), 1, p(16), M, N, K, p(16), p(16), p(16),
                                      p(ws_ptr), need, None)


@pytest.mark.parametrize("args,code", [
    (dict(M=-1), -1), (dict(N=0), -2), (dict(K=8), -3), (dict(ws_ptr=0), -9), (dict(ws_bytes=8), -9),
    (dict(ws_ptr=8), -10), (dict(M=0), 0)])
def test_head_codes(args, code):
    assert _head(**args) == code


def test_workspace_bytes_do_not_wrap():
    b = L.score().b200_fp8_head_logprobs_workspace_bytes
    assert b(0, 5) == 0 and b(5, 0) == 0 and 0 < b(1, 1) <= 4096
    assert b(1 << 20, 1 << 20) > 1 << 32


def test_host_tensors_are_refused():
    q, w = torch.zeros(2, 128, dtype=FP8), torch.zeros(128, 128, dtype=FP8)
    xs, ws, ids = torch.zeros(2, 1), torch.zeros(1, 1), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        P.fp8_block_gemm.fp8_block_gemm(q, w, xs, ws)
    with pytest.raises(ValueError, match="CUDA"):
        P.logprobs.token_logprobs(torch.zeros(2, 5), ids)
    with pytest.raises(ValueError, match="CUDA"):
        P.logprobs.fp8_head_logprobs(q, w, xs, ws, ids)
