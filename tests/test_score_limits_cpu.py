"""Size limits of the scoring entries' C boundary: what 32-bit block numbers cannot hold is refused
before any launch."""
from __future__ import annotations

import ctypes

import pytest

from conftest import load_pkg

L = load_pkg()._lib
p = ctypes.c_void_p
TOP = 1 << 30


@pytest.mark.parametrize("K", [TOP + 16, (1 << 31) - 128, (1 << 31) - 16])
@pytest.mark.parametrize("M", [0, 1])
def test_k_beyond_the_block_count(K, M):
    """K + 127 would pass 32 bits in the kernels' count of 128-K blocks: -3, as every bad K."""
    operands = (p(16), K, p(16), 1, 1, p(16), K, 0, p(16), 1)
    assert L.score().b200_fp8_block_gemm(*operands, p(16), 128, 0, M, 128, K, None) == -3
    assert L.score().b200_fp8_head_logprobs(*operands, p(16), M, 128, K, p(16), p(16), p(16), p(16), 1 << 40, None) == -3


def test_the_largest_k_passes():
    operands = (p(16), TOP, p(16), 1, 1, p(16), TOP, 0, p(16), 1)
    assert L.score().b200_fp8_block_gemm(*operands, p(16), 128, 0, 0, 128, TOP, None) == 0
