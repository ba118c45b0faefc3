"""A scoring kernel whose pipeline wait runs out returns, says so in the error word and leaves NaN, never
a plausible number, and the device goes on. The limit of the waits is set to nothing in a process of its
own, so that each wait gives up after one try; no kernel waits for anything that does not come."""
from __future__ import annotations

import os
import subprocess
import sys

import pytest

from conftest import PKG_NAME, ROOT

pytestmark = pytest.mark.gpu

CHILD = f"""
import importlib, sys
sys.path[:0] = [{ROOT!r}, {os.path.join(ROOT, "tests")!r}]
import torch
P = importlib.import_module({PKG_NAME!r})
from test_fp8_block_gemm_gpu import operands
dev = torch.device("cuda:0")
err = P._lib.score().b200_score_error
# one tile with K split and without, 64, 128 and 256 columns, pairs of CTAs, several tiles a CTA
for M, N, K in [(5, 2560, 2560), (64, 640, 128), (16, 10240, 512), (100, 1040, 2560), (8, 60000, 640), (300, 1000, 384),
                (700, 60000, 1280)]:
    ops = operands(M, N, K, dev, seed=M)
    assert err(1) == 0
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        y = torch.zeros(M, N, dtype=dtype, device=dev)
        P.fp8_block_gemm.fp8_block_gemm(*ops, out=y)
        torch.cuda.synchronize()
        assert torch.isnan(y).all() and err(1) == 1, (M, N, K, dtype)
    r = P.logprobs.fp8_head_logprobs(*ops, torch.arange(M, device=dev))
    torch.cuda.synchronize()
    assert all(torch.isnan(t).all() for t in r) and err(1) == 1, (M, N, K)
# the device goes on, and what waits for nothing is as ever
x = torch.randn(3, 1000, device=dev)
lp = P.logprobs.token_logprobs(x, torch.tensor([0, 5, 999], device=dev)).logprob
want = torch.log_softmax(x.double(), 1)[[0, 1, 2], [0, 5, 999]]
assert (lp.double() - want).abs().max() < 1e-5 and err(1) == 0
print("done")
"""


def test_waits_that_run_out(cuda):
    env = dict(os.environ, B200_SCORE_WAIT_TRIES="0")
    env.pop("B200_LMHEAD_CHECK", None)
    r = subprocess.run([sys.executable, "-c", CHILD], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "done", r.stderr[-2000:]
