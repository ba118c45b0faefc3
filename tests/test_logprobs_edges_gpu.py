"""Rows on which a log probability kernel goes wrong easily, against the formulas in 64 bits: NaN
beside ordinary logits, NaN everywhere, sharply peaked rows.

Ranks and ids are exact; tolerances stand at their tests."""
from __future__ import annotations

import math

import pytest
import torch

from conftest import load_pkg

pytestmark = pytest.mark.gpu
P = load_pkg()
LP = P.logprobs
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def logits(M, V, dtype, dev, seed=0, scale=3.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = (torch.randn(M, V, device=dev, generator=g) * scale).to(dtype)
    return x, torch.randint(V, (M,), device=dev, generator=g)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,off", [(7, 0), (1000, 0), (5003, 5), (151936, 0)])
def test_rank_beside_nan(cuda, dtype, V, off):
    """rank = 1 + the number of larger logits, also where a NaN stands among them (it is not larger, and
    the logits next to it still count), in rows that start anywhere; a NaN token has rank 1."""
    M = 6
    big, ids = logits(M, V + off, dtype, cuda, seed=V + off)
    x, ids = big[:, off:], ids % V
    x[0, V // 2] = math.nan
    x[1, ::7] = math.nan
    x[2, ::2] = math.nan
    x[3, 1:] = math.nan
    x[4, V - 1] = math.nan
    x[5, 0], x[5, V - 1] = math.nan, math.inf
    ids[3], ids[4] = 0, V - 1
    ids[2] = min(V - 1, 2 * (V // 6) + 1)
    r = LP.token_logprobs(x, ids)
    assert torch.equal(r.rank, 1 + (x > x.gather(1, ids[:, None])).sum(1))
    assert r.rank[4] == 1
    for t in (r.logprob, r.entropy, r.logsumexp):
        assert torch.isnan(t).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,V,k", [(1, 64, 64), (2, 9001, 20), (200, 151936, 64)])
def test_top_of_rows_of_nothing_but_nan(cuda, dtype, M, V, k):
    """NaN comes first and equal ones by the lower id: 0, 1, 2 ... where every logit is NaN, also in a CTA
    that has a whole long row and so more of them than it keeps."""
    x = torch.full((M, V), math.nan, dtype=dtype, device=cuda)
    r = LP.token_logprobs(x, torch.zeros(M, dtype=torch.int64, device=cuda), top_k=k)
    assert torch.equal(r.top_ids, torch.arange(k, device=cuda).expand(M, k))
    assert torch.isnan(r.top_logprobs).all() and (r.rank == 1).all()
