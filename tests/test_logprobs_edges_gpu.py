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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,V", [(1, 151936), (9, 151936), (512, 151936), (40, 5003)])
@pytest.mark.parametrize("peak", [12.0, 20.0, 30.0, 39.0, 60.0])
def test_peaked_rows(cuda, dtype, M, V, peak):
    """One logit far above the others, as in most rows of a text: nothing is lost against sums relative to
    the row's maximum, no log probability is above 0 and no entropy below.

    Tolerance, with t = 1 - p_max and W = sum p d (d = x - max). Relative to the maximum its term is 1 to
    exp2's 2^-22, the others together t with 2^-22 + 50 2^-24 for each term's argument and at most 600
    2^-24 for a thread's additions; the additions to the maximum's own sum lose no more than what is added
    (t), and no more than 300 of 2^-24; 16 further operations of 2^-24 join threads, warps and CTAs. So
    ln S is off by a = 2^-22 + 16 2^-24 + t 2^-14 + min(t, 300 2^-24), the entropy by a + |W| 2^-14 and
    the results' own rounding (three operations) is 2^-22 of their size."""
    x, ids = logits(M, V, dtype, cuda, seed=int(peak), scale=2.5)
    at = torch.randint(V, (M,), device=cuda, generator=torch.Generator(device=cuda).manual_seed(M))
    x[torch.arange(M, device=cuda), at] = peak
    ids[::3] = at[::3]
    p = torch.log_softmax(x.double(), 1)
    prob = torch.exp(p)
    others = prob.clone()
    others.scatter_(1, x.argmax(1, keepdim=True), 0.0)
    t = others.sum(1)
    d = x.double() - x.amax(1, keepdim=True).double()
    mean = (prob * d).sum(1).abs()
    a = 2.0 ** -22 + 16 * 2.0 ** -24 + t * 2.0 ** -14 + t.clamp(max=300 * 2.0 ** -24)
    r = LP.token_logprobs(x, ids, top_k=3)
    want = p.gather(1, ids[:, None])[:, 0]
    assert ((r.logprob - want).abs() <= a + 2.0 ** -22 * want.abs()).all()
    lse = torch.logsumexp(x.double(), 1)
    assert ((r.logsumexp - lse).abs() <= a + 2.0 ** -22 * lse.abs()).all()
    entropy = -(prob * p).sum(1)
    assert ((r.entropy - entropy).abs() <= a + mean * 2.0 ** -14 + 2.0 ** -22 * entropy).all()
    top = p.gather(1, r.top_ids)
    assert ((r.top_logprobs - top).abs() <= a[:, None] + 2.0 ** -22 * top.abs()).all()
    assert (r.logprob <= 0).all() and (r.top_logprobs <= 0).all() and (r.entropy >= 0).all()


@pytest.mark.parametrize("M", [4, 128, 300])
@pytest.mark.parametrize("scale", [1.0, 30.0, 100.0, 1000.0])
def test_head_signs(cuda, M, scale):
    """The head's log probabilities are never above 0 and its entropies never below, however sharp a row
    is: exactly, since text is mostly rows whose largest logit has all of the probability."""
    from test_fp8_block_gemm_gpu import operands, reference
    qx, wq, xs, ws = operands(M, 5000, 512, cuda, seed=3)
    xs *= scale
    y, _ = reference(qx, wq, xs, ws)
    r = LP.fp8_head_logprobs(qx, wq, xs, ws, y.argmax(1))
    assert (r.logprob <= 0).all() and (r.entropy >= 0).all()
    assert (r.logsumexp >= y.amax(1).float() * (1 - 1e-5) - 1e-4).all()


@pytest.mark.parametrize("M,rows", [(1, 1024), (70, 32), (300, 1024)])
def test_alternatives_do_not_change_a_score(cuda, M, rows):
    """score_prompt with alternatives and without: both from the product in 32 bits, so both within what
    the head's own test allows (2e-4), the rank and the alternatives exactly those of that product."""
    N, K = 5120, 512
    g = torch.Generator(device=cuda).manual_seed(M + 1)
    hidden = torch.randn(M, K, device=cuda, generator=g).bfloat16()
    w = (torch.randn(N, K, device=cuda, generator=g) * 0.2).bfloat16()
    ids = torch.randint(N, (M,), device=cuda, generator=g)
    wq, ws = P.fp8_target_lmhead.pack_fp8_block(w)
    a = LP.score_prompt(hidden, wq, ws, ids)
    b = LP.score_prompt(hidden, wq, ws, ids, top_k=6, rows_at_once=rows)
    qx, xs = P.fused_silu_mul_quant.per_token_group_quant_fp8(hidden)
    y = torch.cat([P.fp8_block_gemm.fp8_block_gemm(qx[i:i + rows], wq, xs[i:i + rows], ws, out_dtype=torch.float32,
                                                   packed=True) for i in range(0, M, rows)])
    want = torch.log_softmax(y.double(), 1)
    at = want.gather(1, ids[:, None])[:, 0]
    for r in (a, b):
        assert (r.logprob - at).abs().max() <= 2e-4
        assert (r.entropy + (want.exp() * want).sum(1)).abs().max() <= 2e-4 * (1 + y.abs().max().item())
        assert (r.logsumexp - torch.logsumexp(y.double(), 1)).abs().max() <= 2e-4
    assert torch.equal(b.rank, 1 + (y > y.gather(1, ids[:, None])).sum(1))
    assert torch.equal(b.top_ids, torch.sort(y, dim=1, descending=True, stable=True).indices[:, :6])
    assert (b.top_logprobs - want.gather(1, b.top_ids)).abs().max() <= 2e-4


@pytest.mark.parametrize("M", [3, 300])
def test_inside_a_graph_on_new_inputs(cuda, M):
    """Both log probability calls captured in one CUDA graph (the head's merge is a programmatic dependent
    of its product) and replayed after their inputs have changed: what the calls give outside it."""
    from test_fp8_block_gemm_gpu import operands
    qx, wq, xs, ws = operands(M, 5000, 512, cuda, seed=1)
    x, ids = logits(M, 20000, torch.bfloat16, cuda, seed=1)
    ids = ids % 5000

    def both():
        return [*LP.token_logprobs(x, ids, top_k=5), *LP.fp8_head_logprobs(qx, wq, xs, ws, ids)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        both()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = both()
    for seed in (2, 3):
        for old, new in zip((qx, wq, xs, ws), operands(M, 5000, 512, cuda, seed=seed)):
            old.copy_(new)
        x.copy_(logits(M, 20000, torch.bfloat16, cuda, seed=seed)[0])
        ids.copy_((ids + 1) % 5000)
        for t in got:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        for u, v in zip(got, both()):
            assert torch.equal(u, v)
