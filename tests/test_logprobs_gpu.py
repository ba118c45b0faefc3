"""token_logprobs, fp8_head_logprobs and score_prompt against the formulas in 64 bits.

Tolerance. Each exponential is off by a few units of 2^-23 and, through its argument's rounding, by
|d| 2^-23 of itself (d = x - max, and e^d <= 1: at most 2^-23 e^-1 of the sum's largest term); sums of
up to a few hundred terms per thread in fp32 are off by at most 1e3 2^-24 < 6e-5 of themselves, all
added up one way. So ln S is off by at most 7e-5, W / S by 7e-5 (1 + |W / S|), and results near a
logit of size |x| by |x| 2^-23 more. Ranks, ids and the positions of NaN and -inf are exact. For the
head the logits themselves are off by (K + K/64 + 2) 2^-23 of their sum of magnitudes at most; 2e-4
covers that at these sizes when it does not add up one way."""
from __future__ import annotations

import math

import pytest
import torch

from conftest import load_pkg
from test_fp8_block_gemm_gpu import operands, reference

pytestmark = pytest.mark.gpu
P = load_pkg()
LP = P.logprobs
INF = float("inf")
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def formula(x, ids):
    """logprob, entropy, lse, rank of rows x in 64 bits, with the documented special rows."""
    x = x.double()
    V = x.shape[1]
    m = x.amax(1, keepdim=True)
    empty = m[:, 0] == -INF
    bad = torch.isnan(x).any(1) | (x == INF).any(1)
    d = x - torch.where(empty[:, None], torch.zeros_like(m), m)
    e = torch.exp(d)
    S = e.sum(1)
    W = torch.where(e > 0, e * d, torch.zeros_like(d)).sum(1)
    inside = (ids >= 0) & (ids < V)
    xt = x.gather(1, ids.clamp(0, V - 1)[:, None])
    lse = m[:, 0] + torch.log(S)
    logprob = (xt - m)[:, 0] - torch.log(S)
    entropy = torch.log(S) - W / S
    logprob[empty], entropy[empty], lse[empty] = -INF, 0.0, -INF
    for t in (logprob, entropy, lse):
        t[bad] = math.nan
    logprob[~inside] = math.nan
    rank = torch.where(inside, 1 + (x > xt).sum(1), torch.zeros_like(ids))
    return logprob, entropy, lse, rank, W / S


def top_formula(x, k):
    """The k first ids by (value descending, id ascending), NaN before everything."""
    x = torch.where(torch.isnan(x), torch.full_like(x, INF), x.double()) + 0.0 if x.dtype == torch.float64 else x.double()
    return torch.sort(torch.where(torch.isnan(x), torch.full_like(x, math.inf), x), dim=1, descending=True,
                      stable=True).indices[:, :k]


def close(got, want, tol):
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]) and torch.equal(torch.isinf(got), inf)
    ok = torch.isfinite(want)
    tol = tol.expand_as(want) if torch.is_tensor(tol) else torch.full_like(want, tol)
    d = (got - want).abs()
    assert (d[ok] <= tol[ok]).all(), f"worst {(d[ok] / tol[ok]).max().item():.3f} of the bound"


def check(x, ids, k):
    r = LP.token_logprobs(x, ids, top_k=k)
    ids = ids.long()
    logprob, entropy, lse, rank, mean = formula(x, ids)
    finite = torch.where(torch.isfinite(x), x.double().abs(), torch.zeros_like(x, dtype=torch.float64)).amax(1)
    t = 7e-5 + finite * 2.0 ** -22
    close(r.logprob, logprob, t)
    close(r.logsumexp, lse, t)
    close(r.entropy, entropy, 2 * t * (1 + mean.abs().nan_to_num(0, 0, 0)))
    assert torch.equal(r.rank, rank)
    assert r.top_ids.shape == r.top_logprobs.shape == (x.shape[0], k)
    if k:
        want = top_formula(x, k)
        assert torch.equal(r.top_ids, want)
        at = formula(x, ids.clamp(0, x.shape[1] - 1))
        xt = x.double().gather(1, want)
        top = xt - at[2][:, None]
        top[torch.isinf(at[2])] = -INF
        top[torch.isnan(at[2])] = math.nan
        close(r.top_logprobs, top, t[:, None])
    return r


def logits(M, V, dtype, dev, seed=0, scale=3.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = (torch.randn(M, V, device=dev, generator=g) * scale).to(dtype)
    return x, torch.randint(V, (M,), device=dev, generator=g)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,V,k", [(1, 1, 1), (3, 2, 2), (2, 7, 7), (5, 8, 3), (4, 31, 20), (3, 64, 64), (2, 100, 5), (7, 1000, 20),
                                   (9, 4099, 33), (5, 8192, 64), (3, 50001, 8), (1, 151936, 5), (2, 151936, 0),
                                   (65, 32000, 20), (150, 20000, 10), (300, 5003, 4), (700, 1031, 2), (3000, 257, 1)])
def test_sizes(cuda, M, V, k, dtype):
    x, ids = logits(M, V, dtype, cuda, seed=V)
    check(x, ids, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [5, 700, 9001, 151936])
def test_ties_take_the_lowest_id(cuda, dtype, V):
    k = min(V, 40)
    g = torch.Generator(device=cuda).manual_seed(V)
    few = torch.randint(-3, 3, (4, V), device=cuda, generator=g).to(dtype)          # many equal values
    ids = torch.randint(V, (4,), device=cuda, generator=g)
    few[1] = 2.0                                                                    # nothing but equal values
    few[2] = -0.0
    few[2, ::2] = 0.0                                                               # zeros of both signs are equal
    check(few, ids, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [33, 5000, 151936])
def test_order_of_the_row_does_not_matter(cuda, dtype, V):
    """Ascending, descending, and everything large in one stretch: the largest arrive last, first, together."""
    x, ids = logits(3, V, dtype, cuda, seed=4)
    x[0] = x[0].sort().values
    x[1] = x[1].sort(descending=True).values
    a = V // 3
    x[2, a:a + max(1, V // 50)] += 40.0
    check(x, ids, min(V, 64))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [9, 3001, 151936])
def test_masks(cuda, dtype, V):
    """-inf and the type's lowest value: almost everywhere, everywhere, on the token itself; a first stretch
    masked and the rest far below zero; one token left, at either end."""
    x, _ = logits(8, V, dtype, cuda, seed=9)
    low = torch.finfo(dtype).min
    x[0, V // 2 + 1:] = -INF
    x[1] = -INF
    x[2] = low
    x[3] = -INF
    x[3, V - 1] = -5.0
    x[4] = low
    x[4, 0] = 3.0
    x[5, :] -= 300.0
    x[5, :V // 2] = -INF
    x[6] = -INF
    x[6, V // 3] = low
    x[7, ::2] = low
    ids = torch.tensor([V - 1, 0, V - 1, V - 1, 1, V - 1, V // 3, 0], device=cuda)
    check(x, ids, min(V, 20))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [12, 70001])
def test_nan_inf_and_large(cuda, dtype, V):
    x, ids = logits(6, V, dtype, cuda, seed=2)
    x[0, V - 2] = math.nan
    x[1, 1] = INF
    x[2] = math.nan
    x[3] = torch.where(torch.arange(V, device=cuda) % 2 == 0, 60000.0, -60000.0).to(dtype)
    x[4] *= 5000.0
    ids[3] = 1
    logprob, entropy, lse, rank, _ = formula(x, ids)
    r = LP.token_logprobs(x, ids, top_k=3)
    assert torch.isnan(r.logprob[:3]).all() and torch.isnan(r.entropy[:3]).all() and torch.isnan(r.logsumexp[:3]).all()
    assert r.top_ids[0, 0] == V - 2 and r.top_ids[1, 0] == 1 and r.top_ids[2].tolist() == [0, 1, 2]
    assert torch.isnan(r.top_logprobs[:3]).all()
    check(x[3:], ids[3:], 3)


def test_token_ids(cuda):
    """int32 ids, strided ids, ids outside the vocabulary, which are neither read nor counted."""
    x, ids = logits(6, 5000, torch.bfloat16, cuda, seed=1)
    check(x, ids.int(), 2)
    check(x, torch.stack([ids, ids * 0], 1)[:, 0], 2)
    ids[0], ids[1], ids[2], ids[3] = -1, 5000, -(1 << 40), 1 << 40
    r = check(x, ids, 2)
    assert torch.isnan(r.logprob[:4]).all() and (r.rank[:4] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(cuda, dtype):
    """Rows at odd offsets inside a larger tensor whose neighbours are NaN."""
    for V, off, gap in ((1001, 1, 3), (4096, 3, 1), (30000, 5, 8), (30000, 8, 8)):
        big = torch.full((5, V + off + gap), math.nan, dtype=dtype, device=cuda)
        x, ids = logits(5, V, dtype, cuda, seed=off)
        big[:, off:off + V] = x
        check(big[:, off:off + V], ids, 7)


def test_one_row_stretched_over_more_than_32_bits(cuda):
    """Row offsets past 2^32 elements."""
    V = 4000
    big = torch.empty((1 << 31) + (1 << 31) + 3 * V, dtype=torch.bfloat16, device=cuda)
    x = torch.as_strided(big, (3, V), (1 << 31, 1))
    y, ids = logits(3, V, torch.bfloat16, cuda)
    x.copy_(y)
    check(x, ids, 4)


def test_empty_stream_and_repeat(cuda):
    x, ids = logits(40, 30000, torch.float32, cuda)
    r = LP.token_logprobs(x[:0], ids[:0], top_k=3)
    assert r.logprob.shape == (0,) and r.top_ids.shape == (0, 3)
    a = LP.token_logprobs(x, ids, top_k=9)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = LP.token_logprobs(x.clone(), ids, top_k=9)
    torch.cuda.current_stream().wait_stream(s)
    for _ in range(3):
        for u, v in zip(a, LP.token_logprobs(x, ids, top_k=9)):
            assert torch.equal(u, v)
    for u, v in zip(a, b):
        assert torch.equal(u, v)


def test_refusals(cuda):
    x, ids = logits(4, 100, torch.float32, cuda)
    f = LP.token_logprobs
    for call in (lambda: f(x.double(), ids), lambda: f(x[0], ids), lambda: f(x.t(), ids), lambda: f(x, ids[:3]),
                 lambda: f(x, ids.float()), lambda: f(x, ids.cpu()), lambda: f(x, ids, top_k=-1),
                 lambda: f(x, ids, top_k=65), lambda: f(x[:, :5], ids, top_k=6), lambda: f(x[:, :0], ids),
                 lambda: f(x[:1].expand(4, 100), ids)):
        with pytest.raises(ValueError):
            call()


def check_head(ops, ids, packed_w=None):
    qx, wq, xs, ws = ops
    r = LP.fp8_head_logprobs(qx, wq if packed_w is None else packed_w, xs, ws, ids, packed=packed_w is not None)
    y, _ = reference(qx, wq, xs, ws)
    logprob, entropy, lse, _, mean = formula(y, ids.long())
    close(r.logprob, logprob, 2e-4)
    close(r.logsumexp, lse, 2e-4)
    close(r.entropy, entropy, 2e-4 * (1 + mean.abs()))
    assert P._lib.score().b200_score_error(1) == 0
    return r


@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (1, 128, 128), (3, 1000, 2560), (8, 5000, 400), (64, 2560, 512),
                                   (65, 130, 144), (129, 257, 272), (200, 3000, 640), (500, 50001, 144),
                                   (1030, 777, 1280), (2, 151936, 256)])
def test_head(cuda, M, N, K):
    ops = operands(M, N, K, cuda, seed=N)
    g = torch.Generator(device=cuda).manual_seed(1)
    check_head(ops, torch.randint(N, (M,), device=cuda, generator=g))


@pytest.mark.parametrize("M", [5, 300])
def test_head_pack_ids_and_sharp_rows(cuda, M):
    """The strip pack; ids at both ends and outside; rows whose logits span hundreds."""
    N, K = 1040, 384
    qx, wq, xs, ws = operands(M, N, K, cuda, seed=6)
    xs[2] *= 40.0
    xs[3] = 0.0
    ids = torch.randint(N, (M,), device=cuda, dtype=torch.int32)
    ids[0], ids[1], ids[2], ids[3], ids[4] = 0, N - 1, -1, 7, N
    y, _ = reference(qx, wq, xs, ws)
    pack = P.fp8_target_lmhead._strip_swizzle(wq)
    r = LP.fp8_head_logprobs(qx, pack, xs, ws, ids, packed=True)
    q = LP.fp8_head_logprobs(qx, wq, xs, ws, ids)
    for u, v in zip(r, q):
        assert torch.equal(u.nan_to_num(7.0), v.nan_to_num(7.0))
    assert torch.isnan(r.logprob[[2, 4]]).all() and not torch.isnan(r.entropy).any()
    logprob, entropy, lse, _, mean = formula(y, ids.long())
    t = 2e-4 + y.abs().amax(1) * 1e-5
    close(r.logprob, logprob, t)
    close(r.logsumexp, lse, t)
    close(r.entropy, entropy, t * (1 + mean.abs()))
    assert abs(r.entropy[3].item() - math.log(N)) < 1e-4


def test_head_nan_rows(cuda):
    qx, wq, xs, ws = operands(130, 600, 256, cuda, seed=3)
    qx.view(torch.uint8)[1, 3] = 0x7F
    xs[2, 1] = INF
    ids = torch.zeros(130, dtype=torch.int64, device=cuda)
    r = LP.fp8_head_logprobs(qx, wq, xs, ws, ids)
    for t in r:
        assert torch.isnan(t[1:3]).all() and torch.isfinite(t[0]) and torch.isfinite(t[3:]).all()


def test_head_repeatable_and_empty(cuda):
    ops = operands(333, 9000, 640, cuda)
    ids = torch.arange(333, device=cuda)
    a = LP.fp8_head_logprobs(*ops, ids)
    for _ in range(4):
        for u, v in zip(a, LP.fp8_head_logprobs(*ops, ids)):
            assert torch.equal(u, v)
    qx, wq, xs, ws = ops
    assert LP.fp8_head_logprobs(qx[:0], wq, xs[:0], ws, ids[:0]).logprob.shape == (0,)
    with pytest.raises(ValueError):
        LP.fp8_head_logprobs(*ops, ids[:5])


@pytest.mark.parametrize("M,rows", [(1, 1024), (70, 32), (130, 1024)])
def test_score_prompt(cuda, M, rows):
    """Hidden states to log probabilities through the packed head: both forms agree with each other and with
    the quantized operands' formula, the form with alternatives on bf16 logits."""
    N, K = 5120, 512
    g = torch.Generator(device=cuda).manual_seed(M)
    hidden = torch.randn(M, K, device=cuda, generator=g).bfloat16()
    w = (torch.randn(N, K, device=cuda, generator=g) * 0.1).bfloat16()
    ids = torch.randint(N, (M,), device=cuda, generator=g)
    wq, ws = P.fp8_target_lmhead.pack_fp8_block(w)
    a = LP.score_prompt(hidden, wq, ws, ids)
    b = LP.score_prompt(hidden, wq, ws, ids, top_k=6, rows_at_once=rows)
    qx, xs = P.fused_silu_mul_quant.per_token_group_quant_fp8(hidden)
    y, _ = reference(qx, P.fp8_target_lmhead.unpack_fp8_block(wq), xs, ws)
    logprob, entropy, lse, _, mean = formula(y, ids)
    close(a.logprob, logprob, 2e-4)
    close(a.entropy, entropy, 2e-4 * (1 + mean.abs()))
    near = 2.0 ** -8 * y.abs().amax(1) + 2e-4                # bf16's rounding of every logit
    close(b.logprob, logprob, 2 * near)
    close(b.logsumexp, lse, 2 * near)
    assert (b.top_ids[:, 0] == y.bfloat16().float().argmax(1)).float().mean() > 0.9 and b.top_ids.shape == (M, 6)
    with pytest.raises(ValueError):
        LP.score_prompt(hidden, wq, ws, ids, top_k=2, rows_at_once=0)


def test_target_head_scores_its_prompt(cuda):
    """Fp8TargetHead.score is score_prompt on the head's own pack; a scoring product above the decode path's
    64 rows agrees with the decode path's logits row for row."""
    N, K, M = 2048, 256, 90
    g = torch.Generator(device=cuda).manual_seed(5)
    w = (torch.randn(N, K, device=cuda, generator=g) * 0.1).bfloat16()
    head = P.fp8_target_lmhead.Fp8TargetHead(None, w)
    hidden = torch.randn(M, K, device=cuda, generator=g).bfloat16()
    ids = torch.randint(N, (M,), device=cuda, generator=g)
    a, b = head.score(hidden, ids), LP.score_prompt(hidden, head.wq, head.ws, ids)
    for u, v in zip(a, b):
        assert torch.equal(u, v)
    qx, xs = P.fused_silu_mul_quant.per_token_group_quant_fp8(hidden)
    y = P.fp8_block_gemm.fp8_block_gemm(qx, head.wq, xs, head.ws, packed=True)
    decode = torch.cat([P.fp8_target_lmhead.gemm_fp8_block(hidden[i:i + 30].contiguous(), head.wq, head.ws)
                        for i in range(0, M, 30)])
    # both round the same fp32 sums, added in another order, to bf16: at most one step apart
    assert ((y.float() - decode.float()).abs() <= 2.0 ** -7 * decode.float().abs() + 1e-5).all()
