"""fp8_block_gemm against the formula in 64 bits.

Tolerance. The products of two e4m3 codes are exact in fp32. A sum of K of them in fp32, in any order
and whether each addition rounds or truncates, is off by at most K 2^-23 of the sum of magnitudes
A = xs ws sum |qx| |wq|; scaling and adding the K/128 groups adds 2 K/128 more roundings, so
|y - ref| <= (K + K/64 + 2) 2^-23 A before the output's own rounding (2^-8 |ref| for bf16, 2^-11 for
f16, plus f16's smallest step 2^-24). That bound allows errors that all add up one way; the 2-norm of
the f32 outputs' error, where they do not, is held to 1e-5 of the reference's."""
from __future__ import annotations

import pytest
import torch

from conftest import load_pkg

pytestmark = pytest.mark.gpu
P = load_pkg()
G = P.fp8_block_gemm
FP8 = torch.float8_e4m3fn
BLK = 128
U_OUT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def operands(M, N, K, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    kb, nb = -(-K // BLK), -(-N // BLK)
    qx = (torch.randn(M, K, device=dev, generator=g) * 120).clamp(-448, 448).to(FP8)
    wq = (torch.randn(N, K, device=dev, generator=g) * 120).clamp(-448, 448).to(FP8)
    xs = torch.rand(M, kb, device=dev, generator=g) * 0.02 + 1e-3
    ws = torch.rand(nb, kb, device=dev, generator=g) * 2e-4 + 1e-5
    return qx, wq, xs, ws


def reference(qx, wq, xs, ws):
    """(the product, the sum of magnitudes), in 64 bits."""
    K, N = qx.shape[1], wq.shape[0]
    x = qx.double() * xs.double().repeat_interleave(BLK, 1)[:, :K]
    w = wq.double() * ws.double().repeat_interleave(BLK, 1)[:, :K].repeat_interleave(BLK, 0)[:N]
    return x @ w.t(), x.abs() @ w.abs().t()


def check(y, qx, wq, xs, ws):
    ref, mag = reference(qx, wq, xs, ws)
    K = qx.shape[1]
    tol = (K + K / 64 + 2) * 2.0 ** -23 * mag + U_OUT[y.dtype] * ref.abs() + (2.0 ** -24 if y.dtype == torch.float16 else 0)
    d = (y.double() - ref).abs()
    assert torch.isfinite(d).all()
    worst = (d / tol.clamp(min=1e-300)).max().item()
    assert (d <= tol).all(), f"worst error {worst:.2f} of the bound"
    if y.dtype == torch.float32:
        rel = ((y.double() - ref).norm() / ref.norm()).item()
        assert rel < 1e-5, f"2-norm {rel:.2e}"
    assert P._lib.score().b200_score_error(1) == 0


SHAPES = [(1, 1, 16), (1, 128, 128), (2, 24, 8192), (5, 2560, 2560), (16, 640, 512), (31, 8, 16), (63, 264, 640),
          (64, 1000, 2560), (65, 130, 144), (127, 129, 272), (128, 256, 384), (129, 257, 400), (255, 640, 1280),
          (257, 511, 2560), (300, 1000, 1360), (513, 2049, 528), (1000, 640, 512), (2050, 2560, 1024),
          (130, 18944, 256), (3, 151936, 128)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_sizes(cuda, M, N, K, dtype):
    ops = operands(M, N, K, cuda, seed=M + N)
    y = G.fp8_block_gemm(*ops, out_dtype=dtype)
    assert y.shape == (M, N) and y.dtype == dtype
    check(y, *ops)


@pytest.mark.parametrize("M,N,K", [(1, 128, 128), (7, 16, 256), (64, 640, 2560), (100, 1040, 384), (300, 2560, 1280),
                                   (1024, 4096, 256)])
def test_strip_pack_equals_row_major(cuda, M, N, K):
    """The same codes in the head's strip pack give the same bits."""
    qx, wq, xs, ws = operands(M, N, K, cuda, seed=3)
    pack = P.fp8_target_lmhead._strip_swizzle(wq)
    a = G.fp8_block_gemm(qx, wq, xs, ws, out_dtype=torch.float32)
    b = G.fp8_block_gemm(qx, pack, xs, ws, out_dtype=torch.float32, packed=True)
    assert torch.equal(a, b)
    check(b, qx, wq, xs, ws)


@pytest.mark.parametrize("M,N,K", [(9, 200, 272), (200, 520, 656), (300, 1030, 1296)])
def test_strides_and_neighbours(cuda, M, N, K):
    """Strided rows whose gaps hold e4m3 NaN, group-major and gapped scales, an output inside a larger
    one at an odd offset: nothing outside is read into the result or written."""
    qx, wq, xs, ws = operands(M, N, K, cuda, seed=11)
    xb = torch.full((M + 2, K + 48), 0x7F, dtype=torch.uint8, device=cuda).view(FP8)
    wb = torch.full((N + 2, K + 16), 0x7F, dtype=torch.uint8, device=cuda).view(FP8)
    xb[1:M + 1, 16:16 + K] = qx
    wb[1:N + 1, :K] = wq
    xst = torch.full((xs.shape[1], M + 5), float("nan"), device=cuda)
    xst[:, 2:M + 2] = xs.t()
    wsb = torch.full((ws.shape[0], ws.shape[1] + 3), float("nan"), device=cuda)
    wsb[:, 1:-2] = ws
    for dtype, off in ((torch.bfloat16, 1), (torch.float32, 3), (torch.float16, 8)):
        big = torch.full((M + 2, N + 24), -77.0, dtype=dtype, device=cuda)
        view = big[1:M + 1, off:off + N]
        got = G.fp8_block_gemm(xb[1:M + 1, 16:16 + K], wb[1:N + 1, :K], xst[:, 2:M + 2].t(), wsb[:, 1:-2], out=view)
        assert got.data_ptr() == view.data_ptr()
        check(view, qx, wq, xs, ws)
        view.fill_(-77.0)
        assert (big == -77.0).all()


@pytest.mark.parametrize("M", [3, 200, 700])
def test_extreme_operands(cuda, M):
    """A zero scale, saturated codes, a NaN code in one activation row and in one weight row."""
    N, K = 300, 384
    qx, wq, xs, ws = operands(M, N, K, cuda, seed=5)
    qx[0] = 448.0
    wq[1] = -448.0
    xs[1] = 0.0
    check(G.fp8_block_gemm(qx, wq, xs, ws, out_dtype=torch.float32), qx, wq, xs, ws)
    qx.view(torch.uint8)[2, 7] = 0x7F
    wq.view(torch.uint8)[5, 200] = 0xFF
    y = G.fp8_block_gemm(qx, wq, xs, ws)
    nan = torch.isnan(y)
    assert nan[2].all() and nan[:, 5].all()
    nan[2] = False
    nan[:, 5] = False
    assert not nan.any()


def test_empty_and_repeatable(cuda):
    qx, wq, xs, ws = operands(333, 1000, 2560, cuda)
    assert G.fp8_block_gemm(qx[:0], wq, xs[:0], ws).shape == (0, 1000)
    a = G.fp8_block_gemm(qx, wq, xs, ws, out_dtype=torch.float32)
    for _ in range(5):
        assert torch.equal(a, G.fp8_block_gemm(qx, wq, xs, ws, out_dtype=torch.float32))


@pytest.mark.parametrize("M,N", [(7, 2560), (600, 2560)])
def test_other_stream_and_graph(cuda, M, N):
    """On a side stream behind its producer, and replayed from a CUDA graph on new inputs."""
    ops = operands(M, N, 1280, cuda, seed=1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        qx = ops[0].clone()
        y = G.fp8_block_gemm(qx, *ops[1:], out_dtype=torch.float32)
    torch.cuda.current_stream().wait_stream(s)
    check(y, *ops)
    out = torch.empty(M, N, device=cuda)
    x = ops[0].clone()
    G.fp8_block_gemm(x, *ops[1:], out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        G.fp8_block_gemm(x, *ops[1:], out=out)
    fresh = operands(M, N, 1280, cuda, seed=2)[0]
    x.copy_(fresh)
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    check(out, fresh, *ops[1:])


def test_output_offsets_past_32_bits(cuda):
    """More than 2^32 bytes and 2^31 elements of output: the last rows are where they belong."""
    M, N, K = 14400, 151936, 16
    qx, wq, xs, ws = operands(M, N, K, cuda, seed=8)
    y = G.fp8_block_gemm(qx, wq, xs, ws)
    assert y.numel() > 1 << 31
    for r in (slice(0, 3), slice(7000, 7003), slice(M - 3, M)):
        check(y[r], qx[r], wq, xs[r], ws)


def test_refusals(cuda):
    qx, wq, xs, ws = operands(8, 256, 256, cuda)
    f = G.fp8_block_gemm
    bad = [
        lambda: f(qx.float(), wq, xs, ws), lambda: f(qx, wq.view(torch.uint8), xs, ws), lambda: f(qx[0], wq, xs, ws),
        lambda: f(qx[:, :128], wq, xs, ws), lambda: f(qx, wq, xs[:, :1], ws), lambda: f(qx, wq, xs.double(), ws),
        lambda: f(qx, wq, xs, ws[:1]), lambda: f(qx, wq, xs, ws.t().contiguous().t()),
        lambda: f(qx[:, :24].contiguous(), wq[:, :24].contiguous(), xs[:, :1], ws[:, :1]),
        lambda: f(qx[:, 8:136], wq[:, :128], xs[:, :1], ws[:, :1]),
        lambda: f(qx.t().contiguous().t(), wq, xs, ws), lambda: f(qx, wq[:0], xs, ws[:0]),
        lambda: f(qx, wq, xs, ws, out_dtype=torch.float64), lambda: f(qx, wq, xs, ws, out=torch.empty(8, 255, device=cuda)),
        lambda: f(qx, wq, xs, ws, out=torch.empty(256, 8, device=cuda).t()),
        lambda: f(qx, wq, xs, ws, out=torch.empty(8, 256)),
        lambda: f(qx, wq[:250], xs, ws, packed=True), lambda: f(qx, wq.cpu(), xs, ws),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_streams_side_by_side(cuda):
    """Products of every launch form, the decode head and the scoring head on two streams at once: each takes
    whole SMs, none waits for another's, and every result is what it is alone."""
    sizes = [(5, 2560, 2560), (300, 4096, 1280), (64, 640, 2560), (700, 2560, 512)]
    ops = [operands(*s, cuda, seed=i) for i, s in enumerate(sizes)]
    w = (torch.randn(4096, 512, device=cuda) * 0.05).bfloat16()
    hq, hs = P.fp8_target_lmhead.pack_fp8_block(w)
    x = torch.randn(40, 512, device=cuda).bfloat16()
    ids = torch.arange(300, device=cuda)

    def everything():
        out = [G.fp8_block_gemm(*o, out_dtype=torch.float32) for o in ops]
        out += list(P.logprobs.fp8_head_logprobs(*ops[1], ids))
        return out + list(P.fp8_target_lmhead.fp8_lmhead(x, hq, hs)[1:])

    alone = everything()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = [[], []]
    for _ in range(20):
        for s, r in zip(streams, results):
            with torch.cuda.stream(s):
                r.append(everything())
    torch.cuda.synchronize()
    for r in results:
        for got in r:
            assert all(torch.equal(u, v) for u, v in zip(alone, got))
    assert P._lib.score().b200_score_error(1) == 0


@pytest.mark.parametrize("M,N,K", [(33, 136, 20480), (200, 520, 16400)])
def test_long_k(cuda, M, N, K):
    ops = operands(M, N, K, cuda, seed=K)
    check(G.fp8_block_gemm(*ops, out_dtype=torch.float32), *ops)
