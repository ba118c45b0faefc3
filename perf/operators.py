"""The scoring operators' cases: the FP8 block-scaled matrix product for any number of tokens, the
log probabilities of given tokens (with entropy, rank and top alternatives), and the FP8 head
straight to log probabilities. Plain forms in 32 bits, the framework's calls where ``own``."""
import importlib

import torch

own = False

BLK = 128
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}

HIDDEN, VOCAB = 2560, 151936        # the head of this repository's benchmark


def listed():
    return [
        # a decode step's batch through a square projection of the hidden size: latency
        {"name": "gemm_decode", "op": "gemm", "m": 5, "n": HIDDEN, "k": HIDDEN, "out": "bf16"},
        # a short prompt, and sizes that no tile divides: rows, columns and a half-full last group
        {"name": "gemm_ragged", "op": "gemm", "m": 333, "n": 1000, "k": 1360, "out": "f16"},
        # a few hundred prompt tokens through the experts' gate and up projection, kept in 32 bits
        {"name": "gemm_gate_up_f32", "op": "gemm", "m": 512, "n": 1024, "k": HIDDEN, "out": "f32"},
        # a prefill chunk through a wide projection
        {"name": "gemm_prefill", "op": "gemm", "m": 8192, "n": 10240, "k": HIDDEN, "out": "bf16"},
        # the logits of a prompt's rows
        {"name": "gemm_head", "op": "gemm", "m": 1024, "n": VOCAB, "k": HIDDEN, "out": "bf16"},
        # one decoded token with its five alternatives: latency
        {"name": "logprobs_decode", "op": "logprobs", "m": 1, "v": VOCAB, "dtype": "bf16", "top": 5, "masked": 0.0},
        # a decode batch in 32 bits, the largest number of alternatives that servers offer
        {"name": "logprobs_batch_f32", "op": "logprobs", "m": 64, "v": VOCAB, "dtype": "f32", "top": 20, "masked": 0.0},
        # a small odd vocabulary under a grammar's mask
        {"name": "logprobs_masked", "op": "logprobs", "m": 777, "v": 50001, "dtype": "f16", "top": 8, "masked": 0.5},
        # a long prompt's rows
        {"name": "logprobs_prompt", "op": "logprobs", "m": 4096, "v": VOCAB, "dtype": "bf16", "top": 20, "masked": 0.0},
        # drafted tokens checked against the head
        {"name": "score_draft", "op": "score", "m": 8, "n": VOCAB, "k": HIDDEN},
        # a short text over a small odd vocabulary
        {"name": "score_ragged", "op": "score", "m": 500, "n": 50001, "k": 1040},
        # a long prompt's perplexity
        {"name": "score_prompt", "op": "score", "m": 4096, "n": VOCAB, "k": HIDDEN},
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["gemm", "logprobs", "score"])
    if op == "gemm":
        c = {"op": op, "m": _log_int(rng, 1, 8192), "n": _log_int(rng, 40, 16384), "k": 16 * _log_int(rng, 8, 640),
             "out": rng.choice(["bf16", "bf16", "f16", "f32"])}
        while c["m"] * c["n"] * c["k"] > 8192 * 10240 * HIDDEN:
            c["m"] = (c["m"] + 1) // 2
        return c
    if op == "logprobs":
        c = {"op": op, "m": _log_int(rng, 1, 4096), "v": _log_int(rng, 1000, VOCAB),
             "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "top": rng.choice([0, 1, 5, 20, rng.randint(2, 32)]),
             "masked": rng.choice([0.0, 0.0, 0.5, 0.9])}
        while c["m"] * c["v"] * SIZE[c["dtype"]] > 4096 * VOCAB * 2:
            c["m"] = (c["m"] + 1) // 2
        return c
    return {"op": op, "m": _log_int(rng, 1, 4096), "n": _log_int(rng, 1000, VOCAB), "k": 16 * _log_int(rng, 8, 160)}


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _pad128(t, dim):
    short = -t.shape[dim] % BLK
    if not short:
        return t
    shape = list(t.shape)
    shape[dim] = short
    return torch.cat([t, t.new_zeros(shape)], dim)


def _quantized(m, n, k, g):
    """Activations e4m3 with a scale for each row's group of 128, weights e4m3 with a scale for each
    block of 128 x 128, both quantized from normal values as a checkpoint and its user do."""
    kb, nb = -(-k // BLK), -(-n // BLK)
    x = _pad128(torch.randn(m, k, device=DEV, generator=g), 1).view(m, kb, BLK)
    x *= torch.exp(0.5 * torch.randn(m, 1, 1, device=DEV, generator=g))
    xs = x.abs().amax(2).clamp_(min=1e-10) / 448
    qx = (x / xs[:, :, None]).clamp_(-448, 448).to(torch.float8_e4m3fn).view(m, kb * BLK)[:, :k].contiguous()
    w = torch.randn(n, k, device=DEV, generator=g).mul_(0.02)
    w = _pad128(_pad128(w, 1), 0).view(nb, BLK, kb, BLK)
    ws = w.abs().amax((1, 3)).clamp_(min=1e-12) / 448
    wq = (w / ws[:, None, :, None]).clamp_(-448, 448).to(torch.float8_e4m3fn).view(nb * BLK, kb * BLK)[:n, :k].contiguous()
    return qx, wq, xs, ws


def prepare(case, seed):
    g = _gen(seed)
    state = dict(case)
    m = case["m"]
    if case["op"] == "logprobs":
        v = case["v"]
        x = torch.randn(m, v, device=DEV, generator=g).mul_(2.5)
        ids = torch.randint(v, (m,), device=DEV, generator=g)
        best = x.argmax(1)
        ids = torch.where(torch.rand(m, device=DEV, generator=g) < 0.6, best, ids)     # text is mostly likely tokens
        x = x.to(DT[case["dtype"]])
        if case["masked"]:
            gone = torch.rand(m, v, device=DEV, generator=g) < case["masked"]
            gone[:, :64] = False                   # what a mask leaves is never empty here
            gone.scatter_(1, ids[:, None], False)
            x.masked_fill_(gone, float("-inf"))
        state.update(logits=x, ids=ids)
        return state
    qx, wq, xs, ws = _quantized(m, case["n"], case["k"], g)
    state.update(qx=qx, wq=wq, xs=xs, ws=ws)
    if case["op"] == "score":
        state["ids"] = torch.randint(case["n"], (m,), device=DEV, generator=g)
    return state


def _package():
    return importlib.import_module("r9700-lru-expert-cache_b200")


def _plain_product(s):
    k, n = s["qx"].shape[1], s["wq"].shape[0]
    x = s["qx"].float() * s["xs"].repeat_interleave(BLK, 1)[:, :k]
    w = s["wq"].float() * s["ws"].repeat_interleave(BLK, 1)[:, :k].repeat_interleave(BLK, 0)[:n]
    return x @ w.t()


def _plain_stats(x, ids):
    """x float32: the log probability of ids, the entropy, the log of the sum of exponentials."""
    d = x - x.amax(1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(1)
    log_total = torch.log(total)
    weighted = torch.where(e > 0, e * d, torch.zeros_like(d)).sum(1)
    return (d.gather(1, ids[:, None])[:, 0] - log_total, log_total - weighted / total, x.amax(1) + log_total)


def _plain_top(x, k):
    """Ids of the k largest of each row, the lowest id first among equals: one whole number for value and id."""
    v = x.shape[1]
    bits = (x + 0.0).view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() << 32
    order += torch.arange(v - 1, -1, -1, device=x.device)
    return v - 1 - (torch.topk(order, k, dim=1).values & 0xFFFFFFFF)


def run(state):
    s, op = state, state["op"]
    if op == "gemm":
        if own:
            return _package().fp8_block_gemm.fp8_block_gemm(s["qx"], s["wq"], s["xs"], s["ws"], out_dtype=DT[s["out"]])
        return _plain_product(s).to(DT[s["out"]])
    if op == "score":
        if own:
            return list(_package().logprobs.fp8_head_logprobs(s["qx"], s["wq"], s["xs"], s["ws"], s["ids"]))
        return list(_plain_stats(_plain_product(s), s["ids"]))
    if own:
        r = _package().logprobs.token_logprobs(s["logits"], s["ids"], top_k=s["top"])
        out = [r.logprob, r.entropy, r.logsumexp, r.rank]
        return out + [r.top_ids, r.top_logprobs] if s["top"] else out
    x = s["logits"].float()
    logprob, entropy, lse = _plain_stats(x, s["ids"])
    rank = 1 + (x > x.gather(1, s["ids"][:, None])).sum(1)
    out = [logprob, entropy, lse, rank]
    if s["top"]:
        top = _plain_top(x, s["top"])
        out += [top, (x.gather(1, top) - x.amax(1, keepdim=True)) - (lse - x.amax(1))[:, None]]
    return out


def work(case):
    m = case["m"]
    if case["op"] == "logprobs":
        v, k = case["v"], case["top"]
        return {"bytes": m * v * SIZE[case["dtype"]] + m * (8 + 20 + 12 * k), "flops": 5 * m * v}
    n, k = case["n"], case["k"]
    kb, nb = -(-k // BLK), -(-n // BLK)
    operands = m * k + n * k + 4 * kb * (m + nb)
    if case["op"] == "gemm":
        return {"bytes": operands + m * n * SIZE[case["out"]], "flops": 2 * m * n * k}
    return {"bytes": operands + m * (8 + 12), "flops": 2 * m * n * k + 5 * m * n}


def _exact_logits(s, rows):
    """Rows of the product in 64 bits, group by group."""
    k = s["qx"].shape[1]
    y = torch.zeros(rows.stop - rows.start, s["wq"].shape[0], dtype=torch.float64, device=DEV)
    for b in range(s["xs"].shape[1]):
        c = slice(b * BLK, min(k, (b + 1) * BLK))
        part = s["qx"][rows, c].double() @ s["wq"][:, c].double().t()
        per_row = s["ws"][:, b].double().repeat_interleave(BLK)[:s["wq"].shape[0]]
        y += part * s["xs"][rows, b].double()[:, None] * per_row[None]
    return y


def _exact_stats(x, ids):
    p = torch.log_softmax(x, 1)
    entropy = -(torch.exp(p) * torch.where(torch.isinf(p), torch.zeros_like(p), p)).sum(1)
    return p, [p[torch.arange(x.shape[0], device=DEV), ids], entropy, torch.logsumexp(x, 1)]


def exact(case, seed):
    s = prepare(case, seed)
    m = case["m"]
    step = max(1, min(m, (1 << 28) // (case["v"] if case["op"] == "logprobs" else case["n"])))
    pieces = []
    for r0 in range(0, m, step):
        rows = slice(r0, min(m, r0 + step))
        if case["op"] == "gemm":
            pieces.append([_exact_logits(s, rows)])
        elif case["op"] == "score":
            pieces.append(_exact_stats(_exact_logits(s, rows), s["ids"][rows])[1])
        else:
            x = s["logits"][rows].double()
            p, found = _exact_stats(x, s["ids"][rows])
            if case["top"]:
                found.append(torch.topk(p, case["top"], dim=1).values)
            pieces.append(found)
    whole = [torch.cat(t) for t in zip(*pieces)]
    if case["op"] == "gemm":
        return whole[0]
    if case["op"] == "score":
        return whole
    return whole[:3] + [None] + ([None, whole[3]] if case["top"] else [])
