"""Scoring calls belong to their tensors' device, whichever device is current: checked on the host with
a stand-in for the current device, since the launches themselves need GPUs."""
from __future__ import annotations

import types

import pytest
import torch

from conftest import load_pkg

P = load_pkg()
LP = P.logprobs


class CurrentDevice:
    """torch.cuda.device on a machine of several devices: cuda:0 is current at first."""

    now = 0

    def __init__(self, device):
        self.index = device if isinstance(device, int) else torch.device(device).index

    def __enter__(self):
        self.before, CurrentDevice.now = CurrentDevice.now, self.index

    def __exit__(self, *exc):
        CurrentDevice.now = self.before


@pytest.fixture
def current(monkeypatch):
    monkeypatch.setattr(CurrentDevice, "now", 0)
    monkeypatch.setattr(torch.cuda, "device", CurrentDevice)
    return CurrentDevice


@pytest.mark.parametrize("top_k", [0, 3])
def test_score_prompt_runs_on_its_tensors_device(monkeypatch, current, top_k):
    """Every launch of score_prompt, the quantiser's too, is made with the hidden states' device current,
    and so on that device's current stream; afterwards the device is what it was."""
    seen = []

    def stub(name, result):
        def call(*args, **kwargs):
            seen.append((name, current.now))
            return result(*args)
        return call

    dev = torch.device("cuda:1")
    hidden = types.SimpleNamespace(device=dev, is_cuda=True, shape=(5, 128), dtype=torch.bfloat16, ndim=2)
    row = torch.zeros(5, 8)
    monkeypatch.setattr(P.fused_silu_mul_quant, "per_token_group_quant_fp8", stub("quant", lambda x: (row, row)))
    monkeypatch.setattr(LP, "fp8_head_logprobs", stub("head", lambda *a: "head"))
    monkeypatch.setattr(LP, "fp8_block_gemm", stub("product", lambda *a: row))
    monkeypatch.setattr(LP, "token_logprobs", stub("logprobs", lambda *a: LP.TokenLogprobs(*[row] * 6)))
    monkeypatch.setattr(LP, "_ids", lambda what, ids, M, device: ids)
    real_empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, device=None, **k: real_empty(*a, **k))
    LP.score_prompt(hidden, row, row, torch.zeros(5, dtype=torch.int64), top_k=top_k, rows_at_once=4)
    names = ["quant", "head"] if top_k == 0 else ["quant"] + ["product", "logprobs"] * 2
    assert seen == [(n, 1) for n in names]
    assert current.now == 0


def test_score_prompt_refuses_host_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        LP.score_prompt(torch.zeros(2, 128), torch.zeros(16, 128), torch.zeros(1, 1), torch.zeros(2, dtype=torch.int64))


@pytest.mark.parametrize("index", [0, 1])
def test_debug_check_looks_at_the_launch_device(monkeypatch, current, index):
    """With B200_LMHEAD_CHECK=1 a call waits for its own device's stream and reads that device's error word."""
    seen = []

    def note(name, result):
        return lambda *a: (seen.append((name, current.now)), result)[1]

    stream = types.SimpleNamespace(synchronize=note("wait", None))
    lib = types.SimpleNamespace(b200_score_error=note("word", 0))
    monkeypatch.setattr(P._lib, "_CHECK", True)
    monkeypatch.setattr(P._lib, "score", lambda: lib)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: stream)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current.now, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 100 + i, raising=False)
    P._lib.launch("call", lambda *a: (seen.append(("launch", current.now)), seen.append(a))[0] or 0,
                  torch.device("cuda", index), 7)
    assert seen == [("launch", index), (7, 100 + index), ("wait", index), ("word", index)]
    assert current.now == 0
