"""A wait of the 8-bit attention kernels that ran out is an error for the caller (the extension is a fake here)."""

import contextlib
from types import SimpleNamespace

import pytest
import torch

from verl_omni_b200.ops import paged8


def _fake(monkeypatch, codes):
    calls = []

    def error(reset):
        calls.append("read" if not reset else "read and reset")
        return codes.pop(0) if codes else 0

    monkeypatch.setattr(paged8, "_ext", lambda: SimpleNamespace(paged8_error=error))
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: SimpleNamespace(synchronize=lambda: calls.append("wait")))
    return calls


def test_code_is_raised_once_and_read_behind_the_stream(monkeypatch):
    calls = _fake(monkeypatch, [44])
    with pytest.raises(RuntimeError, match="code 44"):
        paged8.raise_on_timeout("cuda")
    paged8.raise_on_timeout(torch.device("cuda", 0))
    assert calls == ["wait", "read and reset"] * 2
    paged8.raise_on_timeout("cpu")
    assert len(calls) == 4


def test_rollout_on_the_8_bit_cache_raises(monkeypatch):
    from verl_omni_b200.models.moe_llm import MoEConfig, MoELLM
    from verl_omni_b200.utils.dataproto import DataProto
    from verl_omni_b200.workers.rollout import llm_rollout

    torch.manual_seed(0)
    m = MoELLM(MoEConfig.tiny()).eval()
    batch = DataProto({"input_ids": torch.randint(0, 500, (2, 5))}, {})
    seen = []

    def check(device):
        seen.append(torch.device(device).type)
        raise RuntimeError("a wait ran out")

    monkeypatch.setattr(llm_rollout, "raise_on_timeout", check, raising=False)
    kw = dict(max_new_tokens=2, device=torch.device("cpu"))
    with pytest.raises(RuntimeError, match="ran out"):
        llm_rollout.LLMRolloutEngine(m, kv_cache_dtype="fp8_e4m3", **kw).generate(batch)
    assert seen == ["cpu"]
    llm_rollout.LLMRolloutEngine(m, **kw).generate(batch)  # no 8-bit cache, nothing to ask
    assert seen == ["cpu"]
