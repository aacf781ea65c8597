"""Rollout with grammar masks that allow nothing: ended rows are filled up, others are an error."""

import pytest
import torch

from verl_omni_b200.ops.logits import pack_allowed

EOS = 3


def _engine(**kw):
    from verl_omni_b200.models.moe_llm import MoEConfig, MoELLM
    from verl_omni_b200.workers.rollout.llm_rollout import LLMRolloutEngine

    torch.manual_seed(0)
    m = MoELLM(MoEConfig.tiny()).eval()
    return LLMRolloutEngine(m, **{"max_new_tokens": 6, "eos_id": EOS, "device": torch.device("cpu"), **kw}), m.cfg.vocab


def _batch(rows=3):
    from verl_omni_b200.utils.dataproto import DataProto

    return DataProto({"input_ids": torch.randint(0, 500, (rows, 5), generator=torch.Generator().manual_seed(1))}, {})


@pytest.mark.parametrize("temperature", [0.0, 1.0])
@pytest.mark.parametrize("kv", ["auto", "fp8_e4m3"])
def test_rows_that_ended_are_filled_up(kv, temperature):
    """Row r may say one token a step, then ends after r + 1 of them; its grammar is complete and allows nothing from there on."""

    def grammar(said):
        ok = torch.zeros(3, V, dtype=torch.bool)
        for r in range(3):
            t = said.shape[1]
            if t <= r:
                ok[r, 10 + t] = True
            elif t == r + 1:
                ok[r, EOS] = True
        return pack_allowed(ok)

    eng, V = _engine(kv_cache_dtype=kv, temperature=temperature, allowed_tokens=grammar)
    out = eng.generate(_batch(), seed=0).batch
    for r in range(3):
        assert out["responses"][r].tolist() == [10 + t for t in range(r + 1)] + [EOS] * (5 - r)
        assert out["response_mask"][r].tolist() == [1.0] * (r + 2) + [0.0] * (4 - r)
    assert bool((out["rollout_log_probs"] == 0).all())  # one choice each, and none


@pytest.mark.parametrize("eos", [None, EOS])
def test_rows_that_have_not_ended_are_an_error(eos):
    def grammar(said):
        ok = torch.ones(3, V, dtype=torch.bool)
        ok[:, EOS] = False
        ok[1] &= said.shape[1] < 2
        return pack_allowed(ok)

    eng, V = _engine(eos_id=eos, allowed_tokens=grammar)
    with pytest.raises(RuntimeError, match="no token to 1 of 3 rows"):
        eng.generate(_batch(), seed=0)
