"""Padding ahead of a prompt is no history for the rollout's penalties."""

import pandas as pd
import torch


def _dataset(tmp_path, prompts):
    from verl_omni_b200.utils.datasets_parquet import ParquetOmniRLDataset

    pd.DataFrame({"prompt_ids": prompts}).to_parquet(tmp_path / "p.parquet")
    return ParquetOmniRLDataset([str(tmp_path / "p.parquet")], vocab=512, max_prompt_length=8)


def test_dataset_counts_its_padding(tmp_path):
    b = _dataset(tmp_path, [[5, 0, 7], list(range(20, 30)), [0]]).get_batch([0, 1, 2]).batch
    assert b["prompt_pad"].tolist() == [5, 0, 7] and b["prompt_pad"].dtype == torch.int32
    assert b["input_ids"][0].tolist() == [0] * 5 + [5, 0, 7]


def test_padding_gets_no_repetition_penalty(tmp_path, monkeypatch):
    """Short prompts padded with token 0: the logit of token 0 is penalised only where the prompt itself holds it."""
    from verl_omni_b200.models.moe_llm import MoEConfig, MoELLM
    from verl_omni_b200.workers.rollout import llm_rollout

    batch = _dataset(tmp_path, [[5, 6, 7], [5, 0, 7]]).get_batch([0, 1]).repeat(2)
    torch.manual_seed(0)
    m = MoELLM(MoEConfig.tiny()).eval()
    seen, orig = [], llm_rollout.process_logits

    def record(x, *a, **k):
        y = orig(x, *a, **k)
        seen.append((x, y))
        return y

    monkeypatch.setattr(llm_rollout, "process_logits", record)
    eng = llm_rollout.LLMRolloutEngine(m, max_new_tokens=2, repetition_penalty=2.0, device=torch.device("cpu"))
    out = eng.generate(batch, seed=0)
    x, y = seen[0]
    assert torch.equal(y[:2, 0], x[:2, 0]) and bool((y[2:, 0] != x[2:, 0]).all())
    assert bool((y[:, 5] != x[:, 5]).all())
    assert torch.equal(out.batch["prompts"], batch.batch["input_ids"]) and out.batch["prompt_pad"].tolist() == [5] * 4


def _tp(rank, world):
    import torch.distributed as dist

    from verl_omni_b200.models.moe_llm import MoEConfig, MoELLM
    from verl_omni_b200.parallel.tensor_parallel import TPContext
    from verl_omni_b200.utils.dataproto import DataProto
    from verl_omni_b200.workers.rollout.llm_rollout import LLMRolloutEngine

    torch.manual_seed(0)
    m = MoELLM(MoEConfig.tiny())
    ids = torch.randint(1, 500, (2, 6), generator=torch.Generator().manual_seed(rank))
    pad = torch.tensor([2 * rank, 3], dtype=torch.int32)
    ids[torch.arange(6) < pad[:, None]] = 0
    batch = DataProto({"input_ids": ids, "prompt_pad": pad}, {})
    kw = dict(max_new_tokens=4, temperature=0.0, repetition_penalty=3.0, logit_bias=torch.nn.functional.one_hot(torch.tensor(0), 512) * 0.01,
              device=torch.device("cpu"))
    a = LLMRolloutEngine(m, tp=TPContext(dist.group.WORLD), **kw).generate(batch, seed=1)
    b = LLMRolloutEngine(m, **kw).generate(batch, seed=1)
    assert torch.equal(a.batch["responses"], b.batch["responses"])
    torch.testing.assert_close(a.batch["rollout_log_probs"], b.batch["rollout_log_probs"], rtol=1e-4, atol=1e-5)


def test_padding_of_a_tensor_parallel_rollout():
    from tests._dist_util import run_ranks

    run_ranks(_tp, 2)
