"""Training under a rollout's penalties: log-probs and gradients are those of the distribution that responses are drawn from."""

import pytest
import torch

from tests._dist_util import run_ranks
from verl_omni_b200.models.moe_llm import MoEConfig, MoELLM
from verl_omni_b200.ops.logits import process_logits
from verl_omni_b200.ops.vocab_logprob import shaped_token_logprobs

PENALTIES = dict(repetition=1.3, presence=0.4, frequency=0.2)
ENGINE = dict(repetition_penalty=1.3, presence_penalty=0.4, frequency_penalty=0.2)


def _plain(logits, ids, P, temperature, bias=None, pad=0):
    """log p of the response tokens [R], one position after the other, in 64 bits (logits [S, V] of one sequence)."""
    out = []
    for t in range(P, ids.shape[0]):
        z = logits[t - 1].double()
        said = ids[P:t].tolist()
        f = torch.ones_like(z)
        for v in set(ids[pad:t].tolist()):
            f[v] = 1 / PENALTIES["repetition"] if z[v] > 0 else PENALTIES["repetition"]
        z = z * f
        for v in set(said):
            z = z - torch.nn.functional.one_hot(torch.tensor(v), z.shape[0]) * (PENALTIES["frequency"] * said.count(v) + PENALTIES["presence"])
        if bias is not None:
            z = z + bias.double()
        out.append(torch.log_softmax(z / temperature, -1)[ids[t]])
    return torch.stack(out)


@pytest.mark.parametrize("rows_at_once", [1, 4, 512])
@pytest.mark.parametrize("first", [0, 3, 7])
def test_definition_and_gradient(first, rows_at_once):
    torch.manual_seed(0)
    B, L, P, V, D = 2, 12, 5, 40, 16
    ids = torch.randint(0, 8, (B, L))
    w = torch.randn(V, D, requires_grad=True)
    h = torch.randn(B, L, D, requires_grad=True)
    bias = torch.randn(V)
    head = lambda x: x @ w.t()  # noqa: E731
    got = shaped_token_logprobs(h[:, first:-1], w, ids[:, first + 1:], 0.7, history=ids, prompt_len=P, bias=bias, first=first,
                                rows_at_once=rows_at_once, **PENALTIES)
    want = torch.stack([_plain(head(h[b]), ids[b], P, 0.7, bias) for b in range(B)])
    cut = max(0, P - 1 - first)
    skip = max(0, first - (P - 1))
    assert got.shape == (B, L - 1 - first) and not got[:, :cut].any()
    torch.testing.assert_close(got[:, cut:].double(), want[:, skip:], rtol=1e-5, atol=1e-5)
    g = torch.randn(B, L - 1 - first - cut)
    a = torch.autograd.grad((got[:, cut:] * g).sum(), (h, w))
    b = torch.autograd.grad((want[:, skip:] * g).sum(), (h, w))
    for x, y in zip(a, b):
        torch.testing.assert_close(x, y.to(x.dtype), rtol=1e-4, atol=1e-5)


def test_a_part_of_the_prompt_alone_keeps_the_graph():
    h = torch.randn(1, 3, 8, requires_grad=True)
    w = torch.randn(20, 8)
    ids = torch.randint(0, 20, (1, 9))
    out = shaped_token_logprobs(h, w, ids[:, 1:4], 1.0, history=ids, prompt_len=8, **PENALTIES)
    assert not out[:, :2].any() and out.requires_grad


def _trainer(**kw):
    from verl_omni_b200.trainer.omni.omni_trainer import OmniGRPOTrainer
    from verl_omni_b200.workers.config.diffusion import DiffusionActorConfig

    ac = DiffusionActorConfig()
    ac.optim.lr = 1e-3
    return OmniGRPOTrainer(MoEConfig.tiny(), ac, device=torch.device("cpu"), n=2, response_len=6, **kw)


@pytest.mark.parametrize("temperature", [1.0, 0.6])
@pytest.mark.parametrize("micro", [None, 1])
def test_trainer_log_probs_equal_the_rollouts(micro, temperature):
    bias = torch.zeros(MoEConfig.tiny().vocab)
    bias[:10] = 3.0  # tokens come again and again
    t = _trainer(rollout_kw=dict(**ENGINE, logit_bias=bias), micro_batch_size=micro, temperature=temperature)
    out = t.rollout.generate(t.make_prompts(2, seed=5).repeat(2), seed=1)
    with torch.no_grad():
        old = t._resp_logprobs(out)
    torch.testing.assert_close(old, out.batch["rollout_log_probs"], rtol=1e-4, atol=1e-4)
    m = t.step(2)
    assert m["rollout_corr/logprob_abs_diff_mean"] < 1e-4 and m["actor/grad_norm"] > 0


def test_trainer_log_probs_of_padded_prompts(tmp_path):
    import pandas as pd

    from verl_omni_b200.utils.datasets_parquet import ParquetOmniRLDataset

    pd.DataFrame({"prompt_ids": [[5, 6, 7], [9, 0, 4, 4, 2]]}).to_parquet(tmp_path / "p.parquet")
    bias = torch.zeros(512)
    bias[0] = 6.0  # the padding id is drawn
    t = _trainer(rollout_kw=dict(repetition_penalty=2.0, logit_bias=bias), micro_batch_size=1)
    t.dataset = ParquetOmniRLDataset([str(tmp_path / "p.parquet")], vocab=512, max_prompt_length=8)
    m = t.step(2)
    assert m["rollout_corr/logprob_abs_diff_mean"] < 1e-4


def test_a_grammar_mask_is_refused_by_the_trainer():
    with pytest.raises(ValueError, match="grammar"):
        _trainer(rollout_kw=dict(allowed_tokens=lambda said: None))


def test_without_penalties_the_log_probs_are_the_models():
    t = _trainer()
    assert t.rollout.shaping is None
    assert t.step(2)["rollout_corr/logprob_abs_diff_mean"] < 1e-4


def _tp_check(rank, world):
    import torch.distributed as dist

    from verl_omni_b200.parallel.tensor_parallel import TPContext

    torch.manual_seed(0)
    m = MoELLM(MoEConfig.tiny())
    for P in (2, 9):  # 9: the first rank's half is prompt alone
        ids = torch.randint(0, 20, (2, 12), generator=torch.Generator().manual_seed(3))
        tgt = ids[:, 1:]
        gy = torch.randn(2, 12 - P, generator=torch.Generator().manual_seed(4))
        kw = dict(targets=tgt, temperature=0.9, shaping=dict(history=ids, prompt_len=P, **PENALTIES))
        m.tp = None
        m.zero_grad(set_to_none=True)
        ref = m(ids[:, :-1], **kw)[:, P - 1:]
        (ref * gy).sum().backward()
        ref_g = {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}
        m.zero_grad(set_to_none=True)
        m.tp = TPContext(dist.group.WORLD)
        out = m(ids[:, :-1], **kw)[:, P - 1:]
        torch.testing.assert_close(out, ref.detach(), rtol=1e-4, atol=1e-5)
        (out * gy).sum().backward()
        for n, p in m.named_parameters():
            if n in ref_g:
                g = p.grad.clone()
                dist.all_reduce(g)  # each rank holds its heads' / tokens' share
                torch.testing.assert_close(g, ref_g[n], rtol=1e-3, atol=1e-5, msg=lambda s: f"{n}: {s}")


def test_tensor_parallel_scores():
    run_ranks(_tp_check, 2)
