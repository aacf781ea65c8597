"""Log-probs under a rollout's penalties on the GPU: values and gradients against 64 bits, and the trainer's against the rollout's."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_values_and_gradients():
    from verl_omni_b200.models.layers import Linear
    from verl_omni_b200.ops.vocab_logprob import shaped_token_logprobs
    from test_shaped_logprobs_on_cpu import PENALTIES, _plain

    torch.manual_seed(0)
    B, L, P, V, D, T = 2, 40, 9, 1000, 256, 0.8
    head = Linear(D, V, bias=False).to("cuda", torch.bfloat16)
    with torch.no_grad():
        head.weight.copy_(torch.randn(V, D) * D ** -0.5)
    ids = torch.randint(0, 30, (B, L), device="cuda")
    h = torch.randn(B, L - 1, D, device="cuda").bfloat16().requires_grad_(True)
    got = shaped_token_logprobs(h, head.weight, ids[:, 1:], T, history=ids, prompt_len=P, rows_at_once=23, **PENALTIES)
    z = head(h.detach()).float().cpu().double().requires_grad_(True)  # the same bf16 logits
    want = torch.stack([_plain(z[b], ids[b].cpu(), P, T) for b in range(B)])
    assert not got[:, :P - 1].any()
    # fp32: logits of a few units, sums over V of exponentials that agree to 2^-22 or so
    torch.testing.assert_close(got[:, P - 1:].detach().cpu().double(), want.detach(), rtol=1e-5, atol=1e-5)
    g = torch.randn(B, L - P)
    (got[:, P - 1:] * g.cuda()).sum().backward()
    (dz,) = torch.autograd.grad((want * g).sum(), z)
    w64, h64 = head.weight.detach().cpu().double(), h.detach().cpu().double()
    # dlogits are rounded to bf16 (2^-8 of each), products summed in fp32, results rounded to bf16
    dh, dw = dz @ w64, torch.einsum("bsv,bsd->vd", dz, h64)
    tol_h = 2.0 ** -8 * 1.1 * (dz.abs() @ w64.abs()) + 2.0 ** -8 * dh.abs()
    tol_w = 2.0 ** -8 * 1.1 * torch.einsum("bsv,bsd->vd", dz.abs(), h64.abs()) + 2.0 ** -8 * dw.abs()
    dw_got = head.weight.grad
    assert bool(((h.grad.cpu().double() - dh).abs() <= tol_h + 1e-9).all())
    # two chunks of rows, each rounded to bf16 before they are added
    assert bool(((dw_got.cpu().double() - dw).abs() <= 4 * tol_w + 1e-9).all())


def test_trainer_log_probs_follow_the_rollouts():
    """bf16 model: with penalties the recompute and the rollout differ no more than twice what they do without."""
    from verl_omni_b200.models.moe_llm import MoEConfig
    from verl_omni_b200.trainer.omni.omni_trainer import OmniGRPOTrainer
    from verl_omni_b200.workers.config.diffusion import DiffusionActorConfig

    cfg = MoEConfig(vocab=2048, hidden=512, layers=2, q_heads=16, kv_heads=2, head_dim=128, experts=8, top_k=2,
                    expert_ffn=256, audio_layers=1, audio_dim=128, audio_mel=16, vision_layers=1, vision_dim=128,
                    vision_patch_dim=48, audio_token=2046, image_token=2047)
    diff = []
    for kw in ({}, dict(repetition_penalty=1.4, presence_penalty=0.5, frequency_penalty=0.3)):
        t = OmniGRPOTrainer(cfg, DiffusionActorConfig(), device=torch.device("cuda", 0), n=4, response_len=48, rollout_kw=kw)
        m = t.step(2)
        assert m["actor/grad_norm"] > 0
        diff.append(m["rollout_corr/logprob_abs_diff_mean"])
    assert diff[1] <= 2 * diff[0] + 1e-4


def test_chunks_add_up_in_the_engines_gradient(monkeypatch):
    """The projection's weight gradient goes into the engine's fp32 buffer, once per chunk of rows."""
    import functools

    from verl_omni_b200.models.moe_llm import MoEConfig
    from verl_omni_b200.ops import vocab_logprob
    from verl_omni_b200.trainer.omni.omni_trainer import OmniGRPOTrainer
    from verl_omni_b200.workers.config.diffusion import DiffusionActorConfig

    cfg = MoEConfig(vocab=2048, hidden=512, layers=1, q_heads=16, kv_heads=2, head_dim=128, experts=8, top_k=2,
                    expert_ffn=256, audio_layers=1, audio_dim=128, audio_mel=16, vision_layers=1, vision_dim=128,
                    vision_patch_dim=48, audio_token=2046, image_token=2047)
    t = OmniGRPOTrainer(cfg, DiffusionActorConfig(), device=torch.device("cuda", 0), n=2, response_len=20,
                        rollout_kw=dict(repetition_penalty=1.4, frequency_penalty=0.3))
    out = t.rollout.generate(t.make_prompts(2, seed=1).repeat(2), seed=0)
    t.engine.train_mode()
    w, orig, got = t.model.lm_head.weight, vocab_logprob.shaped_token_logprobs, []
    for rows in (512, 13):
        monkeypatch.setattr(vocab_logprob, "shaped_token_logprobs", functools.partial(orig, rows_at_once=rows))
        t.engine.zero_grad()
        t._resp_logprobs(out).sum().backward()
        got.append(w.main_grad.clone())
    assert got[0].dtype == torch.float32 and bool(got[0].any())
    # the same bf16 dlogits and hidden states, summed in another order in fp32
    torch.testing.assert_close(got[1], got[0], rtol=1e-4, atol=1e-4 * float(got[0].abs().max()))
