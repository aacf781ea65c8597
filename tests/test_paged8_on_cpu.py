"""8-bit paged KV cache on the CPU: the oracle's number format, the block manager (sharing, forks, compaction, freeing)
and the rollout on it."""

import math

import pytest
import torch

from verl_omni_b200.ops.paged8 import (PagedKVCache8, append_paged8, attend_paged8, copy_pages, gather_paged8, page_scale)


def _rows(cache, sid, layer=0):
    n = cache.length[sid]
    t = torch.tensor([cache.blocks[sid]], dtype=torch.int32)
    return tuple(gather_paged8(p[layer], s[layer], t, n)[0] for p, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))


def _fill(cache, sids, n, seed=0):
    g = torch.Generator().manual_seed(seed)
    b = cache.batch(sids)
    for v in b.views():
        v.append(torch.randn(len(sids), cache.k.shape[2], n, cache.k.shape[4], generator=g),
                 torch.randn(len(sids), cache.k.shape[2], n, cache.k.shape[4], generator=g))


def _consistent(cache):
    """Every page is free or owned as often as its count says."""
    owned = [0] * len(cache.refs)
    for b in cache.blocks.values():
        for i in b:
            owned[i] += 1
    assert owned == cache.refs
    assert sorted(cache.free) == [i for i, r in enumerate(cache.refs) if r == 0]


def test_page_scale_is_the_smallest_power_of_two():
    amax = torch.cat([torch.tensor([0.0, 448.0, 448.0001, 1e-45, 3e38, 1.0]), torch.rand(500) * torch.exp2(torch.randint(-90, 90, (500,)).float())])
    s = page_scale(amax).double()
    assert torch.equal(torch.exp2(torch.log2(s).round()), s)
    assert bool((amax.double() <= 448 * s).all())
    small = s == 2.0 ** -100
    assert bool((amax.double()[~small] > 448 * s[~small] / 2).all())
    assert s[:2].tolist() == [2.0 ** -100, 1.0] and float(s[2]) == 2.0


def test_append_keeps_values_within_the_format():
    torch.manual_seed(0)
    c = PagedKVCache8(1, 8, 2, 16, 32, "cpu")
    s = c.add_sequence()
    view = c.batch([s]).views()[0]
    k, v = torch.randn(2, 1, 2, 70, 32).unbind(0)
    at = 0
    for n in (1, 14, 1, 3, 51):
        view.append(k[:, :, at:at + n], v[:, :, at:at + n])
        at += n
    assert view.len == c.length[s] == 70 and len(c.blocks[s]) == 5
    for got, x in zip(_rows(c, s), (k[0], v[0])):
        # e4m3 rounds to 2^-4 of the value, twice at most where a page's scale grew into subnormals (2^-10 of the scale)
        assert bool(((got - x).abs() <= 2.0 ** -4 * x.abs() + 2.0 ** -9 * c.k_scale.max()).all())
    q = torch.randn(1, 4, 1, 32)
    o = view.attend(q)
    kk, vv = (x.repeat_interleave(2, 0) for x in _rows(c, s))
    p = torch.softmax(torch.einsum("hd,htd->ht", q[0, :, 0], kk) / math.sqrt(32), -1)
    torch.testing.assert_close(o[0, 0], torch.einsum("ht,htd->hd", p, vv), rtol=1e-5, atol=1e-5)


def test_several_tokens_are_causal():
    torch.manual_seed(0)
    c = PagedKVCache8(1, 20, 2, 8, 16, "cpu")
    a, b = c.add_sequence(), c.add_sequence()
    k, v = torch.randn(2, 1, 2, 21, 16).unbind(0)
    q = torch.randn(1, 4, 21, 16)
    one, many = c.batch([a]).views()[0], c.batch([b]).views()[0]
    outs = []
    for t in range(21):
        one.append(k[:, :, t:t + 1], v[:, :, t:t + 1])
        outs.append(one.attend(q[:, :, t:t + 1]))
    many.append(k, v)
    whole = many.attend(q)
    # rows of one page may carry an earlier scale than the page written at once: the difference is the format's
    torch.testing.assert_close(torch.cat(outs, 1), whole, rtol=0.2, atol=0.2)
    torch.testing.assert_close(outs[-1][0, 0], whole[0, -1], rtol=0.05, atol=0.05)
    short = attend_paged8(q[:, :, :3], c.k[0], c.v[0], c.k_scale[0], c.v_scale[0], many.batch.table, torch.tensor([1], dtype=torch.int32))
    assert not short[0, :2].any() and bool(short[0, 2].any())  # two of three tokens stand before the cache's start


def test_fork_shares_pages_and_copies_the_last():
    c = PagedKVCache8(3, 20, 2, 4, 16, "cpu")
    s, full = c.add_sequence(), c.add_sequence()
    _fill(c, [s], 10)
    _fill(c, [full], 8, seed=1)
    kids = c.fork([s, full], 3)
    _consistent(c)
    for kid in kids[0]:
        assert c.blocks[kid][:2] == c.blocks[s][:2] and c.blocks[kid][2] != c.blocks[s][2]
    assert all(c.blocks[k] == c.blocks[full] for k in kids[1])
    assert len(c.free) == 20 - (3 + 3) - 2
    want = [_rows(c, s, i) for i in range(3)]
    _fill(c, [kids[0][0], kids[1][2], s], 3, seed=2)  # each writes its own pages
    _consistent(c)
    for kid in kids[0][1:]:
        for i in range(3):
            for x, y in zip(_rows(c, kid, i), want[i]):
                assert torch.equal(x, y)
    c.free_sequence(s)
    c.free_sequence(full)
    _consistent(c)
    for kid in kids[0][1:]:
        assert torch.equal(_rows(c, kid)[0], want[0][0])  # shared pages outlive the parent
    for k in kids[0] + kids[1]:
        c.free_sequence(k)
    assert sorted(c.free) == list(range(20)) and not c.blocks


def test_fork_of_an_empty_sequence_and_without_room():
    c = PagedKVCache8(1, 3, 1, 4, 16, "cpu")
    e = c.add_sequence()
    assert [c.length[k] for k in c.fork([e], 2)[0]] == [0, 0]
    s = c.add_sequence()
    _fill(c, [s], 6)
    before = (list(c.free), dict(c.blocks), list(c.refs))
    with pytest.raises(RuntimeError, match="out of pages"):
        c.fork([s], 2)
    with pytest.raises(RuntimeError, match="out of pages"):
        c.reserve([s, e], 8)
    assert (c.free, c.blocks, c.refs) == before


def test_compact_moves_live_pages_down():
    c = PagedKVCache8(2, 24, 2, 4, 16, "cpu")
    sids = [c.add_sequence() for _ in range(5)]
    for i, s in enumerate(sids):
        _fill(c, [s], 5 + 3 * i, seed=i)
    kid = c.fork([sids[3]], 1)[0][0]
    batch = c.batch([sids[3], sids[4]])
    want = {s: [_rows(c, s, i) for i in range(2)] for s in sids + [kid]}
    for s in (sids[0], sids[2]):
        c.free_sequence(s)
    live = c.compact()
    _consistent(c)
    assert live == sum(r > 0 for r in c.refs) and all(c.refs[:live]) and not any(c.refs[live:])
    for s in (sids[1], sids[3], sids[4], kid):
        for i in range(2):
            for x, y in zip(_rows(c, s, i), want[s][i]):
                assert torch.equal(x, y)
    # a batch made before sees the moved pages
    view = batch.views()[0]
    view.append(torch.zeros(2, 2, 1, 16), torch.zeros(2, 2, 1, 16))
    assert batch.table[0, 0] == c.blocks[sids[3]][0]
    assert c.compact() == live + sum(len(c.blocks[s]) for s in sids[3:]) - sum(-(-(5 + 3 * i) // 4) for i in (3, 4))


def test_refusals():
    c = PagedKVCache8(1, 4, 2, 4, 16, "cpu")
    for bad in [(0, 4, 2, 4, 16), (1, 0, 2, 4, 16), (1, 4, 2, 0, 16), (1, 4, 2, 4, 20), (1, 4, 2, 4, 512)]:
        with pytest.raises(ValueError):
            PagedKVCache8(*bad, "cpu")
    s = c.add_sequence()
    with pytest.raises(ValueError, match="twice"):
        c.batch([s, s])
    for src, dst in [([0], [4]), ([-1], [0]), ([0, 1], [2]), ([0, 1], [2, 2]), ([0, 1], [1, 2])]:
        with pytest.raises(ValueError):
            copy_pages(c.pools, src, dst)
    t, n = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 2, 1, 16)
    pools = [p[0] for p in c.pools]
    with pytest.raises(ValueError):
        append_paged8(x, x[:, :1], *pools, t, n)
    with pytest.raises(ValueError):
        append_paged8(x, x, pools[0].float(), *pools[1:], t, n)
    with pytest.raises(ValueError):
        attend_paged8(torch.zeros(1, 3, 1, 16), *pools, t, n)
    with pytest.raises(ValueError, match="no backward"):
        attend_paged8(torch.zeros(1, 2, 1, 16, requires_grad=True), *pools, t, n)


# ------------------------------------------------------------------------------------------------ rollout
def _model():
    from verl_omni_b200.models.moe_llm import MoEConfig, MoELLM

    torch.manual_seed(0)
    return MoELLM(MoEConfig.tiny()).eval()


def _engine(m, **kw):
    from verl_omni_b200.workers.rollout.llm_rollout import LLMRolloutEngine

    return LLMRolloutEngine(m, **{"max_new_tokens": 6, "temperature": 1.0, "device": torch.device("cpu"), **kw})


def _batch(rows=2, group=3, P=9):
    from verl_omni_b200.utils.dataproto import DataProto

    ids = torch.randint(0, 500, (rows, P), generator=torch.Generator().manual_seed(5)).repeat_interleave(group, 0)
    return DataProto({"input_ids": ids}, {})


def test_rollout_on_shared_pages_equals_unshared():
    m = _model()
    for bs in (0, 4):
        eng = _engine(m, kv_cache_dtype="fp8_e4m3", kv_block_size=bs)
        a, b = eng.generate(_batch(), seed=3, group=3), eng.generate(_batch(), seed=3)
        assert torch.equal(a.batch["responses"], b.batch["responses"])
        torch.testing.assert_close(a.batch["rollout_log_probs"], b.batch["rollout_log_probs"])
    ref = _engine(m).generate(_batch(), seed=3)
    # the same tokens scored: the cache's 8 bits move the log-probs a little
    assert float((ref.batch["rollout_log_probs"][:, 0] - a.batch["rollout_log_probs"][:, 0]).abs().max()) < 1e-4
    with pytest.raises(ValueError, match="group=4"):
        eng.generate(_batch(), group=4)


def test_rollout_continues_a_prompt_in_chunks():
    m = _model()
    c = PagedKVCache8(len(m.layers), 16, m.cfg.kv_heads, 4, m.cfg.head_dim, "cpu")
    views = c.batch([c.add_sequence(), c.add_sequence()]).views()
    ids = torch.randint(0, 500, (2, 14), generator=torch.Generator().manual_seed(1))
    with torch.no_grad():
        whole = m(ids)
        parts = [m(ids[:, a:b], caches=views, pos0=a) for a, b in ((0, 6), (6, 13), (13, 14))]
    got = torch.cat(parts, 1)
    torch.testing.assert_close(got[:, :6], whole[:, :6])
    assert float((got - whole).norm() / whole.norm()) < 0.05


def test_rollout_device_positions_match_host_positions():
    m = _model()
    ids = torch.randint(0, 500, (2, 7), generator=torch.Generator().manual_seed(1))
    got = []
    for device_pos in (False, True):
        c = PagedKVCache8(len(m.layers), 16, m.cfg.kv_heads, 4, m.cfg.head_dim, "cpu")
        views = c.batch([c.add_sequence(), c.add_sequence()], 12).views()
        with torch.no_grad():
            m(ids[:, :4], caches=views, pos0=0)
            out = []
            for t in range(4, 7):
                if device_pos:
                    views[0].batch.at(views[0].off)
                    out.append(m(ids[:, t:t + 1], caches=views, pos_t=torch.tensor([t])))
                    for v in views:
                        v.off += 1
                else:
                    out.append(m(ids[:, t:t + 1], caches=views, pos0=t))
        got.append(torch.cat(out, 1))
        assert [c.length[s] for s in (0, 1)] == [7, 7]
    torch.testing.assert_close(got[0], got[1])


def test_rollout_penalties_bias_and_mask():
    from verl_omni_b200.ops.logits import pack_allowed

    m = _model()
    V = m.cfg.vocab
    batch = _batch(rows=4, group=1)
    plain = _engine(m).generate(batch, seed=1)
    same = _engine(m, logit_bias=torch.zeros(V)).generate(batch, seed=1)
    assert torch.equal(plain.batch["responses"], same.batch["responses"])
    # a grammar that allows one token more at each step
    ok = lambda said: pack_allowed((torch.arange(V) <= said.shape[1])[None])  # noqa: E731
    out = _engine(m, allowed_tokens=ok).generate(batch, seed=1)
    assert bool((out.batch["responses"] <= torch.arange(6)).all())
    torch.testing.assert_close(out.batch["rollout_log_probs"][:, 0], torch.zeros(4))  # one choice
    out = _engine(m, presence_penalty=1e4).generate(batch, seed=1).batch["responses"]
    assert all(len(set(r)) == 6 for r in out.tolist())  # nothing twice
    out = _engine(m, logit_bias=torch.nn.functional.one_hot(torch.tensor(7), V) * 1e4).generate(batch, seed=1)
    assert bool((out.batch["responses"] == 7).all())
    out = _engine(m, repetition_penalty=1e4, temperature=0.0, logit_bias=-30.0 * torch.ones(V)).generate(batch, seed=1)
    assert out.batch["responses"].shape == (4, 6)


def test_rollout_refusals():
    m = _model()
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        _engine(m, kv_cache_dtype="int4")
    with pytest.raises(ValueError, match="positive"):
        _engine(m, repetition_penalty=0.0)
    with pytest.raises(ValueError, match="pipeline"):
        _engine(m, pp=object(), kv_cache_dtype="fp8_e4m3")
    with pytest.raises(ValueError, match="pipeline"):
        _engine(m, pp=object(), presence_penalty=0.5)


def test_trainer_rolls_out_on_the_8_bit_cache():
    from verl_omni_b200.models.moe_llm import MoEConfig
    from verl_omni_b200.trainer.omni.omni_trainer import OmniGRPOTrainer
    from verl_omni_b200.workers.config.diffusion import DiffusionActorConfig

    t = OmniGRPOTrainer(MoEConfig.tiny(), DiffusionActorConfig(), device=torch.device("cpu"), n=2, kv_block_size=8,
                        rollout_kw=dict(kv_cache_dtype="fp8_e4m3", frequency_penalty=0.1))
    m = t.step(2)
    assert m["actor/grad_norm"] == m["actor/grad_norm"]
