"""A step on the 8-bit paged cache captured in a CUDA graph: replays follow the batch, and the table it reads is not replaced."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_captured_step():
    from verl_omni_b200.ops.paged8 import PagedKVCache8

    torch.manual_seed(0)
    B, Hk, rep, hd, bs, most = 2, 2, 4, 64, 8, 24
    k, v = (torch.randn(B, Hk, most + bs, hd, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(B, Hk * rep, most + bs, hd, device="cuda").bfloat16()
    eager, graph = (PagedKVCache8(1, 16, Hk, bs, hd, "cuda") for _ in range(2))
    want = []
    view = eager.batch([eager.add_sequence() for _ in range(B)]).views()[0]
    for t in range(most):
        view.append(k[:, :, t:t + 1], v[:, :, t:t + 1])
        want.append(view.attend(q[:, :, t:t + 1]))
    batch = graph.batch([graph.add_sequence() for _ in range(B)], most)
    view = batch.views()[0]
    kt, vt, qt = (torch.zeros_like(x[:, :, :1]) for x in (k, v, q))
    step = None
    for t in range(most):
        batch.at(t)
        for x, y in ((kt, k), (vt, v), (qt, q)):
            x.copy_(y[:, :, t:t + 1])
        if t == 0:
            view.append_at(kt, vt)
            got = view.attend_at(qt)
            assert not batch.captured
        else:
            if step is None:
                step = torch.cuda.CUDAGraph()
                with torch.cuda.graph(step):
                    view.append_at(kt, vt)
                    got = view.attend_at(qt)
                assert batch.captured
            step.replay()
        assert torch.equal(got, want[t])
    at = batch.table.data_ptr()
    with pytest.raises(RuntimeError, match="max_len"):
        batch.at(most)
    assert batch.table.data_ptr() == at and graph.length[0] == most
