"""The block table of a batch of the 8-bit paged cache once a captured step holds its address."""

import pytest
import torch

from verl_omni_b200.ops.paged8 import PagedKVCache8


def _batch(max_len=0):
    c = PagedKVCache8(1, 16, 1, 4, 16, "cpu")
    return c, c.batch([c.add_sequence(), c.add_sequence()], max_len)


def test_table_grows_until_it_is_captured():
    c, b = _batch(max_len=6)
    b.grow(3)
    b.grow(9)  # a third page
    assert b.table.shape[1] == 3
    at = b.table.data_ptr()
    b.captured = True
    b.at(11)
    b.reserve(0)
    assert b.table.data_ptr() == at and c.length[0] == 12
    state = (list(c.free), {s: list(p) for s, p in c.blocks.items()}, dict(c.length), b.off, b.pos.clone())
    for more in (lambda: b.at(12), lambda: b.grow(14), lambda: b.reserve(1)):
        with pytest.raises(RuntimeError, match="max_len"):
            more()
        now = (list(c.free), {s: list(p) for s, p in c.blocks.items()}, dict(c.length), b.off, b.pos)
        assert all(torch.equal(x, y) if isinstance(x, torch.Tensor) else x == y for x, y in zip(state, now))
    assert b.table.data_ptr() == at


def test_pages_reserved_behind_the_batch():
    c, b = _batch(max_len=4)
    b.at(0)
    b.captured = True
    c.reserve(b.sids, 8)
    with pytest.raises(RuntimeError, match="max_len"):
        b.at(1)
    assert b.table.shape[1] == 1 and c.length[0] == 1 and b.off == 1


def test_a_step_is_captured_only_while_a_stream_captures(monkeypatch):
    c, b = _batch(max_len=8)
    v = b.views()[0]
    x = torch.zeros(2, 1, 1, 16)
    b.at(0)
    v.append_at(x, x)
    v.attend_at(x)
    assert not b.captured
