"""Processing of next-token logits before sampling: penalties for repeated tokens, a bias and a grammar bitmask.

For a row with ``history`` tokens ``h[:len]`` of which the first ``prompt_len`` are the prompt::

    y = x > 0 ? x / repetition : x * repetition     where the token occurs in h[:len]
    y -= frequency * count + presence               where it occurs count > 0 times in h[prompt_len:len]
    y += bias
    y = -inf                                        where its bit of ``allowed`` is clear

One launch (``csrc/logits.cu``), differentiable in the logits; CPU tensors run an fp32 torch oracle.
Counterpart of vLLM's logits processors and guided-decoding bitmask under the reference's AR rollout
(``verl_omni/workers/rollout/vllm_rollout/vllm_omni_async_server.py:537-579``).
"""

from __future__ import annotations

from typing import Optional, Union

import torch
from torch.autograd.forward_ad import unpack_dual

Param = Union[float, torch.Tensor]


def _ext():
    from verl_omni_b200.ops._ext import ext

    return ext()


def pack_allowed(mask: torch.Tensor) -> torch.Tensor:
    """Boolean ``[rows, vocab]`` -> int32 bitmask ``[rows, ceil(vocab / 32)]`` (bit ``v % 32`` of word ``v // 32``)."""
    R, V = mask.shape
    m = torch.zeros(R, -(-V // 32) * 32, dtype=torch.int64, device=mask.device)
    m[:, :V] = mask.to(torch.int64)
    w = (m.view(R, -1, 32) << torch.arange(32, device=mask.device)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


def _col(p: Param, x: torch.Tensor) -> torch.Tensor:
    if not isinstance(p, torch.Tensor):
        return torch.full((x.shape[0], 1), float(p), device=x.device)
    if p.shape != (x.shape[0],) or p.dtype != torch.float32:
        raise ValueError("repetition, presence, frequency: a number or float32 [rows]")
    return p[:, None]


def _counts(x, history, lens, prompt_lens, rows):
    """(token seen [R, V], occurrences in the response [R, V]) of every logits row."""
    R, V = x.shape
    if history is None:
        z = torch.zeros(R, V, device=x.device)
        return z > 0, z
    if history.dim() != 2 or history.dtype not in (torch.int64, torch.int32) or (rows is None and history.shape[0] != R):
        raise ValueError("history: int64 or int32 [sequences, tokens], one row per logits row (or pass rows)")
    for t in (lens, prompt_lens, rows):
        if t is not None and (t.shape != (R,) or t.dtype != torch.int32):
            raise ValueError("lens, prompt_lens, rows: int32 [rows]")
    h = history.long()
    live = torch.ones(R, 1, dtype=torch.bool, device=x.device)
    if rows is not None:
        live = ((rows >= 0) & (rows < h.shape[0]))[:, None]
        h = h[rows.long().clamp(0, max(0, h.shape[0] - 1))]
    at = torch.arange(h.shape[1], device=x.device)[None]
    live = live & (h >= 0) & (h < V)
    if lens is not None:
        live = live & (at < lens[:, None])
    said = live if prompt_lens is None else live & (at >= prompt_lens[:, None])
    h = h.clamp(0, V - 1)
    zero = torch.zeros(R, V, device=x.device)
    return zero.scatter_add(1, h, live.float()) > 0, zero.scatter_add(1, h, said.float())


def _allowed(allowed, x):
    if allowed is None:
        return None
    R, V = x.shape
    if allowed.dtype != torch.int32 or allowed.dim() != 2 or allowed.shape[1] != -(-V // 32) or allowed.shape[0] not in (1, R):
        raise ValueError("allowed: int32 bitmask [rows or 1, ceil(vocab / 32)]")
    at = torch.arange(V, device=x.device)
    return (allowed[:, at // 32] >> (at % 32)) & 1 == 1


def process_logits_reference(x, history=None, lens=None, prompt_lens=None, rows=None, repetition: Param = 1.0,
                             presence: Param = 0.0, frequency: Param = 0.0, bias=None, allowed=None) -> torch.Tensor:
    """fp32 oracle (differentiable through torch)."""
    if x.dim() != 2:
        raise ValueError("logits: [rows, vocab]")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape[-1] != x.shape[1]):
        raise ValueError("bias: float32 [vocab] or [rows, vocab]")
    f = x.float()
    seen, said = _counts(x, history, lens, prompt_lens, rows)
    rep = _col(repetition, x)
    y = torch.where(seen, torch.where(f > 0, f / rep, f * rep), f)
    y = torch.where(said > 0, y - (_col(frequency, x) * said + _col(presence, x)), y)
    if bias is not None:
        y = y + bias
    ok = _allowed(allowed, x)
    if ok is not None:
        y = torch.where(ok, y, float("-inf"))
    return y.to(x.dtype)


def _split(p: Param) -> tuple[Optional[torch.Tensor], float]:
    return (p, 0.0) if isinstance(p, torch.Tensor) else (None, float(p))


class _ProcessLogits(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, args):
        ctx.save_for_backward(x, *(t for t in args if isinstance(t, torch.Tensor)))
        ctx.slots = [None if isinstance(t, torch.Tensor) else t for t in args]
        ctx.where = [isinstance(t, torch.Tensor) for t in args]
        return _ext().process_logits(x, None, *args)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        x, *ts = ctx.saved_tensors
        it = iter(ts)
        args = [next(it) if w else v for w, v in zip(ctx.where, ctx.slots)]
        return _ext().process_logits(x, g, *args), None


def process_logits(x: torch.Tensor, history: Optional[torch.Tensor] = None, lens: Optional[torch.Tensor] = None,
                   prompt_lens: Optional[torch.Tensor] = None, rows: Optional[torch.Tensor] = None,
                   repetition: Param = 1.0, presence: Param = 0.0, frequency: Param = 0.0,
                   bias: Optional[torch.Tensor] = None, allowed: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Processed logits, new tensor of x's type: x ``[R, V]`` fp32 or bf16.

    ``history [N, L]`` int64 or int32 token ids (ids outside ``[0, V)`` are ignored), ``lens`` / ``prompt_lens [R]``
    int32 (all ``L`` / 0 without); ``rows [R]`` int32: the history row of each logits row where they are not one to one
    (training: every position of a sequence has its own ``lens``).  ``repetition``, ``presence``, ``frequency``:
    numbers or fp32 ``[R]``.  ``bias`` fp32 ``[V]`` or ``[R, V]``; ``allowed`` int32 bitmask ``[R or 1, ceil(V / 32)]``
    (:func:`pack_allowed`).  A row whose mask allows nothing is ``-inf`` throughout.  The gradient is that of x; the
    other arguments are constants.  On the GPU there is a first derivative in reverse mode, others are refused."""
    for t in (bias, repetition, presence, frequency):
        if isinstance(t, torch.Tensor) and t.requires_grad:
            raise ValueError("process_logits differentiates the logits only: detach bias and penalties")
    if not x.is_cuda:
        return process_logits_reference(x, history, lens, prompt_lens, rows, repetition, presence, frequency, bias, allowed)
    if unpack_dual(x).tangent is not None:
        raise ValueError("process_logits has no forward-mode derivative on the GPU")
    args = (history, lens, prompt_lens, rows, *_split(repetition), *_split(presence), *_split(frequency), bias, allowed)
    if x.requires_grad and torch.is_grad_enabled():
        return _ProcessLogits.apply(x, args)
    return _ext().process_logits(x, None, *args)
