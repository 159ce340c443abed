"""Decoding a block of masked slots: a token for every slot, then the commit of the surest ones.

``sample_tokens`` draws one token per row of logits from given uniform numbers (temperature, top-k, top-p, min-p) and returns
with it what a denoising round ranks its slots by; ``unmask`` commits the best-ranked open slots of every sequence
(reference ``src/ttt/generate.py:227-355``: the proposals and the commit of one round; the reference draws by Gumbel noise and
has no truncation).  On a CUDA device both are kernels of ``csrc/sampling.cu``, one launch a call, or two and a scratch area for
untruncated draws from 6.2 million elements on; elsewhere the statements of ``ops.reference`` run.  Neither is differentiable.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Union

import torch

from . import reference as ref

PRIORITIES = ("logp", "margin", "entropy")
Param = Union[float, int, torch.Tensor]


class Drawn(NamedTuple):
    tokens: torch.Tensor          # int64 [...]
    logp: torch.Tensor            # f32: log-probability of the token under the untempered, untruncated distribution
    priority: torch.Tensor        # f32: larger means surer (ranked by logp, it may be the same tensor)


class Committed(NamedTuple):
    ids: torch.Tensor
    known: torch.Tensor
    logp: torch.Tensor            # the log-probability every slot was committed with
    where: torch.Tensor           # bool: the slots this call committed


def _param(name: str, value: Param, rows, dtype: torch.dtype, device, lo: float, hi: float, open_lo: bool = False):
    """A checked number, or a tensor expanded to one value per row."""
    if isinstance(value, torch.Tensor) and (value.dim() > 0 or value.is_cuda):
        if value.device != device:
            raise ValueError(f"sample_tokens: {name} is on {value.device}, the logits on {device}")
        whole = not (value.dtype.is_floating_point or value.dtype.is_complex or value.dtype == torch.bool)
        if not (whole if dtype == torch.int32 else value.dtype.is_floating_point):
            raise ValueError(f"sample_tokens: {name} of {value.dtype}")
        try:
            value = value.detach().clamp(-1, 2 ** 31 - 1) if value.dtype == torch.int64 else value.detach()
            return value.to(dtype).expand(rows).contiguous()
        except RuntimeError:
            raise ValueError(f"sample_tokens: {name} {tuple(value.shape)} does not broadcast to the rows {tuple(rows)}") from None
    v = value.item() if isinstance(value, torch.Tensor) else value
    if not ((lo < v if open_lo else lo <= v) and v <= hi) or (dtype == torch.int32 and v != int(v)):
        whole = " whole numbers of" if dtype == torch.int32 else ""
        raise ValueError(f"sample_tokens: {name} = {v!r} is outside{whole} {'(' if open_lo else '['}{lo}, {hi}]")
    return int(v) if dtype == torch.int32 else float(v)


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, *, temperature: Param = 1.0, top_k: Param = 0, top_p: Param = 1.0,
                  min_p: Param = 0.0, bias: Optional[torch.Tensor] = None, priority: str = "logp") -> Drawn:
    """One token per row of ``logits [..., V]`` (f32, bf16 or f16; two or more dimensions), drawn with ``u [...]`` (f32 in [0, 1)).

    ``x = logits + bias[:, None]`` in f32 (``bias [logits.shape[0], V]`` f32: presence penalties, bans as ``-inf``).  With
    ``w = exp((x - max x) / temperature)`` and the tokens ordered by descending ``x`` (lowest index first among equals), the draw
    keeps the first ``top_k`` (0: all), of those the shortest prefix holding ``top_p`` of their mass, and of those the ones with
    ``w >= min_p``; the token is the first kept one, in index order, at which the running mass exceeds ``u`` times the kept
    mass.  ``temperature = 0`` takes the lowest index of the maximum.  ``logp`` and the ``priority`` (``logp``; ``margin``: the
    difference of the two largest probabilities; ``entropy``: ``sum p log p``) are those of ``softmax(x)``.

    Every parameter is a number for all rows or a tensor that broadcasts to the rows.  Numbers are checked; values in tensors are
    not read by the host and are taken as ``temperature <= 0``: greedy, else clamped to [1e-6, 1e6]; ``top_k <= 0`` or ``>= V``:
    off; ``top_p >= 1``: off, ``<= 0``: the best token alone; ``min_p <= 0``: off, above 1: as 1; NaN: as off (``temperature``:
    greedy).  ``u`` outside [0, 1) is clamped, NaN taken as 0.  A row without a distribution (NaN or +inf in it, or every token
    at -inf) gives token -1 and NaN: no index, so look for it before the tokens are embedded or scattered by.  On a CUDA device
    ``V`` goes up to 393216."""
    rows, dev = logits.shape[:-1], logits.device
    if not rows or logits.shape[-1] == 0:
        raise ValueError(f"sample_tokens: logits {tuple(logits.shape)}, at least [rows, V] are wanted")
    V = logits.shape[-1]
    if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError(f"sample_tokens: logits of {logits.dtype}")
    if priority not in PRIORITIES:
        raise ValueError(f"sample_tokens: priority {priority!r} ({' | '.join(PRIORITIES)})")
    if u.shape != rows or u.dtype != torch.float32 or u.device != dev:
        raise ValueError(f"sample_tokens: u {tuple(u.shape)} {u.dtype} on {u.device}, {tuple(rows)} float32 on {dev} is wanted")
    if bias is not None and (bias.shape != (rows[0], V) or bias.dtype != torch.float32 or bias.device != dev):
        raise ValueError(f"sample_tokens: bias {tuple(bias.shape)} {bias.dtype} on {bias.device}, {(rows[0], V)} float32 on {dev} is wanted")
    t, k, p, m = temperature, top_k, top_p, min_p
    if not (type(t) is float and 0.0 <= t <= 1e6):
        t = _param("temperature", t, rows, torch.float32, dev, 0.0, 1e6)
    if not (type(k) is int and 0 <= k < 2 ** 31):
        k = _param("top_k", k, rows, torch.int32, dev, 0, 2 ** 31 - 1)
    if not (type(p) is float and 0.0 < p <= 1.0):
        p = _param("top_p", p, rows, torch.float32, dev, 0.0, 1.0, open_lo=True)
    if not (type(m) is float and 0.0 <= m <= 1.0):
        m = _param("min_p", m, rows, torch.float32, dev, 0.0, 1.0)
    from . import kernels
    if not logits.is_cuda or "sampling" in kernels._DISABLED:
        with torch.no_grad():
            full = lambda v, dtype: v.to(dtype) if isinstance(v, torch.Tensor) else torch.full(rows, v, dtype=dtype, device=dev)
            return Drawn(*ref.sample_tokens(logits, u.nan_to_num(0.0), bias, full(t, torch.float64), full(k, torch.int64),
                                            full(p, torch.float64).nan_to_num(1.0), full(m, torch.float64).nan_to_num(0.0), priority))
    if V > kernels.SAMPLE_VOCAB_MAX:
        raise ValueError(f"sample_tokens: V = {V} is above {kernels.SAMPLE_VOCAB_MAX}")
    x = logits if logits.stride(-1) == 1 or V == 1 else logits.detach().contiguous()
    if len(rows) != 2:
        x = x.unsqueeze(1) if len(rows) == 1 else x.reshape(rows[0], math.prod(rows[1:]), V)
    return Drawn(*kernels.sample(x, u.detach().contiguous() if u.requires_grad else u.contiguous(),
                                 None if bias is None else bias.contiguous(), t, k, p, m, PRIORITIES.index(priority)))


def unmask(ids: torch.Tensor, known: torch.Tensor, held: torch.Tensor, tokens: torch.Tensor, logp: torch.Tensor,
           priority: torch.Tensor, quota: torch.Tensor, *, allowed: Optional[torch.Tensor] = None,
           sure: Optional[float] = None) -> Committed:
    """Commit proposals into open slots: of every row of ``[B, C]`` the ``quota [B]`` slots of highest ``priority`` that are open
    (not ``known``, and ``allowed`` where given), and with ``sure`` also every slot that is not known and whose ``logp`` reaches
    it.  ``ids``, ``known`` and ``held`` (the log-probability a slot was committed with) come back with ``tokens`` / True /
    ``logp`` at the committed slots.  Slots of equal priority rank by position, NaN ranks last; a slot that is not open ranks as
    one of priority ``-inf``.  Tokens are copied as they are (a -1 of ``sample_tokens`` too).  One launch for
    ``C`` up to 32768 on a CUDA device, the statement of ``ops.reference`` beyond."""
    shape, dev = ids.shape, ids.device
    if len(shape) != 2:
        raise ValueError(f"unmask: ids {tuple(shape)}, [B, C] is wanted")
    for name, t, dtype in (("ids", ids, torch.int64), ("known", known, torch.bool), ("held", held, torch.float32),
                           ("tokens", tokens, torch.int64), ("logp", logp, torch.float32), ("priority", priority, torch.float32),
                           ("allowed", allowed, torch.bool)):
        if t is not None and (t.shape != shape or t.dtype != dtype or t.device != dev):
            raise ValueError(f"unmask: {name} {tuple(t.shape)} {t.dtype} on {t.device}, {tuple(shape)} {dtype} on {dev} is wanted")
    if quota.shape != shape[:1] or quota.dtype != torch.int64 or quota.device != dev:
        raise ValueError(f"unmask: quota {tuple(quota.shape)} {quota.dtype} on {quota.device}, {tuple(shape[:1])} torch.int64 on {dev} is wanted")
    if sure is not None and math.isnan(sure):
        raise ValueError("unmask: sure is NaN")
    from . import kernels
    if not ids.is_cuda or "sampling" in kernels._DISABLED or shape[1] > kernels.UNMASK_SLOTS_MAX:
        with torch.no_grad():
            return Committed(*ref.unmask(ids, known, held, tokens, logp, priority, quota, allowed, sure))
    return Committed(*kernels.unmask(ids.contiguous(), known.contiguous(), held.contiguous(), tokens.contiguous(), logp.contiguous(),
                                     priority.contiguous(), quota.contiguous(), None if allowed is None else allowed.contiguous(), sure))
