"""Decoding a block of masked slots: a token for every slot, then the commit of the surest ones.

``sample_tokens`` draws one token per row of logits from given uniform numbers (temperature, top-k, top-p, min-p) and returns
with it what a denoising round ranks its slots by; ``unmask`` commits the best-ranked open slots of every sequence
(reference ``src/ttt/generate.py:227-355``: the proposals and the commit of one round; the reference draws by Gumbel noise and
has no truncation).  On a CUDA device both are one launch of ``csrc/sampling.cu``; elsewhere the statements of
``ops.reference`` run.  Neither is differentiable.
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
    priority: torch.Tensor        # f32: larger means surer


class Committed(NamedTuple):
    ids: torch.Tensor
    known: torch.Tensor
    logp: torch.Tensor            # the log-probability every slot was committed with
    where: torch.Tensor           # bool: the slots this call committed


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def _param(name: str, value: Param, rows, dtype: torch.dtype, device, lo: float, hi: float, open_lo: bool = False):
    """A checked number, or a tensor expanded to one value per row."""
    if torch.is_tensor(value) and (value.dim() > 0 or value.is_cuda):
        _need(value.device == device, f"sample_tokens: {name} is on {value.device}, the logits on {device}")
        whole = not (value.dtype.is_floating_point or value.dtype.is_complex or value.dtype == torch.bool)
        _need(whole if dtype == torch.int32 else value.dtype.is_floating_point, f"sample_tokens: {name} of {value.dtype}")
        try:
            value = value.clamp(-1, 2 ** 31 - 1) if value.dtype == torch.int64 else value
            return value.to(dtype).expand(rows).contiguous()
        except RuntimeError:
            raise ValueError(f"sample_tokens: {name} {tuple(value.shape)} does not broadcast to the rows {tuple(rows)}") from None
    v = value.item() if torch.is_tensor(value) else value
    _need((lo < v if open_lo else lo <= v) and v <= hi and math.isfinite(v),
          f"sample_tokens: {name} = {v!r} is outside {'(' if open_lo else '['}{lo}, {hi}]")
    return int(v) if dtype == torch.int32 else float(v)


@torch.no_grad()
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
    at -inf) gives token -1 and NaN.  ``V`` up to 393216 on a CUDA device."""
    _need(logits.dim() >= 2 and logits.shape[-1] > 0, f"sample_tokens: logits {tuple(logits.shape)}, at least [rows, V] are wanted")
    _need(logits.dtype in (torch.float32, torch.bfloat16, torch.float16), f"sample_tokens: logits of {logits.dtype}")
    _need(priority in PRIORITIES, f"sample_tokens: priority {priority!r} ({' | '.join(PRIORITIES)})")
    rows, V, dev = logits.shape[:-1], logits.shape[-1], logits.device
    _need(u.shape == rows and u.dtype == torch.float32 and u.device == dev,
          f"sample_tokens: u {tuple(u.shape)} {u.dtype} on {u.device}, {tuple(rows)} float32 on {dev} is wanted")
    if bias is not None:
        _need(bias.shape == (rows[0], V) and bias.dtype == torch.float32 and bias.device == dev,
              f"sample_tokens: bias {tuple(bias.shape)} {bias.dtype} on {bias.device}, {(rows[0], V)} float32 on {dev} is wanted")
    t = _param("temperature", temperature, rows, torch.float32, dev, 0.0, 1e6)
    k = _param("top_k", top_k, rows, torch.int32, dev, 0, 2 ** 31 - 1)
    p = _param("top_p", top_p, rows, torch.float32, dev, 0.0, 1.0, open_lo=True)
    m = _param("min_p", min_p, rows, torch.float32, dev, 0.0, 1.0)
    if not logits.is_cuda:
        full = lambda v, dtype: v.to(dtype) if torch.is_tensor(v) else torch.full(rows, v, dtype=dtype)
        return Drawn(*ref.sample_tokens(logits, u.nan_to_num(0.0), bias, full(t, torch.float64), full(k, torch.int64),
                                        full(p, torch.float64).nan_to_num(1.0), full(m, torch.float64).nan_to_num(0.0), priority))
    from . import kernels
    if not kernels.available("sampling"):
        raise RuntimeError("sample_tokens: the sampling kernels are not in the loaded library")
    _need(V <= kernels.SAMPLE_VOCAB_MAX, f"sample_tokens: V = {V} is above {kernels.SAMPLE_VOCAB_MAX}")
    x = logits if logits.stride(-1) == 1 or V == 1 else logits.contiguous()
    x = x.unsqueeze(1) if x.dim() == 2 else x.reshape(rows[0], math.prod(rows[1:]), V) if x.dim() > 3 else x
    flat = lambda v: v.reshape(x.shape[:2]).contiguous() if torch.is_tensor(v) else v
    out = kernels.sample(x, flat(u), None if bias is None else bias.contiguous(), flat(t), flat(k), flat(p), flat(m),
                         PRIORITIES.index(priority))
    return Drawn(*(o.view(rows) for o in out))


@torch.no_grad()
def unmask(ids: torch.Tensor, known: torch.Tensor, held: torch.Tensor, tokens: torch.Tensor, logp: torch.Tensor,
           priority: torch.Tensor, quota: torch.Tensor, *, allowed: Optional[torch.Tensor] = None,
           sure: Optional[float] = None) -> Committed:
    """Commit proposals into open slots: of every row of ``[B, C]`` the ``quota [B]`` slots of highest ``priority`` that are open
    (not ``known``, and ``allowed`` where given), and with ``sure`` also every slot that is not known and whose ``logp`` reaches
    it.  ``ids``, ``known`` and ``held`` (the log-probability a slot was committed with) come back with ``tokens`` / True /
    ``logp`` at the committed slots.  Slots of equal priority rank by position, NaN ranks last; a slot that is not open ranks as
    one of priority ``-inf``.  ``C`` up to 32768 on a CUDA device."""
    _need(ids.dim() == 2, f"unmask: ids {tuple(ids.shape)}, [B, C] is wanted")
    for name, t, dtype in (("ids", ids, torch.int64), ("known", known, torch.bool), ("held", held, torch.float32),
                           ("tokens", tokens, torch.int64), ("logp", logp, torch.float32), ("priority", priority, torch.float32),
                           ("allowed", allowed, torch.bool)):
        _need(t is None or (t.shape == ids.shape and t.dtype == dtype and t.device == ids.device),
              f"unmask: {name}: {tuple(ids.shape)} {dtype} on {ids.device} is wanted")
    _need(quota.shape == ids.shape[:1] and quota.dtype == torch.int64 and quota.device == ids.device,
          f"unmask: quota: {tuple(ids.shape[:1])} torch.int64 on {ids.device} is wanted")
    _need(sure is None or not math.isnan(sure), "unmask: sure is NaN")
    if not ids.is_cuda:
        return Committed(*ref.unmask(ids, known, held, tokens, logp, priority, quota, allowed, sure))
    from . import kernels
    if not kernels.available("sampling"):
        raise RuntimeError("unmask: the sampling kernels are not in the loaded library")
    _need(ids.shape[1] <= kernels.UNMASK_SLOTS_MAX, f"unmask: {ids.shape[1]} slots, above {kernels.UNMASK_SLOTS_MAX}")
    c = lambda t: None if t is None else t.contiguous()
    return Committed(*kernels.unmask(c(ids), c(known), c(held), c(tokens), c(logp), c(priority), c(quota), c(allowed), sure))
