"""Newton-Schulz orthogonalisation of an update, the direction of the ``muon5`` write (``ttt.inner.direction``).

``newton_schulz(g)`` drives the singular values of every matrix of ``g [..., rows, cols]`` toward one: from
``x = g / |g|_F``, ``steps`` times ``x <- a x + (b G + c G G) x`` with ``G = x x^T`` on the smaller side and the coefficients of
the inner step (reference ``src/ttt/inner_loop.py:350-397``, which runs two iterations in bf16).  On a CUDA device the products
run on the tensor cores with f16 operands and f32 sums (``csrc/newton_schulz.cu``); elsewhere in f32.

The result is the linear map ``g -> M g / |g|`` with a symmetric polynomial ``M`` of the matrix; as in the reference, ``M`` is held
constant by the derivative, and so is the norm: the backward applies the same map to the cotangent, and so does the
backward's own backward.  Along ``g`` itself that is not the slope of the result, which does not depend on the scale of ``g``; a use
that needs it projects the component along ``g`` out of the backward's result (the write does, ``ttt.inner.direction``).
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import reference as ref


def _flat(t: torch.Tensor) -> torch.Tensor:
    t = t if t.dtype in (torch.float32, torch.bfloat16) else t.float()
    t = t if t.dim() == 3 else t.reshape(-1, *t.shape[-2:])
    return t if t.is_contiguous() else t.contiguous()


def _linear(r: torch.Tensor, norms, maps, steps: int, dtype: torch.dtype) -> torch.Tensor:
    """``M r / |g|`` with what a forward kept of ``g``."""
    if isinstance(maps, list):
        return ref.newton_schulz_apply(r, norms, maps).to(dtype)
    from . import kernels
    return kernels.newton_schulz_apply(_flat(r), norms, maps, steps, dtype).view(r.shape)


def _maps(saved, listed: bool):
    """Norms and maps as ``_run`` gave them, from what a context saved."""
    norms, *maps = saved
    return norms, (maps if listed else maps[0])


class _Apply(torch.autograd.Function):
    """``_linear`` as a differentiable operation: linear and self-adjoint."""

    @staticmethod
    def forward(ctx, r, steps, dtype, listed, *kept):
        ctx.save_for_backward(*kept)
        ctx.steps, ctx.listed, ctx.dtype = steps, listed, r.dtype
        return _linear(r, *_maps(kept, listed), steps, dtype)

    @staticmethod
    def backward(ctx, c):
        kept = ctx.saved_tensors
        return (_Apply.apply(c, ctx.steps, ctx.dtype, ctx.listed, *kept), None, None, None, *[None] * len(kept))


class _NewtonSchulz(torch.autograd.Function):
    @staticmethod
    def forward(ctx, g, steps):
        y, norms, maps = _run(g, steps, True)
        ctx.steps, ctx.listed, ctx.dtype = steps, isinstance(maps, list), g.dtype
        ctx.save_for_backward(norms, *(maps if ctx.listed else (maps,)))
        return y

    @staticmethod
    def backward(ctx, gy):
        kept = ctx.saved_tensors
        if torch.is_grad_enabled():
            return _Apply.apply(gy, ctx.steps, ctx.dtype, ctx.listed, *kept), None
        return _linear(gy, *_maps(kept, ctx.listed), ctx.steps, ctx.dtype), None


def _run(g: torch.Tensor, steps: int, keep: bool):
    from . import kernels
    if not g.is_cuda or "newton_schulz" in kernels._DISABLED:
        y, norms, polys = ref.newton_schulz(g, steps)
        return y.to(torch.bfloat16), norms, polys
    y, norms, maps = kernels.newton_schulz(_flat(g), steps, keep)
    return y.view(g.shape), norms, maps


def newton_schulz(g: torch.Tensor, steps: int = 5) -> torch.Tensor:
    """The orthogonalised direction of every matrix of ``g [..., rows, cols]`` (f32 or bf16), in bf16.

    The norms are taken in 64 bits, so any finite scale of ``g`` will do; a zero matrix gives zeros (and a zero derivative), one
    that holds NaN or infinities gives NaN.  On a CUDA device the products take f16 operands, with what ``x`` loses by that carried
    along: after five steps the result is off by 2e-3 to 4e-3 in the 2-norm, of which its own type 1.7e-3, whatever the rank of
    ``g``; where a matrix has no singular value a step multiplies what it holds there by 3.4445, in any arithmetic, so that the 2^-22
    left of ``x`` come to a tenth of the result after twelve steps (an f32 computation's 2^-24 after thirteen).  The derivative has the
    accuracy of bf16 whatever the type of ``g``.  The same matrix may come out with other last bits in a batch of another size.
    At most 65535 matrices a call; no forward-mode derivative; the first call on a device cannot be captured into a graph."""
    if g.dim() < 2 or g.shape[-1] == 0 or g.shape[-2] == 0:
        raise ValueError(f"newton_schulz: g {tuple(g.shape)}, [..., rows, cols] with non-empty matrices is wanted")
    if g.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"newton_schulz: g of {g.dtype} (float32 or bfloat16)")
    if isinstance(steps, bool) or not isinstance(steps, int) or not 1 <= steps <= 32:
        raise ValueError(f"newton_schulz: steps = {steps!r}, a number from 1 to 32 is wanted")
    if g.numel() // (g.shape[-1] * g.shape[-2]) > 65535:
        raise ValueError(f"newton_schulz: {g.numel() // (g.shape[-1] * g.shape[-2])} matrices, at most 65535 are taken in one call")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(g).tangent is not None:
        raise NotImplementedError("newton_schulz: there is no forward-mode derivative (a dual tensor would lose its tangent)")
    if g.numel() == 0:
        return g.to(torch.bfloat16)
    if torch.is_grad_enabled() and g.requires_grad:
        return _NewtonSchulz.apply(g, steps)
    return _run(g, steps, False)[0]
