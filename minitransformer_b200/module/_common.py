"""Concatenation of parameter views that avoids a copy when the views already sit back to
back in one buffer (what `parameters_split` creates; same role as
miniTransformer/module/_common.py:98-113), and the refusal of derivatives that a layer has none of."""
import functools
from typing import Optional, Sequence

import torch
from torch.autograd import forward_ad

from .._lib import MtError


def refuse_tangents(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """Raises where an input carries a forward-mode tangent: the kernels would lose it in silence."""
    if forward_ad._current_level < 0:            # outside of any dual level: no tensor has one
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise MtError(f"{what}: forward-mode derivatives are not implemented")


class _NoSecondDerivative(torch.autograd.Function):
    """Its inputs, with a gradient that is an error."""

    @staticmethod
    def forward(ctx, what, *grads):
        ctx.what = what
        return tuple(g.view_as(g) for g in grads)

    @staticmethod
    def backward(ctx, *_):
        raise MtError(f"{ctx.what}: second derivatives are not implemented")


def first_derivatives_only(what: str):
    """Decorator of an autograd function's backward whose kernels autograd cannot see into: with create_graph its results
    depend on the inputs and on the incoming gradient, and differentiating them raises instead of leaving that out."""
    def decorate(backward):
        @functools.wraps(backward)
        def run(ctx, *grads):
            if not torch.is_grad_enabled():
                return backward(ctx, *grads)
            with torch.no_grad():
                out = list(backward(ctx, *grads))
            # (an incoming gradient handed through keeps what it depends on)
            at = [i for i, t in enumerate(out) if t is not None and not any(t is g for g in grads)]
            if not at:
                return tuple(out)
            for i, t in zip(at, _NoSecondDerivative.apply(what, *(out[i].detach().requires_grad_() for i in at))):
                out[i] = t
            return tuple(out)
        return run
    return decorate


class _NoopCat(torch.autograd.Function):
    @staticmethod
    def forward(ctx, dim, *tensors):
        first = tensors[0]
        ctx.dim = dim
        ctx.sizes = [t.shape[dim] for t in tensors]
        if dim != 0 or not _adjacent(tensors):
            return torch.cat(tensors, dim=dim)
        shape = list(first.shape)
        shape[0] = sum(ctx.sizes)
        out = first.new_empty(0)
        out.set_(first.untyped_storage(), first.storage_offset(), shape, first.stride())
        return out

    @staticmethod
    def backward(ctx, grad):
        return (None, *torch.split(grad, ctx.sizes, dim=ctx.dim))


def _adjacent(tensors: Sequence[torch.Tensor]) -> bool:
    first = tensors[0]
    if not first.is_contiguous():
        return False
    ptr = first.data_ptr()
    for t in tensors:
        if (not t.is_contiguous() or t.dtype != first.dtype or t.device != first.device
                or t.shape[1:] != first.shape[1:] or t.data_ptr() != ptr
                or t.untyped_storage().data_ptr() != first.untyped_storage().data_ptr()):
            return False
        ptr += t.numel() * t.element_size()
    return True


def noop_cat(tensors: Sequence[torch.Tensor], dim: int = 0) -> torch.Tensor:
    if not tensors:
        raise ValueError("noop_cat needs at least one tensor")
    if len(tensors) == 1:
        return tensors[0]
    return _NoopCat.apply(dim, *tensors)


_STACKED_OK: dict = {}


def stacked_view(tensors: Sequence[torch.Tensor]):
    """[len(tensors), *shape] view over tensors that sit back to back in one buffer (expert
    weights allocated from one block, or their main_grad buffers), or None when they do not."""
    if not tensors:
        return None
    # the full adjacency walk (contiguity, storage, dtype per tensor) is remembered per set of
    # tensors at these exact addresses: every address is part of the key, so re-pointing any
    # one of them (`.data = ...`, a replaced main_grad) is noticed
    first = tensors[0]
    key = (tuple(t.data_ptr() for t in tensors), tuple(first.shape), tuple(first.stride()), first.dtype,
           first.device)
    ok = _STACKED_OK.get(key)
    if ok is None:
        ok = _adjacent(tensors)
        if len(_STACKED_OK) >= 64:
            _STACKED_OK.clear()
        _STACKED_OK[key] = ok
    if not ok:
        return None
    out = first.detach().new_empty(0)
    out.set_(first.untyped_storage(), first.storage_offset(), [len(tensors), *first.shape],
             [first.numel(), *first.stride()])
    return out
