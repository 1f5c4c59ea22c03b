"""Argument and autograd helpers."""

import functools
from typing import Any, List, Tuple, Union

import torch
from torch.autograd import forward_ad

__all__ = ["make_ntuple", "once_differentiable", "refuse_tangents"]


def make_ntuple(value: Union[int, float, Tuple[Any, ...], List[Any]], n: int) -> Tuple[Any, ...]:
    """Expand a scalar to an n-tuple; truncate or right-pad (with the last item) a sequence.

    Same behaviour as ``sparsetriton/utils/utils.py:17-47``.
    """
    if isinstance(value, (list, tuple)):
        if len(value) >= n:
            return tuple(value[:n])
        return tuple(value) + (value[-1],) * (n - len(value))
    if isinstance(value, (int, float)):
        return (value,) * n
    raise TypeError(f"Expected int, float, tuple, or list, got {type(value)}")


def once_differentiable(backward):
    """``torch.autograd.function.once_differentiable`` that costs nothing where no graph of the
    gradients is asked for (grad mode is then off in a backward pass)."""
    checked = torch.autograd.function.once_differentiable(backward)

    @functools.wraps(backward)
    def run(ctx, *grads):
        return checked(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


def refuse_tangents(what: str, *tensors) -> None:
    """Raise where one of ``tensors`` (``None`` among them) carries a forward-mode tangent: the kernels read values
    alone, and a result without a tangent would count as one whose derivative is zero."""
    if getattr(forward_ad, "_current_level", 0) < 0:  # (outside every level: next to nothing a call)
        return
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"sparsetriton_amd: {what} has no forward-mode derivative; use reverse mode")
