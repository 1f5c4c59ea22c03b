"""Argument and autograd helpers."""

import functools
from typing import Any, List, Tuple, Union

import torch

__all__ = ["make_ntuple", "once_differentiable"]


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
