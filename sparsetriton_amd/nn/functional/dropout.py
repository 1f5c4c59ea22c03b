"""Dropout of features with the residual add, its mask made from a counter and never stored (HIP kernel
``st_dropout``; no counterpart in the reference)."""

from typing import Optional, Union

import torch

from sparsetriton_amd import _lib
from sparsetriton_amd.tensor import SparseTensor
from sparsetriton_amd.utils.utils import refuse_tangents

__all__ = ["sparse_dropout"]


def _drop(x, residual, numbers, p):
    x = x.contiguous()
    res = residual.contiguous() if residual is not None else None
    y = torch.empty_like(x)
    _lib.call_on(x.device, "st_dropout", x.data_ptr(), _lib.ptr(res), x.numel(), _lib.FEAT_DTYPES[x.dtype],
                 numbers.data_ptr(), p, y.data_ptr())
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, numbers, p):
        ctx.save_for_backward(numbers)
        ctx.p = p
        return _drop(x, residual, numbers, p)

    @staticmethod
    def backward(ctx, dy):
        (numbers,) = ctx.saved_tensors
        dx = None
        if ctx.needs_input_grad[0]:  # (linear in dy: the same operator, so that a gradient of the gradient is one too)
            dx = (_Dropout.apply if torch.is_grad_enabled() else _drop)(dy, None, numbers, ctx.p)
        return dx, dy if ctx.needs_input_grad[1] else None, None, None


def sparse_dropout(
    input: Union[SparseTensor, torch.Tensor],
    p: float = 0.5,
    training: bool = True,
    residual: Optional[Union[SparseTensor, torch.Tensor]] = None,
    numbers: Optional[torch.Tensor] = None,
) -> Union[SparseTensor, torch.Tensor]:
    """``input / (1 - p)`` where an element is kept, zero (whatever it holds) with probability ``p``,
    plus ``residual`` (same shape and dtype) in the same pass: ``residual + dropout(input)``.

    ``input`` (and ``residual``) are a ``SparseTensor`` or a tensor of float32, float16 or bfloat16;
    the result is of the same kind as ``input``, computed in fp32 and rounded once.  Without
    ``training``, or with ``p = 0``, nothing is dropped (and no numbers are drawn).

    Which elements are kept follows from ``numbers``, two int64 on the input's device, and each
    element's index: the same numbers give the same mask, in any type, and the backward makes it again from them.
    By default they are drawn from torch's generator of the device, so ``torch.manual_seed``,
    activation checkpointing and graph capture (each replay draws anew) work as they do for torch's
    own dropout.  Given numbers belong to one call: use others for the next one, and do not
    change them in place before its backward.  There is no forward-mode derivative: a tangent on an
    input raises.
    """
    x = input.F if isinstance(input, SparseTensor) else input
    res = residual.F if isinstance(residual, SparseTensor) else residual
    _lib.require_device(x, "dropout input")
    _lib.feat_code(x.dtype)
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout needs a probability (got p = {p})")
    if res is not None and (res.shape != x.shape or res.dtype != x.dtype or res.device != x.device):
        raise ValueError("the residual must match the input's shape, dtype and device")
    if numbers is not None:
        if numbers.dtype != torch.int64:
            raise TypeError(f"numbers must be int64 (got {numbers.dtype})")
        if numbers.shape != (2,) or numbers.device != x.device:
            raise ValueError(f"numbers must be (2,) on {x.device} (got {tuple(numbers.shape)} on {numbers.device})")
    refuse_tangents("sparse_dropout", x, res)
    if not training or p == 0.0:
        y = x if res is None else res + x
    else:
        if numbers is None:
            numbers = torch.empty((2,), dtype=torch.int64, device=x.device).random_()
        numbers = numbers.contiguous()
        if torch.is_grad_enabled() and (x.requires_grad or (res is not None and res.requires_grad)):
            y = _Dropout.apply(x, res, numbers, p)
        else:
            y = _drop(x, res, numbers, p)
    return input.replace(y) if isinstance(input, SparseTensor) else y
