"""Rotary positions of queries and keys over the axes of the voxel grid (HIP kernel ``st_rotary``).

No counterpart in the reference.  A head's first ``sum(axes)`` channels are paired; the pairs are
dealt to the axes in order (``axes[a] // 2`` pairs to axis ``a``), and pair ``i`` of axis ``a``
turns by ``position[a] * base ** (-2 i / axes[a])`` radians, the frequency rounded to fp32.
"""

import ctypes
import math
from typing import Optional, Sequence, Tuple, Union

import torch

from sparsetriton_amd import _lib
from sparsetriton_amd.tensor import SparseTensor

__all__ = ["RotaryAxes", "sparse_rotary"]


class RotaryAxes:
    """Which channel pairs of a head turn with which axis, and how fast.

    ``head_dim`` channels a head, ``axes`` the even number of them that each axis turns (their sum
    at most ``head_dim``; the channels after them keep no position), ``base`` of the frequencies,
    ``interleaved`` for pairs (2p, 2p + 1) in place of (p, p + sum(axes) / 2).  A program keeps one
    beside its weights: the device copy of the frequencies is made at the first call on a device.
    """

    def __init__(self, head_dim: int, axes: Sequence[int], base: float = 10000.0, interleaved: bool = False) -> None:
        self.head_dim, self.axes, self.base = int(head_dim), tuple(int(a) for a in axes), float(base)
        self.interleaved = bool(interleaved)
        if not self.axes or any(a < 0 or a % 2 for a in self.axes):
            raise ValueError(f"each axis turns an even number of channels (got {self.axes})")
        if sum(self.axes) > self.head_dim:
            raise ValueError(f"the axes turn {sum(self.axes)} channels of a head of {self.head_dim}")
        if not (self.base > 0 and math.isfinite(self.base)):
            raise ValueError(f"base must be positive and finite (got {base})")
        self.pairs = sum(self.axes) // 2
        freq = [self.base ** (-2.0 * i / a) for a in self.axes for i in range(a // 2)]
        self.frequencies = torch.tensor(freq, dtype=torch.float64).to(torch.float32)
        self._turns = self.frequencies.double() / (2.0 * math.pi)
        self._axis = torch.tensor([i for i, a in enumerate(self.axes) for _ in range(a // 2)], dtype=torch.int32)
        self._on = {}

    def on(self, device: torch.device) -> Tuple[torch.Tensor, torch.Tensor]:
        """(whole turns per unit, axis) of each pair on ``device``."""
        got = self._on.get(device)
        if got is None:
            got = self._on[device] = (self._turns.to(device), self._axis.to(device))
        return got

    def __getstate__(self):
        return {**self.__dict__, "_on": {}}


def _rotate(q, k, positions, axes, inverse):
    dev = (q if q is not None else k).device
    turns, axis = axes.on(dev)
    out = [torch.empty(t.shape, dtype=t.dtype, device=dev) if t is not None else None for t in (q, k)]
    # channels side by side; rows and heads at any stride
    q, k = (t if t is None or t.stride(2) == 1 else t.contiguous() for t in (q, k))
    qp = kp = qo = ko = None
    qs = ks = (0, 0, 0)
    heads = kv_heads = 0
    if q is not None:
        qp, qo, qs, heads = q.data_ptr(), out[0].data_ptr(), q.stride(), q.shape[1]
    if k is not None:
        kp, ko, ks, kv_heads = k.data_ptr(), out[1].data_ptr(), k.stride(), k.shape[1]
    n, _, dim = (q if q is not None else k).shape
    a = _lib.RotaryArgs(qp, kp, qo, ko, qs[0], qs[1], ks[0], ks[1], positions.data_ptr(), positions.stride(0),
                        turns.data_ptr(), axis.data_ptr(), n, heads, kv_heads, dim, axes.pairs,
                        _lib.FEAT_DTYPES[out[0 if q is not None else 1].dtype], _lib.POSITION_DTYPES[positions.dtype],
                        axes.interleaved, inverse)
    _lib.call("st_rotary", ctypes.byref(a), _lib.stream_of(dev))
    return tuple(out)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, axes):
        ctx.save_for_backward(positions)
        ctx.axes = axes
        ctx.set_materialize_grads(False)
        return _rotate(q, k, positions, axes, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        (positions,) = ctx.saved_tensors
        dq = dq if ctx.needs_input_grad[0] else None
        dk = dk if ctx.needs_input_grad[1] else None
        if dq is not None or dk is not None:
            dq, dk = _rotate(dq, dk, positions, ctx.axes, True)
        return dq, dk, None, None


def sparse_rotary(
    q: Optional[torch.Tensor],
    k: Optional[torch.Tensor],
    positions: Union[SparseTensor, torch.Tensor],
    axes: RotaryAxes,
) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """``(q, k)`` with each head's channel pairs turned by the row's position.

    ``q`` (N, heads, D) and ``k`` (N, kv_heads, D) share rows and dtype (one of them may be
    ``None``); rows and heads may lie at any stride.  ``positions``: a ``SparseTensor`` (the x, y, z
    of its coordinates) or (N, A) of int16, int32, int64 or float32 with ``A >= len(axes.axes)``.
    The outputs are contiguous; the gradient turns back.  Positions get no gradient.
    """
    given = [t for t in (q, k) if t is not None]
    if not given:
        raise ValueError("sparse_rotary needs q or k")
    pos = positions.C[:, 1:] if isinstance(positions, SparseTensor) else positions
    first = given[0]
    for t in given:
        _lib.require_device(t, "rotary input")
        _lib.feat_code(t.dtype)
        if t.dim() != 3 or t.shape[2] != axes.head_dim or t.shape[1] == 0:
            raise ValueError(f"expected (rows, heads, {axes.head_dim}), got {tuple(t.shape)}")
        if t.shape[0] != first.shape[0] or t.dtype != first.dtype or t.device != first.device:
            raise ValueError("q and k must have the same rows, dtype and device")
    if pos.dim() != 2 or pos.shape[0] != first.shape[0] or pos.shape[1] < len(axes.axes):
        raise ValueError(f"positions must be ({first.shape[0]}, at least {len(axes.axes)}), got {tuple(pos.shape)}")
    if pos.dtype not in _lib.POSITION_DTYPES:
        raise TypeError(f"unsupported position dtype {pos.dtype}; use int16, int32, int64 or float32")
    if pos.device != first.device:
        raise ValueError(f"positions are on {pos.device}, q and k on {first.device}")
    pos = pos.detach()
    if pos.shape[1] > 1 and pos.stride(1) != 1:
        pos = pos.contiguous()
    if torch.is_grad_enabled() and any(t.requires_grad for t in given):
        return _Rotary.apply(q, k, pos, axes)
    return _rotate(q, k, pos, axes, False)
