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
from sparsetriton_amd.utils.utils import once_differentiable, refuse_tangents

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
            got = self._on[device] = [self._turns.to(device), self._axis.to(device), None]
        turns, axis, last = got
        if turns.is_cuda:
            s = _lib.stream_of(device)
            if s != last:  # (their memory is not handed out before this stream is through with it)
                for t in (turns, axis):
                    t.record_stream(torch.cuda.current_stream(device))
                got[2] = s
        return turns, axis

    def __getstate__(self):
        return {**self.__dict__, "_on": {}}


def _rotate(q, k, positions, axes, inverse):
    dev = (q if q is not None else k).device
    turns, axis = axes.on(dev)
    qp = kp = qo = ko = q_out = k_out = None
    qs = ks = (0, 0, 0)
    heads = kv_heads = 0
    # channels side by side; rows and heads at any stride
    if q is not None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        if q.stride(2) != 1:
            q = q.contiguous()
        qp, qo, qs, heads = q.data_ptr(), q_out.data_ptr(), q.stride(), q.shape[1]
    if k is not None:
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
        if k.stride(2) != 1:
            k = k.contiguous()
        kp, ko, ks, kv_heads = k.data_ptr(), k_out.data_ptr(), k.stride(), k.shape[1]
    t = q if q is not None else k
    n, _, dim = t.shape
    a = _lib.RotaryArgs(qp, kp, qo, ko, qs[0], qs[1], ks[0], ks[1], positions.data_ptr(), positions.stride(0),
                        turns.data_ptr(), axis.data_ptr(), n, heads, kv_heads, dim, axes.pairs,
                        _lib.FEAT_DTYPES[t.dtype], _lib.POSITION_DTYPES[positions.dtype],
                        axes.interleaved, inverse)
    _lib.call("st_rotary", ctypes.byref(a), _lib.stream_of(dev))
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, axes):
        ctx.save_for_backward(positions)
        ctx.axes = axes
        ctx.set_materialize_grads(False)
        return _rotate(q, k, positions, axes, False)

    @staticmethod
    @once_differentiable
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
    The outputs are contiguous; the gradient turns back.  Positions get no gradient.  There is no
    forward-mode derivative: a tangent on ``q`` or ``k`` raises.
    """
    first = q if q is not None else k
    if first is None:
        raise ValueError("sparse_rotary needs q or k")
    pos = positions.C[:, 1:] if isinstance(positions, SparseTensor) else positions
    for t in (first,) if q is None or k is None else (q, k):
        if not t.is_cuda:
            _lib.require_device(t, "rotary input")
        if t.dtype not in _lib.FEAT_DTYPES:
            _lib.feat_code(t.dtype)
        if t.dim() != 3 or t.shape[2] != axes.head_dim or t.shape[1] == 0:
            raise ValueError(f"expected (rows, heads, {axes.head_dim}), got {tuple(t.shape)}")
        if t is not first and (t.shape[0] != first.shape[0] or t.dtype is not first.dtype or t.device != first.device):
            raise ValueError("q and k must have the same rows, dtype and device")
    if pos.dim() != 2 or pos.shape[0] != first.shape[0] or pos.shape[1] < len(axes.axes):
        raise ValueError(f"positions must be ({first.shape[0]}, at least {len(axes.axes)}), got {tuple(pos.shape)}")
    if pos.dtype not in _lib.POSITION_DTYPES:
        raise TypeError(f"unsupported position dtype {pos.dtype}; use int16, int32, int64 or float32")
    if pos.device != first.device:
        raise ValueError(f"positions are on {pos.device}, q and k on {first.device}")
    if pos.shape[1] > 1 and pos.stride(1) != 1:
        pos = pos.contiguous()
    refuse_tangents("sparse_rotary", q, k)
    if torch.is_grad_enabled() and ((q is not None and q.requires_grad) or (k is not None and k.requires_grad)):
        return _Rotary.apply(q, k, pos.detach(), axes)
    return _rotate(q, k, pos, axes, False)
