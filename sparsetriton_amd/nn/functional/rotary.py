"""Rotary positions of queries and keys over the axes of the voxel grid (HIP kernel ``st_rotary``), and the
same after a norm of each head, in one pass (``st_qk_norm_rotary``).

No counterpart in the reference.  A head's first ``sum(axes)`` channels are paired; the pairs are
dealt to the axes in order (``axes[a] // 2`` pairs to axis ``a``), and pair ``i`` of axis ``a``
turns by ``position[a] * base ** (-2 i / axes[a])`` radians, the frequency rounded to fp32.
"""

import ctypes
import math
from typing import Optional, Sequence, Tuple, Union

import torch

from sparsetriton_amd import _lib
from sparsetriton_amd.nn.functional.norm import _ln_params
from sparsetriton_amd.tensor import SparseTensor
from sparsetriton_amd.utils.utils import once_differentiable, refuse_tangents

__all__ = ["RotaryAxes", "sparse_rotary", "sparse_qk_norm_rotary"]


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


def _check(what, q, k, positions, axes):
    """The positions as the kernels take them, (rows, at least as many as the axes)."""
    first = q if q is not None else k
    if first is None:
        raise ValueError(f"{what} needs q or k")
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
    return pos


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
    pos = _check("sparse_rotary", q, k, positions, axes)
    refuse_tangents("sparse_rotary", q, k)
    if torch.is_grad_enabled() and ((q is not None and q.requires_grad) or (k is not None and k.requires_grad)):
        return _Rotary.apply(q, k, pos.detach(), axes)
    return _rotate(q, k, pos, axes, False)


def _flat(t):
    """(t, its strides, heads): a contiguous copy where a head's channels are apart or a row's heads past the kernels'
    32-bit offsets."""
    if t is None:
        return None, (0, 0), 0
    strides, heads = t.stride(), t.shape[1]
    if strides[2] != 1 or (strides[0] + heads * strides[1]) * t.element_size() > _lib.QK_REACH:
        t = t.clone(memory_format=torch.contiguous_format)
        strides = t.stride()
    return t, strides, heads


def _qk_args(q, k, q_weight, k_weight, positions, axes, eps):
    """(arguments of both directions, the tensors that they point to)."""
    t = q if q is not None else k
    turns, axis = axes.on(t.device)
    (q, qs, heads), (k, ks, kv_heads) = _flat(q), _flat(k)
    wq, wk, wcode = _ln_params(t, q_weight, k_weight)
    ptr = _lib.ptr
    a = _lib.QkNormArgs(ptr(q), ptr(k), None, None, qs[0], qs[1], ks[0], ks[1], ptr(wq), ptr(wk), positions.data_ptr(),
                        positions.stride(0), turns.data_ptr(), axis.data_ptr(), t.shape[0], heads, kv_heads, t.shape[2],
                        axes.pairs, _lib.FEAT_DTYPES[t.dtype], wcode, _lib.POSITION_DTYPES[positions.dtype],
                        axes.interleaved)
    a.eps = eps
    return a, (q, k, wq, wk)


def _qk_forward(q, k, q_weight, k_weight, positions, axes, eps):
    a, held = _qk_args(q, k, q_weight, k_weight, positions, axes, eps)
    q_out = k_out = None
    if q is not None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        a.q_out = q_out.data_ptr()
    if k is not None:
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
        a.k_out = k_out.data_ptr()
    _lib.call_on(positions.device, "st_qk_norm_rotary", ctypes.byref(a))
    return q_out, k_out, held


class _QkNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, axes, eps):
        q_out, k_out, held = _qk_forward(q, k, q_weight, k_weight, positions, axes, eps)
        ctx.save_for_backward(*held, positions)
        ctx.meta = (axes, eps, [None if w is None else w.dtype for w in (q_weight, k_weight)])
        ctx.set_materialize_grads(False)
        return q_out, k_out

    @staticmethod
    @once_differentiable
    def backward(ctx, *dys):
        q, k, wq, wk, positions = ctx.saved_tensors
        axes, eps, dtypes = ctx.meta
        need = ctx.needs_input_grad
        # a tensor whose result no gradient arrives at has none either, and adds nothing to its weight's
        xs = [x if dy is not None and (need[i] or need[2 + i]) else None for i, (x, dy) in enumerate(zip((q, k), dys))]
        dx, dw = [None, None], [None, None]
        for i, w in enumerate((wq, wk)):
            if need[2 + i]:
                dw[i] = torch.zeros_like(w) if xs[i] is None else torch.empty_like(w)
        if xs[0] is not None or xs[1] is not None:
            a, _ = _qk_args(xs[0], xs[1], wq, wk, positions, axes, eps)
            (dq, dqs, _), (dk, dks, _) = (_flat(None if x is None else dy) for x, dy in zip(xs, dys))
            dx = [None if x is None else torch.empty_like(x, memory_format=torch.contiguous_format) for x in xs]
            ptr = _lib.ptr
            a.dq_out, a.dk_out, a.dq, a.dk = (ptr(t) for t in (dq, dk, *dx))
            a.dq_row, a.dq_head, a.dk_row, a.dk_head = *dqs[:2], *dks[:2]
            a.dq_weight, a.dk_weight = (ptr(d) if x is not None else None for d, x in zip(dw, xs))
            if a.dq_weight or a.dk_weight:
                n, dim = positions.shape[0], axes.head_dim
                floats = ctypes.c_int64()
                _lib.call("st_qk_norm_rotary_workspace", n, dim, ctypes.byref(floats))
                ws = torch.empty((floats.value,), dtype=torch.float32, device=positions.device)
                a.workspace, a.workspace_floats = ws.data_ptr(), floats.value
            _lib.call_on(positions.device, "st_qk_norm_rotary_backward", ctypes.byref(a))
        dw = [d if d is None or d.dtype is dt else d.to(dt) for d, dt in zip(dw, dtypes)]
        return dx[0] if need[0] else None, dx[1] if need[1] else None, dw[0], dw[1], None, None, None


def sparse_qk_norm_rotary(
    q: Optional[torch.Tensor],
    k: Optional[torch.Tensor],
    positions: Union[SparseTensor, torch.Tensor],
    axes: RotaryAxes,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """``sparse_rotary`` of normalised heads, in one pass: each head of ``q`` and ``k`` is divided by
    ``sqrt(mean(x^2) + eps)`` over its channels, multiplied by ``q_weight`` (``k_weight``; ones where
    ``None``) and turned by the row's position.

    ``q``, ``k``, ``positions`` and ``axes`` as ``sparse_rotary`` takes them, heads of at most 256
    channels, at most 32,767 of them in both; of a tensor (or a gradient) whose row and row of heads reach over more than 2 GiB
    (heads first, say) a contiguous copy is made.
    The weights are (D,) of float32, float16 or bfloat16, shared by the heads of their tensor.  The outputs are contiguous,
    of ``q``'s and ``k``'s dtype, computed in fp32 and rounded once (a mean square must be in fp32's
    range); the gradients of the weights are added in a fixed order.  The backward keeps the inputs
    alone.  There is no forward-mode derivative: a tangent on an input raises.
    """
    pos = _check("sparse_qk_norm_rotary", q, k, positions, axes)
    first = q if q is not None else k
    if axes.head_dim > _lib.QK_MAX_DIM:
        raise ValueError(f"heads must have at most {_lib.QK_MAX_DIM} channels (got {axes.head_dim})")
    for t, w, what in ((q, q_weight, "q_weight"), (k, k_weight, "k_weight")):
        if w is None:
            continue
        if t is None:
            raise ValueError(f"{what} without its tensor")
        if w.shape != (axes.head_dim,) or w.device != first.device:
            raise ValueError(f"{what} must be ({axes.head_dim},) on {first.device} (got {tuple(w.shape)} on {w.device})")
        if w.dtype not in _lib.FEAT_DTYPES:
            _lib.feat_code(w.dtype)
    eps = float(eps)
    if not (eps >= 0 and math.isfinite(eps)):
        raise ValueError(f"eps must not be negative (got {eps})")
    if (0 if q is None else q.shape[1]) + (0 if k is None else k.shape[1]) >= 1 << 15:
        raise ValueError("q and k have at most 32,767 heads together")
    refuse_tangents("sparse_qk_norm_rotary", q, k, q_weight, k_weight)
    if torch.is_grad_enabled() and (
            (q is not None and q.requires_grad) or (k is not None and k.requires_grad)
            or (q_weight is not None and q_weight.requires_grad) or (k_weight is not None and k_weight.requires_grad)):
        return _QkNormRotary.apply(q, k, q_weight, k_weight, pos.detach(), axes, eps)
    return _qk_forward(q, k, q_weight, k_weight, pos, axes, eps)[:2]
