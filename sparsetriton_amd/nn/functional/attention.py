"""Attention between the rows of a segment: a sample, a window, a patch of a serialised scene (HIP
kernels ``st_attn_forward`` / ``st_attn_backward``; no counterpart in the reference).

The rows of all segments lie one after another, as features do; ``AttentionSegments`` holds their
lengths and the tile lists that the kernels walk.
"""

import ctypes
import math
from typing import Optional, Sequence, Union

import numpy as np
import torch

from sparsetriton_amd import _lib
from sparsetriton_amd.tensor import SparseTensor
from sparsetriton_amd.utils.utils import once_differentiable, refuse_tangents

__all__ = ["AttentionSegments", "sparse_attention"]

# Mean length of the items against the longest, below which their order goes before the key heads' (us, forward, key
# head by key head / longest first: causal 8,191 rows x 16 x 128 on 4 key heads 431 / 322, four of 4,096 x 8 x 64
# 177 / 109; 64 equal patches of 1,024 x 8 x 64 170 / 177).
_EVEN = 0.9
# Keys (rows) that a part of a split tile is a multiple of: a step of the kernels.
_STEP = 64
# Small tiles (one wave) are taken while there are at most so many for each wide one (four waves), that is
# while most waves of the wide ones would have no rows.  bf16, us wide / small: 2,000 windows of 1-96 rows x
# 4 x 32 (1.31 small tiles a wide one) 27 / 16, 1,000 of 1-200 x 8 x 64 (1.65) 50 / 37, forward and backward of
# 2,000 x 8 x 64 (1.34) 294 / 176; 1,000 of 64 rows (2.0) 19.3 / 19.7, 300 of 40 over 300 keys (2.0) 21 / 26.
_SMALL_TILES = 1.8
# Workgroups that a split of the tiles over their keys (rows) aims at, four for each of 256 compute units; a part takes
# four steps at least.  Whether to split goes by an estimate (us, within a fifth): a step of 64 keys (rows) x 128 rows for a
# workgroup alone on its unit, the share of it that each takes when several share the unit (by the size of an element), the
# join's launch, and the bytes of partial results a microsecond.
_UNITS, _SPLIT_TO, _PART_STEPS = 256, 1024, 4
_SHARED, _JOIN_US, _PART_BYTES_US = {2: 0.75, 4: 0.88}, 7.0, 8.0e6


def _step_us(dim: int, elem: int, keys: bool) -> float:
    return (0.065 * dim if elem == 4 else 0.35 + 0.0086 * dim) * (2.0 if keys else 1.0)


def _lengths(lengths, what: str) -> np.ndarray:
    if isinstance(lengths, torch.Tensor):
        if lengths.dtype.is_floating_point or lengths.dtype == torch.bool:
            raise TypeError(f"{what} must be integers (got {lengths.dtype})")
        lengths = lengths.detach().cpu().numpy()
    out = np.asarray(lengths)
    if out.ndim != 1 or (out.size and out.dtype.kind not in "iu"):
        raise ValueError(f"{what} must be a list of row counts")
    out = out.astype(np.int64)
    if (out < 0).any() or (out >= 2 ** 31).any() or out.sum() >= 2 ** 31 - 4096:  # (each, so that the sum cannot wrap)
        raise ValueError(f"{what} must not be negative, and less than 2^31 - 4096 rows in all")
    return out


def _cut(steps: np.ndarray, most: int):
    """(parts, steps of a part) of tiles of so many steps, in parts of much the same length up to ``most``."""
    parts = np.maximum(1, -(-steps // most))
    chunk = -(-steps // parts)
    return np.maximum(1, -(-steps // np.maximum(chunk, 1))), chunk


def _items(parts: np.ndarray, chunk: np.ndarray, steps: np.ndarray) -> np.ndarray:
    """Steps of every part, the last one of a tile what is left."""
    items = np.repeat(chunk, parts)
    items[np.cumsum(parts) - 1] = steps - (parts - 1) * chunk
    return items


def _longest(items: np.ndarray, kv_heads: int) -> int:
    """Steps of the slot (two a unit) with the most of them, each taking the longest item left when it is done."""
    items = np.repeat(np.sort(items)[::-1], kv_heads) + 1  # (a step's worth for the start and the end of each)
    held = np.zeros(2 * _UNITS, dtype=np.int64)
    for at in range(0, items.size, held.size):
        held.sort()
        held[:items.size - at] += items[at:at + held.size]
    return int(held.max())


def _split(steps: np.ndarray, rows: np.ndarray, kv_heads: int, dim: int, elem: int, keys: bool):
    """(parts of each tile, steps of a part), ``rows`` of each tile in use.

    Whole tiles take the longest one's steps, or what the fullest slot has to do; parts an even share of all steps (and
    a seventh for what is not even), and their joins.  bf16, 256 tiles of 16 steps whole / in two / four parts, forward and backward: 64
    channels 20 + 55 / 34 + 74 / 36 + 87 us, 128 channels 28 + 123 / 41 + 137 / 52 + 174; 64 tiles of 128 channels 27 + 119 /
    22 + 86 / 25 + 68, of 64 channels in fp32 78 + 270 / 46 + 151 / 32 + 94; 128 tiles of up to 128 steps beside 1,200 of
    one, 64 channels: 119 + 335 whole, 62 + 180 in parts.
    """
    whole = np.ones_like(steps), steps
    total, us = int(steps.sum()) * kv_heads, _step_us(dim, elem, keys)
    shared = us * _SHARED[elem] * -(-int(rows.max(initial=1)) // 32) * 32 / _lib.ATTN_TILE  # (waves without rows wait)
    longest = int(steps.max(initial=0)) + 1
    if longest * us <= total / _UNITS * shared:
        return whole
    most = max(_PART_STEPS, -(-total // _SPLIT_TO))
    parts = about = _cut(steps, most)
    # Parts of a whole number of steps come to more than aimed at, at times, and the few of a last round keep the rest
    # waiting (8,191 causal rows x 16 x 128 on 4 key heads, dK and dV: 1,152 parts 890 us, 984 800; but 24 samples of up to
    # 1,500 rows x 6 x 48 fp32: 1,056 of up to 5 steps 376, 882 of up to 6 399).
    if steps.size * kv_heads <= _SPLIT_TO:
        while parts[0].sum() * kv_heads > _SPLIT_TO:
            most += max(1, most // 16)
            parts = _cut(steps, most)
        if parts is not about:
            parts = min((about, parts), key=lambda p: _longest(_items(*p, steps), kv_heads))
    n = parts[0]
    cut = n > 1
    if not cut.any():
        return whole
    parts_us = max((int(parts[1].max()) + 1) * us, 1.15 * (total + int(n.sum()) * kv_heads) / _UNITS * shared)
    parts_us += _JOIN_US + float((rows * n)[cut].sum()) * kv_heads * (dim + 2) * 8 * (2 if keys else 1) / _PART_BYTES_US
    whole_us = longest * us
    if steps.size * kv_heads > _UNITS:
        # (two to a unit at its worst; once more wait than run, a long one has had shorter ones beside it)
        whole_us = max(whole_us, _longest(steps, kv_heads) * (2 if steps.size * kv_heads <= 2 * _UNITS else 1.35) * shared)
    return whole if whole_us <= parts_us else parts


class _Tiles:
    """Work items and joins of one pass, on the device: rows (4, 8) int32 as st_attn_args lays them out."""

    def __init__(self, tile, q0, nq, k0, nk, row0, rows, lo, hi, kv_heads, dim, elem, keys, device):
        self.tile, step = tile, _STEP
        steps = -(-(hi - lo) // step)
        n = steps.size
        parts, chunk = _split(steps, rows, kv_heads, dim, elem, keys)
        of = np.repeat(np.arange(n), parts)
        nth = np.arange(of.size) - np.repeat(np.cumsum(parts) - parts, parts)
        first = lo[of] + nth * chunk[of] * step
        end = np.minimum(hi[of], first + chunk[of] * step)
        split = parts > 1
        slot0 = np.cumsum(np.where(split, parts, 0)) - np.where(split, parts, 0)
        part = np.where(split[of], slot0[of] + nth, -1)
        items = np.stack([q0[of], nq[of], k0[of], nk[of], row0[of], first, end, part], 1)
        # Longest first: the last workgroups to start are short ones.  Tiles of much the same length go key head by
        # key head (neighbours read the same keys); else the long ones of every key head come before the short ones.
        self.item_major = int(n > 0 and (end - first).mean() < _EVEN * (end - first).max())
        items = items[np.argsort(first - end, kind="stable")]
        at = np.flatnonzero(split)
        joins = np.stack([q0[at], nq[at], k0[at], nk[at], row0[at], slot0[at], parts[at], np.zeros_like(at)], 1)
        self.n_items, self.n_joins, self.slots = items.shape[0], joins.shape[0], int(parts[split].sum())
        self.words = torch.from_numpy(np.concatenate([items, joins]).astype(np.int32)).to(device)
        self.items = self.words.data_ptr()
        self.joins = self.items + self.n_items * _lib.ATTN_WORDS * 4 if self.n_joins else None
        self._stream = None

    def use(self) -> None:
        """The words' memory is not handed out again before this stream is through with them."""
        if self.n_items and self.words.is_cuda:
            s = _lib.stream_of(self.words.device)
            if s != self._stream:
                self.words.record_stream(torch.cuda.current_stream(self.words.device))
                self._stream = s


class AttentionSegments:
    """Lengths of the row segments that attend among themselves, and the kernels' tile lists.

    ``q_lengths``: rows of each segment, in the order in which the rows lie; ``k_lengths`` the key
    rows where they are not the same (cross attention).  Both are sequences or integer tensors (a
    device tensor is read back).  Either may be zero: a row without keys has a zero output.  Made
    once for a set of rows and shared by the layers over them; the tile lists for a number of heads,
    an order and a type are built at the first call with them, which costs 0.1 to 0.2 ms of host time
    each (forward, and the keys' in the backward) and a blocking copy; a call whose lists are not there
    yet cannot be captured in a graph.  A copy or a pickle builds its own.
    """

    def __init__(self, q_lengths: Union[Sequence[int], torch.Tensor],
                 k_lengths: Optional[Union[Sequence[int], torch.Tensor]] = None,
                 device: Union[str, torch.device] = "cuda") -> None:
        self._nq = _lengths(q_lengths, "q_lengths")
        self._nk = self._nq if k_lengths is None else _lengths(k_lengths, "k_lengths")
        if self._nq.size != self._nk.size:
            raise ValueError(f"{self._nq.size} segments of queries, {self._nk.size} of keys")
        self._q0, self._k0 = (np.cumsum(n) - n for n in (self._nq, self._nk))
        self.count, self.q_rows, self.k_rows = self._nq.size, int(self._nq.sum()), int(self._nk.sum())
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None and torch.cuda.is_available():
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._plans = {}

    def __getstate__(self):
        # (a list holds the address of its own device memory: a copy, or another process, builds its own)
        return {**self.__dict__, "_plans": {}}

    @classmethod
    def from_tensor(cls, tensor: SparseTensor, patch: Optional[int] = None) -> "AttentionSegments":
        """The samples of ``tensor`` (whose rows must lie sample by sample, in ascending order), or
        with ``patch`` each sample's rows in their order cut in patches of ``patch`` rows, the last
        one of a sample shorter."""
        if patch is not None and int(patch) <= 0:
            raise ValueError(f"patch must be positive (got {patch})")
        b = tensor.C[:, 0].long()
        counts = torch.bincount(b, minlength=max(int(tensor.batch_size or 0), 1))
        if b.numel() and bool((b[1:] < b[:-1]).any()):
            raise ValueError("the rows must lie sample by sample, in ascending batch order")
        counts = counts.cpu().numpy()
        if patch is not None:
            full, rest = counts // int(patch), counts % int(patch)
            counts = np.concatenate([np.asarray([int(patch)] * f + [r] * int(r > 0), dtype=np.int64)
                                     for f, r in zip(full, rest)])
        return cls(counts, device=tensor.F.device)

    @staticmethod
    def _tiles(rows, row_bytes):
        """(tile size, segment and first row of each tile) over segments of so many rows (keys)."""
        small, wide = (int((-(-rows // t)).sum()) for t in (_lib.ATTN_SMALL_TILE, _lib.ATTN_TILE))
        narrow = row_bytes <= _lib.ATTN_SMALL_TILE_BYTES and small <= _SMALL_TILES * wide
        tile = _lib.ATTN_SMALL_TILE if narrow else _lib.ATTN_TILE
        n = -(-rows // tile)
        seg = np.repeat(np.arange(n.size), n)
        return tile, seg, (np.arange(seg.size) - np.repeat(np.cumsum(n) - n, n)) * tile

    def _plan(self, which: str, group: int, kv_heads: int, causal: bool, row_bytes: int, elem: int = 2) -> _Tiles:
        dim = -(-row_bytes // elem // 32) * 32  # (as the kernels are built: one list for all sizes of a kernel)
        key = (which, group, kv_heads, causal, dim, elem)
        plan = self._plans.get(key)
        if plan is None:
            nq, nk = self._nq, self._nk
            if int(nq.max(initial=0)) * group >= 2 ** 31 - _lib.ATTN_TILE:
                raise ValueError(f"a segment has at most {(2 ** 31 - _lib.ATTN_TILE) // group} query rows at {group} heads a key head")
            if which == "q":  # tiles of packed rows over keys lo .. hi
                tile, seg, row0 = self._tiles(nq * group, row_bytes)
                rows = np.minimum(nq[seg] * group - row0, tile)
                lo, hi = np.zeros_like(row0), nk[seg]
                if causal:
                    last = np.minimum(row0 + tile, nq[seg] * group) - 1
                    hi = np.clip(last // group + nk[seg] - nq[seg] + 1, 0, nk[seg])
            else:  # tiles of keys over packed rows lo .. hi
                tile, seg, row0 = self._tiles(nk, row_bytes)
                rows = np.minimum(nk[seg] - row0, tile)
                lo, hi = np.zeros_like(row0), nq[seg] * group
                if causal:
                    lo = np.minimum(np.maximum(0, row0 - (nk[seg] - nq[seg])) * group, hi)
            plan = _Tiles(tile, self._q0[seg], nq[seg], self._k0[seg], nk[seg], row0, rows, lo, hi,
                          kv_heads, dim, elem, which == "k", self.device)
            self._plans[key] = plan
        plan.use()
        return plan


def _parts(kv_heads, dim, q_slots, k_slots, device):
    if not q_slots and not k_slots:
        return None
    floats = ctypes.c_int64()
    _lib.call("st_attn_workspace", kv_heads, dim, q_slots, k_slots, ctypes.byref(floats))
    return torch.empty((floats.value,), dtype=torch.float32, device=device)


def _rows(t: torch.Tensor, group: int) -> torch.Tensor:
    """t, or a contiguous copy where the kernels' 16-byte accesses or 32-bit tile offsets do not reach its rows."""
    e = t.element_size()
    row, head, channel = t.stride()
    if (channel == 1 and not (row * e | head * e | t.data_ptr()) & 15 and row < 2 ** 29 and head < 2 ** 29
            and (row * (_lib.ATTN_TILE + 1) + head * (group + 1) + t.shape[2]) * e < 2 ** 31 - 64):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _args(q, k, v, key_mask, o, rest, lse, causal, scale) -> _lib.AttnArgs:
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    ptr = _lib.ptr
    return _lib.AttnArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), ptr(rest), ptr(lse), None, None, None, None,
                         None, qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], 0, 0, ptr(key_mask), None, None, None, None,
                         0, 0, 0, 0, None, q.shape[1], k.shape[1], q.shape[2], _lib.FEAT_DTYPES[q.dtype], causal, _lib.ATTN_TILE,
                         _lib.ATTN_TILE, 0, 0, scale)


def _forward(q, k, v, segments, key_mask, causal, scale, stats):
    n, heads, dim = q.shape
    kv_heads = k.shape[1]
    group = heads // kv_heads
    q, k, v = _rows(q, group), _rows(k, group), _rows(v, group)
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty((n, heads), dtype=torch.float32, device=q.device) if stats else None
    plan = segments._plan("q", group, kv_heads, causal, dim * q.element_size(), q.element_size())
    rest = torch.empty_like(o) if stats and o.element_size() == 2 else None  # what its rounding leaves, for the gradient
    a = _args(q, k, v, key_mask, o, rest, lse, causal, scale)
    a.q_items, a.q_joins, a.n_q_items, a.n_q_joins = plan.items, plan.joins, plan.n_items, plan.n_joins
    a.q_tile, a.q_item_major = plan.tile, plan.item_major
    parts = _parts(kv_heads, dim, plan.slots, 0, q.device)
    if parts is not None:
        a.parts = parts.data_ptr()
    _lib.call("st_attn_forward", ctypes.byref(a), _lib.stream_of(q.device))
    return o, rest, lse, q, k, v


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, segments, key_mask, causal, scale):
        o, rest, lse, q, k, v = _forward(q, k, v, segments, key_mask, causal, scale, True)
        ctx.save_for_backward(q, k, v, o, rest, lse, key_mask)
        ctx.meta = (segments, causal, scale)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, o, rest, lse, key_mask = ctx.saved_tensors
        segments, causal, scale = ctx.meta
        heads, dim = q.shape[1:]
        kv_heads = k.shape[1]
        group = heads // kv_heads
        dout = _rows(dout, group)
        new = lambda t: torch.empty_like(t, memory_format=torch.contiguous_format)  # noqa: E731
        dq, delta = new(q), torch.empty_like(lse)
        plan = segments._plan("q", group, kv_heads, causal, dim * q.element_size(), q.element_size())
        a = _args(q, k, v, key_mask, o, rest, lse, causal, scale)
        a.dout, a.dq, a.delta = dout.data_ptr(), dq.data_ptr(), delta.data_ptr()
        a.dout_row, a.dout_head, _ = dout.stride()
        a.q_items, a.q_joins, a.n_q_items, a.n_q_joins = plan.items, plan.joins, plan.n_items, plan.n_joins
        a.q_tile, a.q_item_major = plan.tile, plan.item_major
        dk = dv = None
        slots = 0
        if ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
            dk, dv = new(k), new(v)
            keys = segments._plan("k", group, kv_heads, causal, dim * q.element_size(), q.element_size())
            a.dk, a.dv = dk.data_ptr(), dv.data_ptr()
            a.k_items, a.k_joins, a.n_k_items, a.n_k_joins = keys.items, keys.joins, keys.n_items, keys.n_joins
            a.k_tile, a.k_item_major = keys.tile, keys.item_major
            slots = keys.slots
        parts = _parts(kv_heads, dim, plan.slots, slots, q.device)
        if parts is not None:
            a.parts = parts.data_ptr()
        _lib.call("st_attn_backward", ctypes.byref(a), _lib.stream_of(q.device))
        need = ctx.needs_input_grad
        return dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, None, None, None, None


def sparse_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    segments: AttentionSegments,
    scale: Optional[float] = None,
    causal: bool = False,
    key_mask: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``softmax(scale * q k^T) v`` in each segment, (rows, heads, D) contiguous in ``q``'s dtype.

    ``q`` (``segments.q_rows``, heads, D); ``k``, ``v`` (``segments.k_rows``, kv_heads, D) of the
    same dtype (float32, float16, bfloat16); ``heads`` a multiple of ``kv_heads``, whose key head
    ``h // (heads / kv_heads)`` query head ``h`` reads; D a multiple of 8, at most 128.  Rows and
    heads may lie at any stride (slices of one projection, say); where channels are apart or rows not
    at 16-byte addresses a copy is made.  ``scale`` is positive, ``D ** -0.5`` by default.

    ``causal``: query ``i`` of ``nq`` sees keys up to ``i + nk - nq`` of its segment.  ``key_mask``
    (``segments.k_rows``) bool: False leaves a key out, whatever its rows hold.  A row that sees no
    key gets zeros, and its gradients are zero.  Scores, softmax and sums are fp32 (fp32 inputs: the
    products too); results do not depend on timing.  16-bit inputs round the probabilities, and in the
    gradient dS, to their type for the products with V, dO, K and Q: errors 1.2 to 1.4 times those of fp32
    arithmetic rounded once.  float16 holds both at powers of two, so that neither overflows where the
    result does not nor loses digits to the type's smallest numbers.  A 16-bit forward that records a
    gradient keeps what the output's rounding left beside it (as large as the output), for the gradients
    of rows with few keys.
    There is no forward-mode derivative: a tangent on ``q``, ``k`` or ``v`` raises.
    """
    for t, what in ((q, "q"), (k, "k"), (v, "v")):
        if not t.is_cuda:
            _lib.require_device(t, f"attention {what}")
        if t.dtype not in _lib.FEAT_DTYPES:
            _lib.feat_code(t.dtype)
        if t.dim() != 3 or t.dtype is not q.dtype or t.device != q.device:
            raise ValueError(f"{what} must be (rows, heads, D) of q's dtype and device (got {tuple(t.shape)} {t.dtype} "
                             f"on {t.device})")
    heads, dim = q.shape[1:]
    if q.shape[0] != segments.q_rows or k.shape[0] != segments.k_rows:
        raise ValueError(f"the segments have {segments.q_rows} query and {segments.k_rows} key rows, q and k have "
                         f"{q.shape[0]} and {k.shape[0]}")
    if k.shape != v.shape or k.shape[2] != dim or k.shape[1] == 0 or heads == 0 or heads % k.shape[1]:
        raise ValueError(f"heads do not fit: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if dim == 0 or dim % 8 or dim > _lib.ATTN_MAX_DIM:
        raise ValueError(f"the head size must be a multiple of 8 up to {_lib.ATTN_MAX_DIM} (got {dim})")
    if segments.device != q.device:
        raise ValueError(f"the segments are on {segments.device}, q on {q.device}")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite (got {scale})")
    if key_mask is not None:
        if key_mask.dtype != torch.bool:
            raise TypeError(f"key_mask must be bool (got {key_mask.dtype})")
        if key_mask.shape != k.shape[:1] or key_mask.device != q.device:
            raise ValueError(f"key_mask must be ({k.shape[0]},) on {q.device} (got {tuple(key_mask.shape)} on "
                             f"{key_mask.device})")
        key_mask = key_mask.contiguous()
    causal = bool(causal)
    refuse_tangents("sparse_attention", q, k, v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _Attention.apply(q, k, v, segments, key_mask, causal, scale)
    return _forward(q, k, v, segments, key_mask, causal, scale, False)[0]
