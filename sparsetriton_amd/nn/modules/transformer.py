"""Transformer layers over voxel features (no counterpart in the reference).

``SparseAttention`` projects the features to queries, keys and values, turns queries and keys by
the voxels' x, y, z (``sparse_rotary``) and attends within the row segments
(``sparse_attention``).  ``SparseTransformerBlock`` is the pre-norm block around it::

    h = x + attention(norm1(x));   out = h + mlp(norm2(h))

whose first add runs inside the second norm (``sparse_layer_norm`` with a residual).  ``norm1`` and
``norm2`` are modules like any other: their hooks run, and another norm in their place is called, on
the ``SparseTensor`` if it is one of this package's, on the features otherwise.  Build the
segments once for a coordinate set and hand them to every block::

    segments = AttentionSegments.from_tensor(x, patch=1024)
    for block in blocks:
        x = block(x, segments)

Under ``torch.autocast`` the projections' products (and so rotary and attention) are 16-bit; the
norms take the stream in its own type, and the sums are of the wider of the two, as torch's are.
"""

from typing import Optional, Sequence

import torch
from torch import nn

from sparsetriton_amd.nn.functional.attention import AttentionSegments, sparse_attention
from sparsetriton_amd.nn.functional.norm import sparse_layer_norm
from sparsetriton_amd.nn.functional.rotary import RotaryAxes, sparse_rotary
from sparsetriton_amd.nn.modules.norm import SparseBatchNorm, SparseLayerNorm
from sparsetriton_amd.tensor import SparseTensor

__all__ = ["SparseAttention", "SparseTransformerBlock"]


def _three_axes(dim: int):
    """An even number of a head's channels for each of x, y and z, all of them or all but two."""
    pair = dim // 2
    return tuple(2 * (pair // 3 + (1 if i < pair % 3 else 0)) for i in range(3))


def _one_type(a: SparseTensor, b: SparseTensor):
    """a and b in the type that torch's sum of them has: under autocast a branch's products are 16-bit where the stream is not."""
    dtype = torch.promote_types(a.F.dtype, b.F.dtype)
    return tuple(t if t.F.dtype is dtype else t.replace(t.F.to(dtype)) for t in (a, b))


class SparseAttention(nn.Module):
    """Multi-head attention between the rows of each segment, with rotary voxel positions.

    ``kv_heads`` (default ``heads``) key heads are shared by ``heads / kv_heads`` query heads each;
    ``axes`` channels of a head turn with x, y and z (default: the whole head, in three parts).
    ``causal``: the rows' order is the order of generation.
    """

    def __init__(self, channels: int, heads: int, kv_heads: Optional[int] = None, head_dim: Optional[int] = None,
                 axes: Optional[Sequence[int]] = None, base: float = 10000.0, causal: bool = False, bias: bool = True):
        super().__init__()
        self.heads, self.kv_heads = heads, heads if kv_heads is None else kv_heads
        if self.heads < 1 or self.kv_heads < 1:
            raise ValueError(f"heads and key heads must be positive (got {heads} and {kv_heads})")
        if head_dim is None and channels % heads:
            raise ValueError(f"{channels} channels do not divide into {heads} heads")
        self.head_dim = channels // heads if head_dim is None else head_dim
        if self.heads % self.kv_heads:
            raise ValueError(f"{heads} heads do not share {kv_heads} key heads evenly")
        self.causal = causal
        self.rotary = RotaryAxes(self.head_dim, _three_axes(self.head_dim) if axes is None else axes, base=base)
        self.qkv = nn.Linear(channels, (self.heads + 2 * self.kv_heads) * self.head_dim, bias=bias)
        self.proj = nn.Linear(self.heads * self.head_dim, channels, bias=bias)

    def forward(self, x: SparseTensor, segments: Optional[AttentionSegments] = None,
                key_mask: Optional[torch.Tensor] = None) -> SparseTensor:
        if segments is None:  # each sample a segment (reads the rows per sample back)
            segments = AttentionSegments.from_tensor(x)
        qkv = self.qkv(x.F).view(x.F.shape[0], self.heads + 2 * self.kv_heads, self.head_dim)
        q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), dim=1)
        q, k = sparse_rotary(q, k, x, self.rotary)
        out = sparse_attention(q, k, v, segments, causal=self.causal, key_mask=key_mask)
        return x.replace(self.proj(out.flatten(1)))


class _StreamNorm(nn.LayerNorm):
    """``sparse_layer_norm`` with a layer norm's parameters; plain features go through torch's."""

    def forward(self, input, residual: Optional[SparseTensor] = None):
        if not isinstance(input, SparseTensor):
            return super().forward(input)
        return sparse_layer_norm(input, self.weight, self.bias, eps=self.eps, residual=residual)


def _normed(norm: nn.Module, x: SparseTensor) -> SparseTensor:
    if isinstance(norm, (_StreamNorm, SparseLayerNorm, SparseBatchNorm)):
        return norm(x)
    return x.replace(norm(x.F))


class SparseTransformerBlock(nn.Module):
    """Pre-norm block: attention within the segments, then a two-layer GELU network."""

    def __init__(self, channels: int, heads: int, kv_heads: Optional[int] = None, mlp_ratio: float = 4.0, eps: float = 1e-5,
                 axes: Optional[Sequence[int]] = None, causal: bool = False):
        super().__init__()
        self.norm1 = _StreamNorm(channels, eps=eps)
        self.attn = SparseAttention(channels, heads, kv_heads, axes=axes, causal=causal)
        self.norm2 = _StreamNorm(channels, eps=eps)
        hidden = int(channels * mlp_ratio)
        self.mlp = nn.Sequential(nn.Linear(channels, hidden), nn.GELU(), nn.Linear(hidden, channels))

    def forward(self, x: SparseTensor, segments: Optional[AttentionSegments] = None,
                key_mask: Optional[torch.Tensor] = None) -> SparseTensor:
        a, x = _one_type(self.attn(_normed(self.norm1, x), segments, key_mask), x)
        if isinstance(self.norm2, _StreamNorm):
            z, h = self.norm2(a, x)
        else:
            h = x.replace(x.F + a.F)
            z = _normed(self.norm2, h)
        return h.replace(h.F + self.mlp(z.F))
