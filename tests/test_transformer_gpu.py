"""SparseAttention and SparseTransformerBlock against the same block in plain float64 torch.

fp32 features: every step is a few fp32 roundings of values near one, so the outputs and gradients
agree to 2e-5 of their norm; bf16 rounds each stored tensor (2^-8), about ten on the way: 5e-2.
"""

import copy
import math

import pytest
import torch
from torch import nn

from sparsetriton_amd import SparseTensor, nn as snn
from sparsetriton_amd.nn.functional import AttentionSegments

pytestmark = pytest.mark.gpu


def _voxels(rows, channels, device, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    coords = torch.cat([torch.cat([torch.full((n, 1), b), torch.randint(0, 60, (n, 3), generator=g)], 1)
                        for b, n in enumerate(rows)]).int()
    feats = torch.randn((sum(rows), channels), generator=g).to(device, dtype)
    return SparseTensor(feats, coords.to(device), spatial_shape=(60, 60, 60), batch_size=len(rows))


def _plain(block, x, coords, lengths, causal):
    """The block in float64: norms, projections, rotation and attention from their formulas."""
    at = block.attn
    d, h, hk = at.head_dim, at.heads, at.kv_heads
    y = block.norm1(x)
    q, k, v = at.qkv(y).view(len(x), h + 2 * hk, d).split((h, hk, hk), 1)
    p = at.rotary.pairs
    axis = [i for i, a in enumerate(at.rotary.axes) for _ in range(a // 2)]
    angle = coords[:, 1:].double()[:, axis] * at.rotary.frequencies.double().to(x.device)
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]

    def turn(t):
        a, b = t[..., :p], t[..., p:2 * p]
        return torch.cat((a * c - b * s, a * s + b * c, t[..., 2 * p:]), -1)

    q, k = turn(q), turn(k)
    out, r0 = [], 0
    for n in lengths:
        rows = slice(r0, r0 + n)
        kk, vv = (t[rows].repeat_interleave(h // hk, 1).transpose(0, 1).contiguous() for t in (k, v))
        z = q[rows].transpose(0, 1).contiguous() @ kk.transpose(1, 2).contiguous() / math.sqrt(d)
        if causal:
            z = z.masked_fill(torch.ones((n, n), dtype=torch.bool, device=x.device).triu(1), float("-inf"))
        out.append((torch.softmax(z, -1) @ vv).transpose(0, 1).reshape(n, -1))
        r0 += n
    hh = x + at.proj(torch.cat(out))
    return hh + block.mlp(block.norm2(hh))


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.bfloat16, 5e-2)])
@pytest.mark.parametrize("heads,kv_heads,channels,causal,patch", [(4, 4, 64, False, None), (8, 2, 128, True, 50),
                                                                 (3, 1, 120, False, 33)])
def test_block_trains_like_the_plain_one(device, dtype, tol, heads, kv_heads, channels, causal, patch):
    torch.manual_seed(1)
    block = snn.SparseTransformerBlock(channels, heads, kv_heads, mlp_ratio=2, causal=causal).to(device, dtype)
    x = _voxels([130, 1, 77], channels, device, dtype, 2)
    segs = AttentionSegments.from_tensor(x, patch)
    lengths = segs._nq.tolist()
    plain = copy.deepcopy(block).double()
    ref_x = x.F.double().requires_grad_(True)
    dy = torch.randn(x.F.shape, device=device).to(dtype)
    ref = _plain(plain, ref_x, x.C, lengths, causal)
    ref.backward(dy.double())
    feats = x.F.clone().requires_grad_(True)
    out = block(x.replace(feats), segs)
    assert isinstance(out, SparseTensor) and out._cache is x._cache
    out.F.backward(dy)

    def near(a, b, what):
        assert (a.double() - b).norm() <= tol * b.norm() + 1e-12, (what, ((a.double() - b).norm() / b.norm()).item())

    near(out.F.detach(), ref.detach(), "output")
    near(feats.grad, ref_x.grad, "features")
    for (name, p), q in zip(block.named_parameters(), plain.parameters()):
        near(p.grad, q.grad, name)


def test_blocks_after_a_convolution_learn(device):
    """A convolution, two blocks over patches and a head, a few steps of training: the loss falls."""
    torch.manual_seed(3)

    class Net(nn.Module):
        def __init__(self):
            super().__init__()
            self.stem = snn.SparseConvBlock(8, 64, 3)
            self.blocks = nn.ModuleList(snn.SparseTransformerBlock(64, 4, mlp_ratio=2) for _ in range(2))
            self.head = snn.SparseLinear(64, 4)

        def forward(self, x):
            x = self.stem(x)
            segs = AttentionSegments.from_tensor(x, patch=128)
            for b in self.blocks:
                x = b(x, segs)
            return self.head(x).F

    net = Net().to(device)
    x = _voxels([400, 300], 8, device, torch.float32, 4)
    want = (x.C[:, 1:].sum(1) % 4).long()
    opt = torch.optim.Adam(net.parameters(), lr=3e-3)
    losses = []
    for _ in range(30):
        loss = nn.functional.cross_entropy(net(x), want)
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.item())
    assert all(map(math.isfinite, losses)) and losses[-1] < 0.8 * losses[0], losses


def test_whole_samples_without_segments_and_state(device):
    torch.manual_seed(5)
    attn = snn.SparseAttention(96, 3, head_dim=40, axes=(12, 12, 8)).to(device)
    x = _voxels([20, 30], 96, device, torch.float32, 6)
    out = attn(x)
    assert torch.equal(out.F, attn(x, AttentionSegments([20, 30], device=device)).F)
    again = copy.deepcopy(attn)
    again.load_state_dict(attn.state_dict())
    assert torch.equal(again(x).F, out.F)
    assert sorted(attn.state_dict()) == ["proj.bias", "proj.weight", "qkv.bias", "qkv.weight"]


def test_refusals():
    with pytest.raises(ValueError, match="divide"):
        snn.SparseAttention(100, 3)
    with pytest.raises(ValueError, match="share"):
        snn.SparseAttention(96, 6, kv_heads=4)


def test_a_frozen_block_refuses_forward_mode(device, own_random):
    block = snn.SparseTransformerBlock(64, 4).to(device).requires_grad_(False)
    x = _voxels([20], 64, device, torch.float32, 8)
    segs = AttentionSegments([20], device=device)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.F, torch.ones_like(x.F))
        with pytest.raises(RuntimeError, match="forward-mode"):
            block(x.replace(dual), segs)


@pytest.mark.parametrize("dtype,tol", [(torch.bfloat16, 5e-2), (torch.float16, 1e-2)])
@pytest.mark.parametrize("features", [torch.float32, None])
def test_block_under_autocast(device, own_random, dtype, tol, features):
    """fp32 parameters, the products in 16 bits: a fp32 stream stays fp32, one in the products' type keeps that.
    (Roundings as in a block of that type: about ten of 2^-8, or of 2^-11.)"""
    torch.manual_seed(9)
    block = snn.SparseTransformerBlock(64, 4, 2, mlp_ratio=2).to(device)
    lengths = [130, 1, 77]
    x = _voxels(lengths, 64, device, features or dtype, 10)
    segs = AttentionSegments.from_tensor(x)
    plain = copy.deepcopy(block).double()
    ref_x = x.F.double().requires_grad_(True)
    dy = torch.randn(x.F.shape, device=device).to(x.F.dtype)
    ref = _plain(plain, ref_x, x.C, lengths, False)
    ref.backward(dy.double())
    feats = x.F.clone().requires_grad_(True)
    with torch.autocast("cuda", dtype):
        out = block(x.replace(feats), segs)
    assert out.F.dtype is x.F.dtype
    out.F.backward(dy)
    near = lambda a, b: (a.double() - b).norm() <= tol * b.norm() + 1e-12  # noqa: E731
    assert near(out.F.detach(), ref.detach()) and near(feats.grad, ref_x.grad)
    for (name, p), q in zip(block.named_parameters(), plain.parameters()):
        assert p.grad.dtype is torch.float32 and near(p.grad, q.grad), name


def test_a_stream_of_another_16_bit_type_is_promoted(device, own_random):
    """float16 features, bfloat16 products: their sum is fp32, as torch's is."""
    torch.manual_seed(9)
    block = snn.SparseTransformerBlock(64, 4).to(device)
    x = _voxels([40], 64, device, torch.float16, 11)
    with torch.autocast("cuda", torch.bfloat16):
        out = block(x)
    assert out.F.dtype is torch.float32
    ref = _plain(copy.deepcopy(block).double(), x.F.double(), x.C, [40], False)
    assert (out.F.double() - ref).norm() <= 5e-2 * ref.norm()


@pytest.mark.parametrize("which", ["norm1", "norm2"])
@pytest.mark.parametrize("make", [lambda c: nn.Sequential(nn.LayerNorm(c), nn.Tanh()), snn.SparseLayerNorm, snn.SparseBatchNorm,
                                  nn.RMSNorm])
def test_another_norm_in_its_place_is_called(device, own_random, which, make):
    """A module over features or over a SparseTensor that a user puts in a norm's place runs, and trains."""
    torch.manual_seed(12)
    block = snn.SparseTransformerBlock(64, 4, mlp_ratio=2)
    setattr(block, which, make(64))
    block = block.to(device)
    x = _voxels([30, 20], 64, device, torch.float32, 13)
    segs = AttentionSegments.from_tensor(x)
    calls = []
    getattr(block, which).register_forward_hook(lambda *_: calls.append(1))
    out = block(x, segs).F
    out.sum().backward()
    assert len(calls) == 1 and all(p.grad is not None for p in getattr(block, which).parameters())
    # by hand, from the block's own parts
    norm = lambda m, t: m(t).F if isinstance(m, (snn.SparseLayerNorm, snn.SparseBatchNorm)) else m(t.F)  # noqa: E731
    plain = lambda m, t: norm(m, t) if m is getattr(block, which) else nn.functional.layer_norm(  # noqa: E731
        t.F, (64,), m.weight, m.bias, m.eps)
    h = x.F + block.attn(x.replace(plain(block.norm1, x)), segs).F
    want = h + block.mlp(plain(block.norm2, x.replace(h)))
    assert (out - want).norm() <= 2e-5 * want.norm()


def test_hooks_of_the_norms_run(device, own_random):
    block = snn.SparseTransformerBlock(64, 4, mlp_ratio=2).to(device)
    x = _voxels([30, 20], 64, device, torch.float32, 14)
    segs = AttentionSegments.from_tensor(x)
    seen = []
    for m in (block.norm1, block.norm2):
        m.register_forward_pre_hook(lambda m, args: seen.append(m))
        m.register_forward_hook(lambda m, args, out: seen.append(m))
    block(x, segs)
    assert [id(m) for m in seen] == [id(m) for m in (block.norm1, block.norm1, block.norm2, block.norm2)]
    # the norms are layer norms with their parameters' names, and take plain features as well
    assert isinstance(block.norm1, nn.LayerNorm) and "norm1.weight" in block.state_dict()
    assert (block.norm1(x.F) - nn.functional.layer_norm(x.F, (64,))).abs().max() < 1e-5


@pytest.mark.parametrize("heads,kv_heads", [(0, None), (4, 0), (-4, None), (4, -2), (4, 8)])
def test_head_counts_that_are_no_counts_are_refused(heads, kv_heads):
    with pytest.raises(ValueError, match="heads"):
        snn.SparseAttention(96, heads, kv_heads)
    with pytest.raises(ValueError, match="heads"):
        snn.SparseTransformerBlock(96, heads, kv_heads)
