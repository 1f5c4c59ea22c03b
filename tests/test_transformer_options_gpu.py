"""Norms of query and key heads, windows with sinks and dropout together, as SparseTransformerBlock runs them, against
the same block in plain float64 torch with the same elements dropped.

fp32 features: every step is a few fp32 roundings of values near one, so the outputs and gradients
agree to 2e-5 of their norm; bf16 rounds each stored tensor (2^-8), about a dozen on the way: 5e-2.
"""

import copy
import math

import pytest
import torch
from torch import nn

from sparsetriton_amd import SparseTensor, nn as snn
from sparsetriton_amd.nn.functional import AttentionSegments, sparse_attention, sparse_qk_norm_rotary
from test_dropout_gpu import _kept


def _voxels(rows, channels, device, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    coords = torch.cat([torch.cat([torch.full((n, 1), b), torch.randint(0, 60, (n, 3), generator=g)], 1)
                        for b, n in enumerate(rows)]).int()
    feats = torch.randn((sum(rows), channels), generator=g).to(device, dtype)
    return SparseTensor(feats, coords.to(device), spatial_shape=(60, 60, 60), batch_size=len(rows))


def _plain(block, x, coords, lengths, kept):
    """The block in float64; ``kept``: the elements that stay of each branch, (rows, channels) twice."""
    at = block.attn
    d, h, hk, p = at.head_dim, at.heads, at.kv_heads, at.rotary.pairs
    q, k, v = at.qkv(block.norm1(x)).view(len(x), h + 2 * hk, d).split((h, hk, hk), 1)
    axis = [i for i, a in enumerate(at.rotary.axes) for _ in range(a // 2)]
    angle = coords[:, 1:].double()[:, axis] * at.rotary.frequencies.double().to(x.device)
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]

    def head(t, w):
        if w is not None:
            t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + at.qk_eps) * w
        a, b = t[..., :p], t[..., p:2 * p]
        return torch.cat((a * c - b * s, a * s + b * c, t[..., 2 * p:]), -1)

    q, k = head(q, at.q_norm), head(k, at.k_norm)
    out, r0 = [], 0
    for n in lengths:
        rows = slice(r0, r0 + n)
        kk, vv = (t[rows].repeat_interleave(h // hk, 1).transpose(0, 1).contiguous() for t in (k, v))
        z = q[rows].transpose(0, 1).contiguous() @ kk.transpose(1, 2).contiguous() / math.sqrt(d)
        away = torch.arange(n, device=x.device)[None] - torch.arange(n, device=x.device)[:, None]
        see = torch.ones_like(away, dtype=torch.bool) if at.window is None else away.abs() < at.window
        see = see | (torch.arange(n, device=x.device) < at.sinks)
        if at.causal:
            see = see & (away <= 0)
        out.append((torch.softmax(z.masked_fill(~see, float("-inf")), -1) @ vv).transpose(0, 1).reshape(n, -1))
        r0 += n
    scale = 1.0 / (1.0 - block.dropout)
    hh = x + at.proj(torch.cat(out)) * kept[0] * scale
    return hh + block.mlp(block.norm2(hh)) * kept[1] * scale


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.bfloat16, 5e-2)])
@pytest.mark.parametrize("heads,kv_heads,channels,options", [
    (4, 4, 64, dict(window=20, sinks=3, qk_norm=True, dropout=0.2)),
    (8, 2, 128, dict(causal=True, window=33, sinks=1, qk_norm=True, dropout=0.1)),
    (3, 1, 120, dict(causal=True, window=50)), (4, 2, 96, dict(qk_norm=True)), (4, 1, 64, dict(dropout=0.5))])
def test_block_trains_like_the_plain_one(device, own_random, dtype, tol, heads, kv_heads, channels, options):
    torch.manual_seed(1)
    block = snn.SparseTransformerBlock(channels, heads, kv_heads, mlp_ratio=2, **options).to(device, dtype)
    if block.attn.q_norm is not None:
        with torch.no_grad():
            block.attn.q_norm.add_(0.2 * torch.randn_like(block.attn.q_norm))
            block.attn.k_norm.mul_(1.5)
    x = _voxels([130, 1, 77], channels, device, dtype, 2)
    segs = AttentionSegments.from_tensor(x)
    dy = torch.randn(x.F.shape, device=device).to(dtype)
    feats = x.F.clone().requires_grad_(True)
    torch.manual_seed(5)
    kept = [_kept(torch.empty((2,), dtype=torch.int64, device=device).random_(), 0, x.F.numel(), block.dropout)
            .view(x.F.shape).to(device).double() for _ in range(2)]
    plain = copy.deepcopy(block).double()
    ref_x = x.F.double().requires_grad_(True)
    ref = _plain(plain, ref_x, x.C, segs._nq.tolist(), kept)
    ref.backward(dy.double())
    torch.manual_seed(5)
    out = block(x.replace(feats), segs)
    assert isinstance(out, SparseTensor) and out._cache is x._cache
    out.F.backward(dy)

    def near(a, b, what):
        assert (a.double() - b).norm() <= tol * b.norm() + 1e-12, (what, ((a.double() - b).norm() / b.norm()).item())

    near(out.F.detach(), ref.detach(), "output")
    near(feats.grad, ref_x.grad, "features")
    for (name, p), q in zip(block.named_parameters(), plain.parameters()):
        near(p.grad, q.grad, name)
    # nothing is dropped in evaluation
    block.eval(), plain.eval()
    with torch.no_grad():
        near(block(x, segs).F, _plain(plain, x.F.double(), x.C, segs._nq.tolist(), [1.0 - block.dropout] * 2), "evaluation")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_one_by_one_as_in_one_pass(device, dtype):
    """Generation over a cache of keys and values: each new row's heads as in one pass over all of them, to the
    rounding of the output (both have their own of P, 2^-8 of the largest value of a row each, and of O)."""
    n, h, hk, d, window, sinks = 150, 8, 2, 64, 40, 4
    attn = snn.SparseAttention(h * d, h, hk, causal=True, window=window, sinks=sinks, qk_norm=True).to(device, dtype)
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn((n, m, d), generator=g).to(device, dtype) for m in (h, hk, hk))
    pos = torch.randint(0, 60, (n, 3), generator=g).short().to(device)
    with torch.no_grad():
        norm = lambda a, b, p: sparse_qk_norm_rotary(a, b, p, attn.rotary, attn.q_norm, attn.k_norm)  # noqa: E731
        qa, ka = norm(q, k, pos)
        whole = sparse_attention(qa, ka, v, AttentionSegments([n], device=device), causal=True, window=window, sinks=sinks)
        cache_k = torch.empty_like(ka)
        unit = 4 * 2.0 ** -8 if dtype == torch.bfloat16 else 512 * 2.0 ** -24
        for i in range(n):
            qi, ki = norm(q[i:i + 1], k[i:i + 1], pos[i:i + 1])
            assert torch.equal(qi[0], qa[i]) and torch.equal(ki[0], ka[i])
            cache_k[i:i + 1] = ki
            one = sparse_attention(qi, cache_k[:i + 1], v[:i + 1], AttentionSegments([1], [i + 1], device=device), causal=True,
                                   window=window, sinks=sinks)
            top = v[:i + 1].abs().max().item()
            assert (one[0].float() - whole[i].float()).abs().max().item() <= unit * top


@pytest.mark.gpu
def test_block_under_autocast(device, own_random):
    torch.manual_seed(2)
    block = snn.SparseTransformerBlock(64, 4, 2, mlp_ratio=2, window=16, sinks=2, qk_norm=True, dropout=0.1).to(device)
    x = _voxels([90, 40], 64, device, torch.float32, 6)
    torch.manual_seed(9)
    want = block(x)
    torch.manual_seed(9)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = block(x)
    assert got.F.dtype is torch.float32
    assert (got.F - want.F).norm() <= 5e-2 * want.F.norm()
    grads = torch.autograd.grad(got.F.square().sum(), list(block.parameters()))
    assert all(g.dtype is torch.float32 and torch.isfinite(g).all() for g in grads)


@pytest.mark.gpu
def test_captured_step_drops_anew(device, own_random):
    """A captured forward: every replay draws other numbers, and without them gives the eager result."""
    torch.manual_seed(4)
    block = snn.SparseTransformerBlock(64, 4, mlp_ratio=2, causal=True, window=20, sinks=1, qk_norm=True, dropout=0.3).to(device)
    x = _voxels([100], 64, device, torch.float32, 8)
    segs = AttentionSegments([100], device=device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad():
        with torch.cuda.stream(side):
            block(x, segs)
        torch.cuda.current_stream().wait_stream(side)
        graphs = {}
        for train in (True, False):
            block.train(train)
            graphs[train] = (torch.cuda.CUDAGraph(),)
            with torch.cuda.graph(graphs[train][0]):
                graphs[train] += (block(x, segs).F,)
        seen = []
        for _ in range(3):
            x.F.copy_(torch.randn_like(x.F))
            for train in (True, False):
                graphs[train][0].replay()
            torch.cuda.synchronize()
            want = block(x, segs).F
            assert torch.equal(graphs[False][1], want)
            seen.append(graphs[True][1] - want)
        assert all(s.abs().max() > 0 for s in seen)


def test_options_that_make_no_sense_are_refused():
    for options in (dict(window=0), dict(window=-1), dict(sinks=2), dict(window=4, sinks=-1), dict(dropout=1.5), dict(dropout=-0.1)):
        with pytest.raises(ValueError):
            snn.SparseTransformerBlock(64, 4, **options)


def test_a_plain_block_keeps_its_parameters():
    names = [n for n, _ in snn.SparseTransformerBlock(64, 4).named_parameters()]
    assert names == [f"{m}.{p}" for m in ("norm1", "attn.qkv", "attn.proj", "norm2", "mlp.0", "mlp.2") for p in ("weight", "bias")]
    more = snn.SparseTransformerBlock(64, 4, qk_norm=True)
    assert {n for n, _ in more.named_parameters()} - set(names) == {"attn.q_norm", "attn.k_norm"}
    assert isinstance(more.attn.q_norm, nn.Parameter) and more.attn.q_norm.shape == (16,)
