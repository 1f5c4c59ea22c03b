"""sparse_attention (st_attn_forward / st_attn_backward) against the formulas in float64.

Bounds, per element, from the roundings on the way (u: half a unit of the type, 2^-8, 2^-11 or 0 for
fp32 products; w = 512 * 2^-24 for what fp32 does to a score of |q||k| c ~ 11 summed over 128
channels, its exponential and the row's sum):
  P    (u + w) P                                  (rounded for the second product)
  O    (u + w) sum P |v|  + u |O|                 (float16 also loses 2^-25 of P below 2^-14)
  dP - delta   w sum |dO||v|  + sum |dO| (error of O)
  dS   (2 u + w) |dS| + P (error of dP - delta)
  dQ, dK, dV   the error of dS or P through the product, plus u of the result.
"""

import concurrent.futures
import copy
import math
import pickle
import threading

import numpy as np
import pytest
import torch

from sparsetriton_amd import SparseTensor, _lib
from sparsetriton_amd.nn.functional import AttentionSegments, sparse_attention

UNIT = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
W = 512 * 2.0 ** -24


def _reference(q, k, v, do, ql, kl, scale, causal, mask):
    """{name: (value, bound)} in float64; gradients of the key heads summed over their query heads."""
    u, tiny = UNIT[q.dtype], 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    last = max(u, 2.0 ** -24)
    group = q.shape[1] // k.shape[1]
    q, k, v, do = (t.detach().double() for t in (q, k, v, do))
    if mask is not None:
        k, v = (t.masked_fill(~mask[:, None, None], 0.0) for t in (k, v))
    val = {n: torch.zeros_like(t) for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    err = {n: torch.zeros_like(t) for n, t in val.items()}
    q0 = k0 = 0
    for nq, nk in zip(ql, kl):
        Q, K = slice(q0, q0 + nq), slice(k0, k0 + nk)
        see = torch.ones((nq, nk), dtype=torch.bool, device=q.device)
        if causal:
            see = see.tril(nk - nq)
        if mask is not None:
            see = see & mask[K]
        for h in range(q.shape[1] if nq and nk else 0):
            a, b, c, g = q[Q, h], k[K, h // group], v[K, h // group], do[Q, h]
            s = (a @ b.T * scale).masked_fill(~see, float("-inf"))
            top = s.amax(1, keepdim=True).clamp_min(-1e300)
            p = torch.exp(s - top)
            total = p.sum(1, keepdim=True)
            p = p / total.masked_fill(total == 0, 1.0)
            o = p @ c
            ep = (u + W) * p + tiny * see
            eo = ep @ c.abs() + last * o.abs()
            delta = (g * o).sum(1, keepdim=True)
            ds = p * (g @ c.T - delta)
            edp = W * (g.abs() @ c.abs().T) + (g.abs() * eo).sum(1, keepdim=True)
            eds = (2 * u + W) * ds.abs() + p * edp + tiny * see
            val["o"][Q, h], err["o"][Q, h] = o, eo
            val["dq"][Q, h] = ds @ b * scale
            err["dq"][Q, h] = eds @ b.abs() * scale
            val["dk"][K, h // group] += ds.T @ a * scale
            err["dk"][K, h // group] += eds.T @ a.abs() * scale
            val["dv"][K, h // group] += p.T @ g
            err["dv"][K, h // group] += ep.T @ g.abs()
        q0, k0 = q0 + nq, k0 + nk
    return {n: (t, err[n] + last * t.abs() + 1e-12) for n, t in val.items()}


def _make(ql, kl, heads, kv_heads, dim, dtype, device, seed, masked=0.0):
    g = torch.Generator().manual_seed(seed)
    rand = lambda n, h: torch.randn((n, h, dim), generator=g).to(device, dtype)  # noqa: E731
    q, do = rand(sum(ql), heads), rand(sum(ql), heads)
    k, v = rand(sum(kl), kv_heads), rand(sum(kl), kv_heads)
    mask = (torch.rand((sum(kl),), generator=g) >= masked).to(device) if masked else None
    return q, k, v, do, mask


def _check(q, k, v, do, ql, kl, causal=False, mask=None, scale=None):
    segs = AttentionSegments(ql, kl, device=q.device)
    with torch.no_grad():
        plain = sparse_attention(q, k, v, segs, scale=scale, causal=causal, key_mask=mask)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = sparse_attention(q, k, v, segs, scale=scale, causal=causal, key_mask=mask)
    assert torch.equal(o, plain) and o.is_contiguous()
    got = dict(zip(("o", "dq", "dk", "dv"), (o.detach(),) + torch.autograd.grad(o, leaves, do)))
    ref = _reference(q, k, v, do, ql, kl, q.shape[2] ** -0.5 if scale is None else scale, causal, mask)
    for n, (want, bound) in ref.items():
        assert got[n].shape == want.shape and got[n].dtype == q.dtype
        over = (got[n].double() - want).abs() - bound
        assert not torch.isnan(got[n]).any(), n
        assert over.numel() == 0 or over.max().item() <= 0, (n, over.max().item(), want.abs().max().item())
    return got


LENGTHS = [
    ([1], [1]), ([1, 1, 1], [1, 1, 1]), ([5], [64]), ([33, 1, 127, 2], [33, 1, 127, 2]), ([128, 129], [65, 64]),
    ([0, 7, 0, 3], [4, 0, 0, 9]), ([300], [300]), ([1, 3], [700, 1]), ([200, 10], [3, 150]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("ql,kl", LENGTHS)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [(torch.bfloat16, 4, 4, 64), (torch.float16, 6, 2, 40),
                                                     (torch.float32, 3, 1, 32), (torch.bfloat16, 8, 1, 128)])
def test_lengths(device, ql, kl, causal, dtype, heads, kv_heads, dim):
    q, k, v, do, _ = _make(ql, kl, heads, kv_heads, dim, dtype, device, sum(ql) + dim)
    _check(q, k, v, do, ql, kl, causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [8, 16, 24, 32, 48, 64, 72, 80, 96, 104, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
def test_head_sizes(device, dim, dtype, causal):
    ql = [70, 3, 190]
    q, k, v, do, mask = _make(ql, ql, 4, 2, dim, dtype, device, dim, masked=0.3)
    _check(q, k, v, do, ql, ql, causal, mask)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 5), (7, 1), (12, 4), (6, 3), (40, 2)])
@pytest.mark.parametrize("causal", [False, True])
def test_shared_key_heads(device, heads, kv_heads, causal):
    ql, kl = [45, 1, 130], [61, 77, 130]
    q, k, v, do, mask = _make(ql, kl, heads, kv_heads, 32, torch.bfloat16, device, heads, masked=0.2)
    _check(q, k, v, do, ql, kl, causal, mask)


@pytest.mark.gpu
@pytest.mark.parametrize("ql,kl,heads,kv_heads,dim,causal", [
    ([1], [5000], 4, 1, 64, False), ([1, 1, 2], [1, 4097, 300], 8, 2, 128, True), ([3], [9001], 1, 1, 32, False),
    ([2500], [40], 2, 1, 32, False), ([1000], [1000], 1, 1, 64, True), ([1500, 20], [1, 2000], 2, 2, 48, False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_work_split_over_the_long_side(device, ql, kl, heads, kv_heads, dim, causal, dtype):
    q, k, v, do, mask = _make(ql, kl, heads, kv_heads, dim, dtype, device, 3 * dim, masked=0.1)
    segs = AttentionSegments(ql, kl, device=device)
    plans = [segs._plan(w, heads // kv_heads, kv_heads, causal, dim * q.element_size()) for w in "qk"]
    assert any(p.n_joins for p in plans)
    _check(q, k, v, do, ql, kl, causal, mask)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float32, 32)])
@pytest.mark.parametrize("times", [3, 8])
def test_many_tiles(device, causal, dtype, dim, times):
    """Three times: partly split.  Eight times: enough workgroups (over 512 in both passes) that nothing is."""
    ql = [700, 1, 333, 900, 64, 128, 2] * times
    q, k, v, do, mask = _make(ql, ql, 8, 4, dim, dtype, device, 17, masked=0.05)
    segs = AttentionSegments(ql, device=device)
    assert times == 3 or not any(segs._plan(w, 2, 4, causal, dim * q.element_size()).n_joins for w in "qk")
    _check(q, k, v, do, ql, ql, causal, mask)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1.0, 1e-3, 30.0])
def test_scales(device, scale):
    ql = [150, 20]
    q, k, v, do, _ = _make(ql, ql, 2, 2, 32, torch.float32, device, 4)
    if scale > 1:  # sharp rows: the scores' rounding grows with them
        q, k = q * 0.1, k * 0.1
    _check(q, k, v, do, ql, ql, False, None, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [-60.0, 60.0])
def test_scores_far_from_zero(device, shift):
    """One direction that all queries and keys share moves every score by the same amount, growing along the keys."""
    ql = [40, 500]
    q, k, v, do, _ = _make(ql, ql, 2, 1, 32, torch.float32, device, 5)
    q[:, :, 0] = 1.0
    k[:, :, 0] = shift * torch.linspace(0, 1, sum(ql), device=device)[:, None]
    _check(q, k, v, do, ql, ql, False, None, 1.0 / 8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("causal", [False, True])
def test_rows_without_keys(device, dtype, causal):
    """A segment whose keys are all masked, one without keys, and (causal) queries before the first key."""
    ql, kl = [70, 5, 90, 100], [70, 0, 30, 200]
    q, k, v, do, _ = _make(ql, kl, 4, 2, 64, dtype, device, 6)
    mask = torch.ones(sum(kl), dtype=torch.bool, device=device)
    mask[:70] = False
    mask[100:140] = False
    got = _check(q, k, v, do, ql, kl, causal, mask)
    assert not got["o"][:75].any() and not got["dq"][:75].any() and not got["dk"][:70].any() and not got["dv"][:70].any()
    if causal:
        assert not got["o"][75:135].any() and not got["dq"][75:135].any()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_what_masked_keys_hold_does_not_matter(device, bad, dtype):
    ql = [90, 40, 130]
    q, k, v, do, mask = _make(ql, ql, 4, 2, 64, dtype, device, 7, masked=0.4)
    clean = _check(q.clone(), k.clone(), v.clone(), do, ql, ql, False, mask)
    k[~mask], v[~mask] = bad, bad
    got = _check(q, k, v, do, ql, ql, False, mask)
    assert all(torch.equal(got[n], clean[n]) for n in got)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 32)])
@pytest.mark.parametrize("at", [37, 100, 128])
def test_later_rows_do_not_reach_earlier_ones(device, bad, dtype, dim, at):
    """Causal: a row that is not finite changes nothing for the rows before it, in its own tile too."""
    ql = [200]
    q, k, v, do, _ = _make(ql, ql, 4, 2, dim, dtype, device, 8)
    clean = _check(q.clone(), k.clone(), v.clone(), do, ql, ql, True)
    # values and keys: rows before `at` keep output and query gradient
    for t in (v, k):
        t2 = t.clone()
        t2[at, :, 3] = bad
        args = [t2 if t is x else x for x in (q, k, v)]
        leaves = [x.detach().clone().requires_grad_(True) for x in args]
        o = sparse_attention(*leaves, AttentionSegments(ql, device=device), causal=True)
        dq, dk, dv = torch.autograd.grad(o, leaves, do)
        assert torch.equal(o[:at], clean["o"][:at]) and torch.equal(dq[:at], clean["dq"][:at])
        assert not torch.isfinite(o[at:]).all()
    # a query and its gradient: keys after it keep theirs
    for which in ("q", "do"):
        q2, do2 = q.clone(), do.clone()
        (q2 if which == "q" else do2)[at, :, 3] = bad
        leaves = [x.detach().clone().requires_grad_(True) for x in (q2, k, v)]
        o = sparse_attention(*leaves, AttentionSegments(ql, device=device), causal=True)
        dq, dk, dv = torch.autograd.grad(o, leaves, do2)
        assert torch.equal(dk[at + 1:], clean["dk"][at + 1:]) and torch.equal(dv[at + 1:], clean["dv"][at + 1:])
        assert not torch.isfinite(dv[:at + 1]).all() or which == "q"


@pytest.mark.gpu
def test_a_row_that_is_not_finite_stays_in_its_segment(device):
    ql = [60, 70, 200]
    q, k, v, do, _ = _make(ql, ql, 2, 2, 32, torch.bfloat16, device, 9)
    clean = _check(q.clone(), k.clone(), v.clone(), do, ql, ql)
    k[70, 1, 0], v[80, 0, 5] = float("nan"), float("inf")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = sparse_attention(q, k, v, AttentionSegments(ql, device=device))
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    for rest in (slice(0, 60), slice(130, 330)):
        assert torch.equal(o[rest], clean["o"][rest]) and torch.equal(dk[rest], clean["dk"][rest])
    assert torch.isnan(o[60:130, 1]).all() and not torch.isfinite(o[60:130, 0, 5]).any()


@pytest.mark.gpu
def test_strides(device):
    """Slices of one projection, heads first, rows off a 16-byte address, channels apart, one key head for all."""
    n, g = 300, torch.Generator().manual_seed(10)
    segs = AttentionSegments([100, 200], device=device)
    qkv = torch.randn((n, 3, 4, 32), generator=g).to(device, torch.bfloat16)
    q, k, v = qkv.unbind(1)
    ref = sparse_attention(q.contiguous(), k.contiguous(), v.contiguous(), segs)
    assert torch.equal(sparse_attention(q, k, v, segs), ref)
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(sparse_attention(*heads_first, segs), ref)
    off = [torch.empty((n * 128 + 1,), dtype=torch.bfloat16, device=device)[1:].view(n, 4, 32).copy_(t) for t in (q, k, v)]
    assert torch.equal(sparse_attention(*off, segs), ref)
    apart = [torch.empty((n, 4, 32, 2), dtype=torch.bfloat16, device=device)[..., 1].copy_(t) for t in (q, k, v)]
    assert torch.equal(sparse_attention(*apart, segs), ref)
    one = k[:, :1].expand(n, 4, 32)
    assert torch.equal(sparse_attention(q, one, v, segs), sparse_attention(q, one.contiguous(), v, segs))
    # gradients of the slices come back into the projection; a gradient that is one value everywhere
    qkv.requires_grad_(True)
    sparse_attention(*qkv.unbind(1), segs).sum().backward()
    leaves = [t.detach().contiguous().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(sparse_attention(*leaves, segs), leaves, torch.ones_like(ref))
    assert all(torch.equal(qkv.grad[:, i], d) for i, d in enumerate(grads))
    # a broadcast key: its gradient is the sum over the heads that it was given to
    k1 = k[:, :1].detach().clone().requires_grad_(True)
    do = torch.randn(ref.shape, generator=g).to(device, torch.bfloat16)
    (d1,) = torch.autograd.grad(sparse_attention(leaves[0], k1.expand(n, 4, 32), leaves[2], segs), [k1], do)
    k4 = k1.detach().expand(n, 4, 32).contiguous().requires_grad_(True)
    (d4,) = torch.autograd.grad(sparse_attention(leaves[0], k4, leaves[2], segs), [k4], do)
    assert torch.equal(d1, d4.sum(1, keepdim=True))


@pytest.mark.gpu
def test_offsets_past_32_bits(device):
    """Keys spread over more than 2^32 bytes of one segment: rows 16 KB apart."""
    n, dim = 400_000, 64
    cache = torch.empty((n, 128, dim), dtype=torch.bfloat16, device=device)
    g = torch.Generator(device=device).manual_seed(11)
    k, v = cache[:, 3:4], cache[:, 77:78]
    k.copy_(torch.randn((n, 1, dim), generator=g, device=device))
    v.copy_(torch.randn((n, 1, dim), generator=g, device=device))
    k[-1], v[-1] = 3.0, 50.0  # the far end counts
    q = torch.full((2, 4, dim), 1.0, device=device, dtype=torch.bfloat16)
    segs = AttentionSegments([2], [n], device=device)
    got = sparse_attention(q, k, v, segs)
    ref = sparse_attention(q, k.contiguous(), v.contiguous(), segs)
    assert torch.equal(got, ref)
    s = (q[0, 0].double() @ k[:, 0].double().T) * dim ** -0.5
    want = torch.softmax(s, 0) @ v[:, 0].double()
    assert (got[0, 0].double() - want).abs().max().item() <= 2 * 2.0 ** -8 * want.abs().max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
def test_gradients_against_differences(device, causal):
    """Along random directions in fp32: central differences with e = 2^-6 (curvature e^2, rounding 2^-22 / e)."""
    ql, kl = [20, 9], [20, 30]
    q, k, v, do, mask = _make(ql, kl, 4, 2, 16, torch.float32, device, 12, masked=0.2)
    segs = AttentionSegments(ql, kl, device=device)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    f = lambda ts: (sparse_attention(*ts, segs, causal=causal, key_mask=mask).double() * do.double()).sum()  # noqa: E731
    grads = torch.autograd.grad(f(leaves), leaves)
    e = 2.0 ** -6
    for i in range(3):
        d = torch.randn_like(leaves[i])
        with torch.no_grad():
            up, down = (f([t + s * e * d if j == i else t for j, t in enumerate(leaves)]) for s in (1, -1))
        slope, got = (up - down) / (2 * e), (grads[i].double() * d.double()).sum()
        assert (slope - got).abs() <= 1e-2 * (grads[i].double() * d.double()).norm(), (i, slope.item(), got.item())


@pytest.mark.gpu
def test_the_same_bits_on_every_run_and_stream(device):
    ql = [1000, 37, 600]
    q, k, v, do, mask = _make(ql, ql, 8, 2, 64, torch.bfloat16, device, 13, masked=0.1)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    segs = AttentionSegments(ql, device=device)

    def once():
        o = sparse_attention(q, k, v, segs, key_mask=mask)
        return (o.detach(),) + torch.autograd.grad(o, leaves, do)

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    for other in (second, once()):
        assert all(torch.equal(a, b) for a, b in zip(first, other))


@pytest.mark.gpu
def test_one_gradient_alone(device):
    ql = [80, 50]
    q, k, v, do, _ = _make(ql, ql, 4, 2, 32, torch.bfloat16, device, 14)
    segs = AttentionSegments(ql, device=device)
    full = [t.clone().requires_grad_(True) for t in (q, k, v)]
    want = torch.autograd.grad(sparse_attention(*full, segs), full, do)
    for i in range(3):
        some = [t.clone().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        (got,) = torch.autograd.grad(sparse_attention(*some, segs), [some[i]], do)
        assert torch.equal(got, want[i])


@pytest.mark.gpu
def test_graph_capture_and_replay(device):
    ql, kl = [1, 1], [3000, 500]
    q, k, v, _, _ = _make(ql, kl, 8, 2, 64, torch.bfloat16, device, 15)
    segs = AttentionSegments(ql, kl, device=device)
    sparse_attention(q, k, v, segs)  # the tile lists are built by an eager call
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sparse_attention(q, k, v, segs)
    for i in range(3):
        q.copy_(torch.randn(q.shape, device=device))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, sparse_attention(q, k, v, segs))


@pytest.mark.gpu
def test_segments_of_a_tensor(device):
    b = torch.tensor([0] * 7 + [2] * 5 + [3] * 4)
    coords = torch.stack([b, torch.arange(16), torch.arange(16), torch.arange(16)], 1).to(device)
    x = SparseTensor(torch.zeros((16, 8), device=device), coords, spatial_shape=(16, 16, 16), batch_size=5)
    assert AttentionSegments.from_tensor(x)._nq.tolist() == [7, 0, 5, 4, 0]
    assert AttentionSegments.from_tensor(x, patch=4)._nq.tolist() == [4, 3, 4, 1, 4]
    with pytest.raises(ValueError, match="sample"):
        AttentionSegments.from_tensor(SparseTensor(x.F, coords.flip(0), spatial_shape=(16, 16, 16), batch_size=5))
    with pytest.raises(ValueError, match="patch"):
        AttentionSegments.from_tensor(x, patch=0)


def test_tile_lists_cover_every_pair_once():
    """Host arithmetic of the lists: each (row, key) that may be seen lies in exactly one item, and parts join in order."""
    for ql, kl, group, kv, causal, row in [([300, 1, 0, 50], [700, 3, 5, 0], 3, 1, False, 128), ([1], [5000], 1, 1, False, 256),
                                           ([1], [5000], 1, 1, False, 64), ([400, 90], [400, 20], 2, 2, True, 64),
                                           ([5], [1000], 7, 1, True, 64), ([5, 20, 3, 40], [9, 60, 3, 33], 1, 4, True, 64)]:
        s = AttentionSegments(ql, kl, device="cpu")
        for which in "qk":
            plan = s._plan(which, group, kv, causal, row)
            items = plan.words[:plan.n_items].tolist()
            joins = plan.words[plan.n_items:].tolist()
            assert len(joins) == plan.n_joins
            slots = sorted(i[7] for i in items if i[7] >= 0)
            assert slots == list(range(plan.slots)) and sum(j[6] for j in joins) == plan.slots
            q0 = k0 = 0
            for nq, nk in zip(ql, kl):
                mine = [i for i in items if i[:4] == [q0, nq, k0, nk]]
                rows, length = (nq * group, nk) if which == "q" else (nk, nq * group)
                for row0 in range(0, rows, plan.tile):
                    tile = sorted((i for i in mine if i[4] == row0), key=lambda i: i[5])
                    seen = [j for i in tile for j in range(i[5], i[6])]
                    assert len(seen) == len(set(seen)) and tile
                    if which == "q":
                        last = (min(rows, row0 + plan.tile) - 1) // group + nk - nq if causal else nk - 1
                        assert seen == list(range(0, min(nk, max(0, last + 1))))
                    else:
                        first = max(0, row0 - (nk - nq)) * group if causal else 0
                        assert seen == list(range(min(first, length), length))
                    if len(tile) > 1:
                        (join,) = [j for j in joins if j[:5] == tile[0][:5]]
                        assert [i[7] for i in tile] == list(range(join[5], join[5] + join[6]))
                    else:
                        assert tile[0][7] == -1
                q0, k0 = q0 + nq, k0 + nk


def test_refusals_before_any_launch():
    for bad, err in (([1, -1], ValueError), ([[1]], ValueError), ([1.5], ValueError), ([2 ** 31], ValueError),
                     (torch.tensor([1.0]), TypeError)):
        with pytest.raises(err):
            AttentionSegments(bad, device="cpu")
    with pytest.raises(ValueError, match="segments of queries"):
        AttentionSegments([1, 2], [3], device="cpu")
    with pytest.raises(RuntimeError, match="GPU"):
        sparse_attention(*[torch.zeros((3, 1, 8))] * 3, AttentionSegments([3], device="cpu"))
    lib = _lib.lib()
    a = _lib.AttnArgs()
    assert lib.st_attn_forward(None, None) == -1 and lib.st_attn_forward(a, None) == -1
    a.heads, a.kv_heads, a.dim, a.scale, a.dtype = 4, 2, 64, 0.125, 2
    a.q_tile, a.k_tile = _lib.ATTN_TILE, _lib.ATTN_SMALL_TILE
    assert lib.st_attn_forward(a, None) == 0 and lib.st_attn_backward(a, None) == 0  # nothing to do
    for field, value, rc in (("kv_heads", 3, -1), ("dim", 20, -3), ("dim", 136, -3), ("dtype", 3, -3), ("scale", 0.0, -1),
                             ("scale", float("nan"), -1), ("n_q_items", -1, -1), ("n_q_items", 1, -1),
                             ("q_tile", 64, -1), ("k_tile", 0, -1)):
        old = getattr(a, field)
        setattr(a, field, value)
        assert lib.st_attn_forward(a, None) == rc, field
        setattr(a, field, old)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float16, 24), (torch.float32, 32), (torch.float32, 64)])
@pytest.mark.parametrize("causal", [False, True])
def test_windows(device, dtype, dim, causal):
    """Many segments of a few rows: tiles of one wave where a row of a head is at most 128 bytes."""
    ql = [1, 17, 32, 33, 5, 90, 31, 0, 64, 2] * 12
    kl = [9, 17, 32, 1, 70, 90, 0, 3, 65, 2] * 12
    q, k, v, do, mask = _make(ql, kl, 4, 2, dim, dtype, device, 18, masked=0.1)
    tile = AttentionSegments(ql, kl, device=device)._plan("k", 2, 2, causal, dim * q.element_size()).tile
    assert tile == (32 if dim * q.element_size() <= 128 else 128)
    _check(q, k, v, do, ql, kl, causal, mask)


@pytest.mark.gpu
def test_refusals(device):
    segs = AttentionSegments([4, 2], device=device)
    q = torch.zeros((6, 4, 16), device=device)
    for args in ((q[:5], q, q), (q, q[:5], q[:5]), (q, q[:, :3], q[:, :3]), (q, q, q[:, :2]), (q[0], q, q),
                 (q, q.half(), q.half()), (q, q[:, :0], q[:, :0])):
        with pytest.raises(ValueError):
            sparse_attention(*args, segs)
    for dim in (4, 20, 136):
        with pytest.raises(ValueError, match="head size"):
            t = torch.zeros((6, 2, dim), device=device)
            sparse_attention(t, t, t, segs)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            sparse_attention(q, q, q, segs, scale=scale)
    with pytest.raises(TypeError, match="bool"):
        sparse_attention(q, q, q, segs, key_mask=torch.ones(6, device=device))
    with pytest.raises(ValueError, match="key_mask"):
        sparse_attention(q, q, q, segs, key_mask=torch.ones(5, device=device, dtype=torch.bool))
    with pytest.raises(ValueError, match="segments are on"):
        sparse_attention(q, q, q, AttentionSegments([4, 2], device="cpu"))
    with pytest.raises(TypeError):
        sparse_attention(q.double(), q.double(), q.double(), segs)
    with pytest.raises(RuntimeError, match="GPU"):
        sparse_attention(q.cpu(), q, q, segs)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim,heads,kv_heads", [(32, 4, 2), (64, 2, 2), (128, 2, 1)])
def test_roundings_of_the_gradients_of_few_keys(device, dtype, causal, dim, heads, kv_heads):
    """Norm of the errors of dQ and dK: the result's own rounding, and what rounding P (for O, in units of the
    row's largest, hence delta) and dS does in float64; O's own rounding has no part in it.  The two are
    independent: their squares add, a tenth more for what of them is chance."""
    lens = list(range(1, 9)) * 40
    q, k, v, do, _ = _make(lens, lens, heads, kv_heads, dim, dtype, device, 5)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = sparse_attention(*leaves, AttentionSegments(lens, device=device), causal=causal)
    got = dict(zip(("dq", "dk"), torch.autograd.grad(o, leaves, do)))
    ref = _reference(q, k, v, do, lens, lens, dim ** -0.5, causal, None)
    rounded = lambda t: t.to(dtype).double()  # noqa: E731
    off = {n: torch.zeros(ref[n][0].shape, dtype=torch.float64) for n in ("dq", "dk")}
    q, k, v, do = (t.detach().cpu().double() for t in (q, k, v, do))
    at = 0
    for n in lens:
        rows = slice(at, at + n)
        at += n
        see = torch.ones((n, n), dtype=torch.bool)
        for h in range(heads):
            hk = h * kv_heads // heads
            s = q[rows, h] @ k[rows, hk].T * dim ** -0.5
            p = torch.softmax(s.masked_fill(~(see.tril() if causal else see), -math.inf), 1)
            top = p.amax(1, keepdim=True)
            dp = do[rows, h] @ v[rows, hk].T
            ds = p * (dp - (p * dp).sum(1, keepdim=True))
            error = rounded(p * (dp - (rounded(p / top) * top * dp).sum(1, keepdim=True))) - ds
            off["dq"][rows, h] = error @ k[rows, hk] * dim ** -0.5
            off["dk"][rows, hk] += error.T @ q[rows, h] * dim ** -0.5
    for n in off:
        want = ref[n][0]
        expected = math.hypot((rounded(want) - want).norm().item(), off[n].norm().item())
        error = (got[n].double() - want).norm().item()
        assert error < 1.1 * expected, (n, error / expected, expected / want.norm().item())


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [16, 64, 128])
@pytest.mark.parametrize("step", range(0, 54, 9))
def test_small_probabilities_in_float16(device, step, dim):
    """One key far above the others, whose probabilities (~2^-16) are below the type's normal numbers.  V and dO
    ask for the others alone; P and the result are rounded once each, 2^-11."""
    n, a = 64, 2.76171875 + step / 512
    q, k, v = (torch.zeros((n, 1, dim), dtype=torch.float16, device=device) for _ in range(3))
    q[:, 0, 0], k[0, 0, 0], v[1:] = a, 4.0, 1.0
    do = torch.full_like(q, 1024.0)
    r = math.exp(-4 * a)
    p = r / (1 + (n - 1) * r)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = sparse_attention(*leaves, AttentionSegments([n], device=device), scale=1.0)
    dv = torch.autograd.grad(o, v, do)[0]
    bound = 2 * 2.0 ** -11 + W
    assert (o.double() / ((n - 1) * p) - 1).abs().max().item() <= bound
    assert (dv[1:].double() / (n * 1024 * p) - 1).abs().max().item() <= bound


@pytest.mark.parametrize("elem,dim", [(2, 32), (2, 128), (4, 64)])
@pytest.mark.parametrize("causal", [False, True])
def test_which_tiles_are_split(elem, dim, causal):
    """Few tiles over many keys are, tiles that fill the chip are not, and a long segment beside many short ones is
    alone among them; every part has work and the parts of a tile follow one another without a gap."""
    for lengths, split in (([1] * 4, False), ([30_000] * 2, True), ([1024] * 64, False), ([30_000] + [50] * 600, True),
                           ([0, 0], False)):
        plan = AttentionSegments([min(n, 128) for n in lengths], lengths, device="cpu")._plan("q", 1, 8, causal, dim * elem, elem)
        words = plan.words.numpy()
        items, joins = words[:plan.n_items], words[plan.n_items:]
        assert (joins.shape[0] > 0) == split
        for q0, nq, k0, nk, row0, first, parts, _ in joins:
            mine = items[(items[:, 0] == q0) & (items[:, 4] == row0)]
            mine = mine[mine[:, 7].argsort()]
            assert nk == 30_000 and parts > 1 and (mine[:, 7] == range(first, first + parts)).all()
            assert mine[0, 5] == 0 and (mine[1:, 5] == mine[:-1, 6]).all() and (mine[:, 6] > mine[:, 5]).all()
            assert (mine[:, 5] % 64 == 0).all() and mine[-1, 6] <= nk


def _float16_gradients(q, k, v, do, ql, kl, scale, causal):
    """{name: (value, error)} in float64: dQ, dK, dV and what the two roundings on the way do to them in float16 -- P
    (in units of its row's largest, times 2^7 for O and 2^14 for dV) and dS, at a power of two of each row (dQ) or
    key (dK), so that it neither overflows nor loses digits below 2^-14."""
    def rounded(t, power=0.0):
        return (t * 2.0 ** power).half().double() * 2.0 ** -power

    def held(t, axis):
        return rounded(t, 9 - torch.frexp(t.abs().amax(axis, keepdim=True)).exponent.double())

    group = q.shape[1] // k.shape[1]
    q, k, v, do = (t.detach().double() for t in (q, k, v, do))
    val = {n: torch.zeros_like(t) for n, t in (("dq", q), ("dk", k), ("dv", v))}
    off = {n: torch.zeros_like(t) for n, t in val.items()}
    q0 = k0 = 0
    for nq, nk in zip(ql, kl):
        Q, K = slice(q0, q0 + nq), slice(k0, k0 + nk)
        see = torch.ones((nq, nk), dtype=torch.bool, device=q.device)
        see = see.tril(nk - nq) if causal else see
        for h in range(k.shape[1]):
            H = slice(h * group, (h + 1) * group)
            a, g = (t[Q, H].transpose(0, 1).reshape(group * nq, -1) for t in (q, do))
            b, c = k[K, h], v[K, h]
            p = torch.softmax((a @ b.T * scale).masked_fill(~see.repeat(group, 1), -math.inf), 1)
            dp, top = g @ c.T, p.amax(1, keepdim=True)
            ds = p * (dp - (p * dp).sum(1, keepdim=True))
            near = p * (dp - (rounded(p / top, 7) * top * dp).sum(1, keepdim=True))
            rows = lambda t: t.view(group, nq, -1).transpose(0, 1)  # noqa: E731
            val["dq"][Q, H], off["dq"][Q, H] = rows(ds @ b * scale), rows((held(near, 1) - ds) @ b * scale)
            val["dk"][K, h], off["dk"][K, h] = ds.T @ a * scale, (held(near, 0) - ds).T @ a * scale
            val["dv"][K, h], off["dv"][K, h] = p.T @ g, (rounded(p, 14) - p).T @ g
        q0, k0 = q0 + nq, k0 + nk
    return {n: (t, off[n]) for n, t in val.items()}


def _check_float16_gradients(q, k, v, do, ql, kl, scale, causal, bands=None):
    """No infinity where the value has none, and the norm of the errors (of each band of query rows) within a tenth
    of its own rounding's and the roundings' on the way: independent, so their squares add."""
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = sparse_attention(*leaves, AttentionSegments(ql, kl, device=q.device), scale=scale, causal=causal)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, do)))
    for n, (want, off) in _float16_gradients(q, k, v, do, ql, kl, scale, causal).items():
        assert want.abs().max().item() < 65504, "the case itself is out of float16's range"
        assert torch.isfinite(got[n]).all(), n
        for rows in (bands if bands and n == "dq" else [slice(None)]):
            w = want[rows]
            expected = math.hypot((w.half().double() - w).norm().item(), off[rows].norm().item())
            error = (got[n][rows].double() - w).norm().item()
            assert error < 1.1 * expected, (n, rows, error / expected, expected / w.norm().item())


@pytest.mark.gpu
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 1, 1), (128, 4, 2), (64, 4, 2), (32, 2, 2)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("seed", range(3))
def test_float16_gradients_of_a_large_loss_scale(device, dim, heads, kv_heads, causal, seed):
    """dO near 8,000: dS passes 65,504 where dQ, dK and dV do not (few keys, so that P is not small)."""
    ql = [8, 3, 8, 40, 8]
    q, k, v, do, _ = _make(ql, ql, heads, kv_heads, dim, torch.float16, device, seed)
    q, k, v = q * 0.5, k * 0.5, v * (24.0 / dim ** 0.5)
    do = (do.float() * 8000).clamp(-30000, 30000).half()
    _check_float16_gradients(q, k, v, do, ql, ql, dim ** -0.5, causal)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-2, 1e-3])
@pytest.mark.parametrize("ql,kl,heads,kv_heads,dim", [
    ([20], [20_000], 2, 1, 32), ([300], [4000], 2, 2, 128), ([2048], [2048], 1, 1, 32), ([6000], [64], 2, 1, 64)])
def test_float16_gradients_of_small_products(device, size, ql, kl, heads, kv_heads, dim):
    """dO of 1e-2 and less over many keys or rows: dS lies below 2^-14, dQ, dK and dV (at a scale of one) less so."""
    q, k, v, do, _ = _make(ql, kl, heads, kv_heads, dim, torch.float16, device, dim + ql[0])
    q = q * dim ** -0.5
    _check_float16_gradients(q, k, v, (do.float() * size).half(), ql, kl, 1.0, False)


@pytest.mark.gpu
@pytest.mark.parametrize("falling", [False, True])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_float16_gradients_of_unlike_rows(device, falling, dim, causal):
    """Rows whose dO grows (falls) from 2^-14 to 2^7 along the segment, keys whose values do from 2^-6 to 2^3: the power
    that a row's or key's sum is held at has to follow, and small rows keep their digits beside large ones."""
    n = 1024
    q, k, v, do, _ = _make([n], [n], 2, 1, dim, torch.float16, device, dim + falling)
    size = torch.linspace(-14, 7, n, device=device)
    keys = torch.linspace(-6, 3, n, device=device)
    if falling:
        size, keys = size.flip(0), keys.flip(0)
    do = (do.float() * torch.exp2(size)[:, None, None]).half()
    v = (v.float() * torch.exp2(keys)[:, None, None]).half()
    _check_float16_gradients(q * dim ** -0.5, k, v, do, [n], [n], 1.0, causal,
                             [slice(i, i + 128) for i in range(0, n, 128)])


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("recorded", [False, True])
def test_forward_mode_is_refused(device, own_random, which, recorded):
    """No forward-mode derivative: a tangent on q, k or v raises, where it is not to be dropped, with or without a graph."""
    t = [torch.randn((6, 2, 16), device=device, requires_grad=recorded) for _ in range(3)]
    segs = AttentionSegments([4, 2], device=device)
    with torch.autograd.forward_ad.dual_level():
        sparse_attention(*t, segs)
        t[which] = torch.autograd.forward_ad.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            sparse_attention(*t, segs)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            sparse_attention(*t, segs)


@pytest.mark.parametrize("copied", [copy.copy, copy.deepcopy, lambda s: pickle.loads(pickle.dumps(s))])
def test_copies_build_their_own_lists(copied):
    """The lists hold addresses of their own device memory: a copy (of a model that holds the segments, or on its way to
    another process) must not keep them.  Same lengths, same lists."""
    segs = AttentionSegments([300, 5], [5000, 7], device="cpu")
    plans = [segs._plan(w, 2, 2, False, 64, 2) for w in "qk"]
    other = copied(segs)
    assert (other.q_rows, other.k_rows, other.count, other.device) == (305, 5007, 2, segs.device)
    for w, plan in zip("qk", plans):
        again = other._plan(w, 2, 2, False, 64, 2)
        assert torch.equal(again.words, plan.words) and again.words.data_ptr() != plan.words.data_ptr()
        assert again.items == again.words.data_ptr() and segs._plan(w, 2, 2, False, 64, 2) is plan


@pytest.mark.parametrize("bad", [[2 ** 62] * 4, [2 ** 63 - 1, 2 ** 63 - 1, 2], [2 ** 33] * 2 ** 3])
def test_lengths_whose_sum_wraps_are_refused(bad):
    """Four segments of 2^62 rows are 2^64 in all: zero in 64 bits."""
    with pytest.raises(ValueError, match="2\\^31"):
        AttentionSegments(bad, device="cpu")
    with pytest.raises(ValueError, match="2\\^31"):
        AttentionSegments([1] * len(bad), bad, device="cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("segments,heads,dim", [((1 << 20) + 3, 16, 72), ((1 << 22) + 3, 16, 8)])
def test_more_workgroups_than_one_launch_takes(device, segments, heads, dim):
    """A grid has fewer than 2^32 threads a dimension: 2^24 workgroups of four waves (wide rows), 2^26 of one."""
    small = 1000
    g = torch.Generator().manual_seed(22)
    part = [torch.randn((small, heads, dim), generator=g).to(device, torch.bfloat16) for _ in range(4)]
    whole = [t.repeat(-(-segments // small), 1, 1)[:segments] for t in part]
    segs, few = AttentionSegments(np.ones(segments, np.int64), device=device), AttentionSegments([1] * small, device=device)
    tile = segs._plan("q", 1, heads, False, 2 * dim, 2).tile
    assert segments * heads * 2 * tile > 2 ** 32

    def once(q, k, v, do, s):
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        o = sparse_attention(*leaves, s)
        return (o.detach(),) + torch.autograd.grad(o, leaves, do)

    for got, want in zip(once(*whole, segs), once(*part, few)):
        for at in range(0, segments, 1 << 18):  # (a few hundred thousand rows of it at once)
            rows = got[at:at + (1 << 18)]
            assert torch.equal(rows, want[torch.arange(at, at + len(rows), device=device) % small])


def _check_calls(q, k, v, do, ql, kl, causal, mask):
    """As _check, with what its bound leaves out: a float16 result below 2^-14 is rounded by up to half a spacing, 2^-25."""
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = sparse_attention(*leaves, AttentionSegments(ql, kl, device=q.device), causal=causal, key_mask=mask)
    got = dict(zip(("o", "dq", "dk", "dv"), (o.detach(),) + torch.autograd.grad(o, leaves, do)))
    least = 2.0 ** -25 if q.dtype is torch.float16 else 0.0
    for n, (want, bound) in _reference(q, k, v, do, ql, kl, q.shape[2] ** -0.5, causal, mask).items():
        over = (got[n].double() - want).abs() - bound - least
        assert not torch.isnan(got[n]).any() and over.max().item() <= 0, (n, over.max().item())


@pytest.mark.gpu
@pytest.mark.parametrize("ql,kl,heads,kv_heads,dim,causal", [
    ([1], [5000], 4, 1, 64, False), ([1, 1, 2], [1, 4097, 300], 8, 2, 128, True), ([2500], [40], 2, 1, 32, False),
    ([1000], [1000], 1, 1, 64, True), ([1500, 20], [1, 2000], 2, 2, 48, False), ([700, 30], [700, 3000], 4, 2, 96, True)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_joins_of_every_type(device, ql, kl, heads, kv_heads, dim, causal, dtype):
    """Split tiles and their joins, by the lists that the calls use."""
    q, k, v, do, mask = _make(ql, kl, heads, kv_heads, dim, dtype, device, 5 * dim, masked=0.1)
    segs = AttentionSegments(ql, kl, device=device)
    e = q.element_size()
    joins = [segs._plan(w, heads // kv_heads, kv_heads, causal, dim * e, e).n_joins for w in "qk"]
    assert joins[0] if max(kl) > max(ql) else joins[1]
    _check_calls(q, k, v, do, ql, kl, causal, mask)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype,dim", [(torch.float16, 64), (torch.float32, 32)])
def test_many_whole_tiles(device, causal, dtype, dim):
    """Enough workgroups that nothing is split, by the lists that the calls use."""
    ql = [700, 1, 333, 900, 64, 128, 2] * 16
    q, k, v, do, mask = _make(ql, ql, 8, 4, dim, dtype, device, 19, masked=0.05)
    segs, e = AttentionSegments(ql, device=device), q.element_size()
    assert not any(segs._plan(w, 2, 4, causal, dim * e, e).n_joins for w in "qk")
    _check_calls(q, k, v, do, ql, ql, causal, mask)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [16, 64, 128])
@pytest.mark.parametrize("step", range(0, 36, 9))
def test_small_probabilities_of_split_rows_in_float16(device, step, dim):
    """As test_small_probabilities_in_float16, one row over keys that are split: the others' ~2^-20 come out of parts
    whose maximum is their own, and out of the first key's, whose maximum is one."""
    n, a = 4096, 3.390625 + step / 512
    q = torch.zeros((1, 1, dim), dtype=torch.float16, device=device)
    k, v = (torch.zeros((n, 1, dim), dtype=torch.float16, device=device) for _ in range(2))
    q[:, 0, 0], k[0, 0, 0], v[1:] = a, 4.0, 1.0
    segs = AttentionSegments([1], [n], device=device)
    assert segs._plan("q", 1, 1, False, 2 * dim, 2).n_joins == 1
    r = math.exp(-4 * a)
    p = r / (1 + (n - 1) * r)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = sparse_attention(*leaves, segs, scale=1.0)
    dv = torch.autograd.grad(o, v, torch.full_like(q, 1024.0))[0]
    bound = 2 * 2.0 ** -11 + W
    assert (o.double() / ((n - 1) * p) - 1).abs().max().item() <= bound
    assert (dv[1:].double() / (1024 * p) - 1).abs().max().item() <= bound


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("causal", [False, True])
def test_training_pass_in_a_graph(device, own_random, dtype, causal):
    """A recorded call and its gradients captured together, replayed on other values between eager calls."""
    ql = [700, 33, 1]
    q, k, v, do, mask = _make(ql, ql, 4, 2, 32, dtype, device, 20, masked=0.1)
    segs = AttentionSegments(ql, device=device)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]

    def once():
        o = sparse_attention(*leaves, segs, causal=causal, key_mask=mask)
        return (o.detach(),) + torch.autograd.grad(o, leaves, do)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()  # the tile lists are built by an eager call
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for i in range(3):
        with torch.no_grad():
            for t in leaves + [do]:
                t.copy_(torch.randn(t.shape, device=device))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, once())), i


@pytest.mark.gpu
def test_threads_share_the_segments(device):
    """Two threads, each on a stream of its own, with one AttentionSegments whose lists are not built yet."""
    ql = [900, 40, 3]
    data = [_make(ql, ql, 4, 2, 64, torch.bfloat16, device, 21 + i)[:4] for i in range(2)]

    def once(i, segs):
        q, k, v, do = data[i]
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        o = sparse_attention(*leaves, segs, causal=True)
        return (o.detach(),) + torch.autograd.grad(o, leaves, do)

    want = [once(i, AttentionSegments(ql, device=device)) for i in range(2)]
    segs, start = AttentionSegments(ql, device=device), threading.Barrier(2)
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            start.wait(30)
            got = [once(i, segs) for _ in range(5)]
            torch.cuda.current_stream().synchronize()
        return got

    with concurrent.futures.ThreadPoolExecutor(2) as pool:
        for i, runs in enumerate(pool.map(work, range(2))):
            assert all(torch.equal(a, b) for got in runs for a, b in zip(got, want[i]))
