"""sparse_attention with a window and sinks against the formulas in float64.

A row at place p = i + nk - nq sees key j where |p - j| < window or j < sinks (and j <= p under causal).
Bounds, per element, from the roundings on the way (u: half a unit of the type, 2^-8, 2^-11 or 0 for
fp32 products; w = 512 * 2^-24 for what fp32 does to a score of |q||k| c ~ 11 summed over 128
channels, its exponential and the row's sum):
  P    (u + w) P                                  (rounded for the second product)
  O    (u + w) sum P |v|  + u |O|                 (float16 also loses 2^-25 of P below 2^-14)
  dP - delta   w sum |dO||v|  + sum |dO| (error of O)
  dS   (2 u + w) |dS| + P (error of dP - delta)
  dQ, dK, dV   the error of dS or P through the product, plus u of the result (float16: 2^-25 at least).
"""

import random

import numpy as np
import pytest
import torch

from sparsetriton_amd import _lib
from sparsetriton_amd.nn.functional import AttentionSegments, sparse_attention

UNIT = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
W = 512 * 2.0 ** -24


def _sees(nq, nk, causal, window, sinks, device="cpu"):
    away = torch.arange(nk, device=device)[None] - (torch.arange(nq, device=device) + (nk - nq))[:, None]
    see = (away.abs() < window) | (torch.arange(nk, device=device) < sinks)[None]
    return see & (away <= 0) if causal else see


def _reference(q, k, v, do, ql, kl, causal, window, sinks, mask):
    """{name: (value, bound)} in float64."""
    u, tiny = UNIT[q.dtype], 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    last, scale = max(u, 2.0 ** -24), q.shape[2] ** -0.5
    group = q.shape[1] // k.shape[1]
    q, k, v, do = (t.detach().double() for t in (q, k, v, do))
    if mask is not None:
        k, v = (t.masked_fill(~mask[:, None, None], 0.0) for t in (k, v))
    val = {n: torch.zeros_like(t) for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    err = {n: torch.zeros_like(t) for n, t in val.items()}
    q0 = k0 = 0
    for nq, nk in zip(ql, kl):
        Q, K = slice(q0, q0 + nq), slice(k0, k0 + nk)
        see = _sees(nq, nk, causal, window, sinks, q.device)
        if mask is not None:
            see = see & mask[K]
        for h in range(q.shape[1] if nq and nk else 0):
            a, b, c, g = q[Q, h], k[K, h // group], v[K, h // group], do[Q, h]
            s = (a @ b.T * scale).masked_fill(~see, float("-inf"))
            p = torch.exp(s - s.amax(1, keepdim=True).clamp_min(-1e300))
            total = p.sum(1, keepdim=True)
            p = p / total.masked_fill(total == 0, 1.0)
            o = p @ c
            ep = (u + W) * p + tiny * see
            eo = ep @ c.abs() + last * o.abs()
            ds = p * (g @ c.T - (g * o).sum(1, keepdim=True))
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
    # (a float16 result below 2^-14 lies between numbers 2^-24 apart: rounding it moves it by up to 2^-25, not by u of itself)
    return {n: (t, err[n] + last * t.abs() + tiny + 1e-12) for n, t in val.items()}


def _make(ql, kl, heads, kv_heads, dim, dtype, device, seed, masked=0.0):
    g = torch.Generator().manual_seed(seed)
    rand = lambda n, h: torch.randn((n, h, dim), generator=g).to(device, dtype)  # noqa: E731
    q, do = rand(sum(ql), heads), rand(sum(ql), heads)
    k, v = rand(sum(kl), kv_heads), rand(sum(kl), kv_heads)
    mask = (torch.rand((sum(kl),), generator=g) >= masked).to(device) if masked else None
    return q, k, v, do, mask


def _run(q, k, v, do, segs, **kw):
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
    o = sparse_attention(*leaves, segs, **kw)
    return dict(zip(("o", "dq", "dk", "dv"), (o.detach(),) + torch.autograd.grad(o, leaves, do)))


def _check(q, k, v, do, ql, kl, causal, window, sinks, mask=None):
    segs = AttentionSegments(ql, kl, device=q.device)
    kw = dict(causal=causal, key_mask=mask, window=window, sinks=sinks)
    got = _run(q, k, v, do, segs, **kw)
    with torch.no_grad():
        assert torch.equal(got["o"], sparse_attention(q, k, v, segs, **kw))
    for n, (want, bound) in _reference(q, k, v, do, ql, kl, causal, window, sinks, mask).items():
        assert got[n].shape == want.shape and got[n].dtype == q.dtype and got[n].is_contiguous()
        assert not torch.isnan(got[n]).any(), n
        over = (got[n].double() - want).abs() - bound
        assert over.numel() == 0 or over.max().item() <= 0, (n, over.max().item(), want.abs().max().item())
    return got


# ------------------------------------------------------------------ the work lists, on the host

LISTS = [([300, 1, 0, 50], [700, 3, 5, 0], 3), ([1], [5000], 1), ([400, 90], [400, 20], 2), ([5], [1000], 7),
         ([5, 20, 3, 40], [9, 60, 3, 33], 1), ([700], [700], 1), ([1000], [300], 4)]


@pytest.mark.parametrize("ql,kl,group", LISTS)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 3), (64, 64), (100, 65), (33, 200), (250, 1), (5, 0)])
def test_tile_lists_cover_what_is_seen_once(ql, kl, group, causal, window, sinks):
    s = AttentionSegments(ql, kl, device="cpu")
    window, sinks = s._window(causal, window, sinks)
    for which in "qk":
        plan = s._plan(which, group, 2, causal, 128, 2, window, sinks)
        items = plan.words[:plan.n_items].tolist()
        slots = sorted(i[7] for i in items if i[7] >= 0)
        assert slots == list(range(plan.slots))
        q0 = k0 = 0
        for nq, nk in zip(ql, kl):
            see = _sees(nq, nk, causal, window, sinks) if window else _sees(nq, nk, causal, 10 ** 6, 0)
            mine = [i for i in items if i[:4] == [q0, nq, k0, nk]]
            rows, end = (nq * group, nk) if which == "q" else (nk, nq * group)
            for row0 in range(0, rows, plan.tile):
                tile = sorted((i for i in mine if i[4] == row0), key=lambda i: i[5])
                assert tile and all(a[6] == b[5] for a, b in zip(tile, tile[1:])) and (len(tile) > 1) == (tile[0][7] >= 0)
                lo, hi = tile[0][5], tile[-1][6]
                if which == "q":
                    assert all((i[5] - lo) % 64 == 0 for i in tile)
                    first, last = row0 // group, (min(rows, row0 + plan.tile) - 1) // group
                    seen = see[first:last + 1].any(0)
                    f = max(0, first + nk - nq - window + 1) if window else 0
                    gap = max(0, f - sinks)
                    assert hi + gap <= nk and lo == 0
                    walked = torch.zeros(nk, dtype=torch.bool)
                    for p in range(lo, hi):
                        key = p + gap if p >= sinks else p
                        assert not walked[key]
                        walked[key] = True
                    assert not (seen & ~walked).any()
                    # and no more than the sinks and what lies between the outer rows' windows
                    assert int(walked.sum()) <= sinks + max(0, last - first + (2 if not causal else 1) * (window or nk))
                else:
                    seen = see[:, row0:row0 + plan.tile].any(1).nonzero().flatten().tolist()
                    if seen:
                        assert lo <= seen[0] * group and hi >= (seen[-1] + 1) * group
                    assert 0 <= lo <= hi <= end
            q0, k0 = q0 + nq, k0 + nk


def test_a_window_that_leaves_nothing_out_is_none():
    s = AttentionSegments([5, 9], [20, 7], device="cpu")
    assert s._window(True, 20, 0) == (0, 0) and s._window(True, 19, 0) == (19, 0)
    assert s._window(True, 16, 4) == (0, 0) and s._window(True, 15, 4) == (15, 4)
    assert s._window(False, 20, 0) == (0, 0) and s._window(False, 16, 4) == (16, 4)
    assert s._window(False, 3, 2 ** 40) == (0, 0) and s._window(False, 2 ** 40, 0) == (0, 0)


def test_segments_of_an_older_pickle():
    """Segments that were saved before they knew their longest ones, with other data of a set of scenes, say."""
    segs = AttentionSegments([300, 5], [5000, 7], device="cpu")
    state = {n: t for n, t in segs.__getstate__().items() if n not in ("_most_q", "_most_k")}
    old = AttentionSegments.__new__(AttentionSegments)
    old.__setstate__(state)
    for window, sinks in ((0, 0), (100, 4)):
        for w in "qk":
            assert torch.equal(old._plan(w, 2, 2, True, 128, 2, window, sinks).words, segs._plan(w, 2, 2, True, 128, 2, window, sinks).words)
    assert old._window(True, 100, 4) == (100, 4) and old._window(True, 5000, 0) == (0, 0)


def test_refusals_of_the_library():
    lib = _lib.lib()
    a = _lib.AttnArgs()
    a.heads, a.kv_heads, a.dim, a.scale, a.dtype = 4, 2, 64, 0.125, 2
    a.q_tile, a.k_tile = _lib.ATTN_TILE, _lib.ATTN_TILE
    for window, sinks, rc in ((0, 0, 0), (5, 0, 0), (5, 7, 0), (-1, 0, -1), (5, -1, -1), (0, 3, -1)):
        a.window, a.sinks = window, sinks
        assert lib.st_attn_forward(a, None) == rc and lib.st_attn_backward(a, None) == rc


# ------------------------------------------------------------------ values

LENGTHS = [([1], [1]), ([1, 1, 1], [1, 700, 90]), ([5], [64]), ([33, 1, 127, 2], [33, 1, 127, 2]), ([0, 7, 0, 3], [4, 0, 0, 9]),
           ([300], [300]), ([200, 10], [3, 150]), ([70], [900])]


@pytest.mark.gpu
@pytest.mark.parametrize("ql,kl", LENGTHS)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 3), (100, 0), (65, 70), (3, 130)])
@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [(torch.bfloat16, 4, 4, 64), (torch.float16, 6, 2, 40),
                                                     (torch.float32, 3, 1, 32), (torch.bfloat16, 8, 1, 128)])
def test_lengths(device, ql, kl, causal, window, sinks, dtype, heads, kv_heads, dim):
    q, k, v, do, _ = _make(ql, kl, heads, kv_heads, dim, dtype, device, sum(ql) + dim)
    _check(q, k, v, do, ql, kl, causal, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [8, 24, 32, 48, 64, 80, 96, 104, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
def test_head_sizes(device, dim, dtype, causal):
    ql = [70, 3, 250]
    q, k, v, do, mask = _make(ql, ql, 4, 2, dim, dtype, device, dim, masked=0.3)
    _check(q, k, v, do, ql, ql, causal, 40, 5, mask)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (7, 1), (12, 4), (40, 2)])
@pytest.mark.parametrize("causal", [False, True])
def test_shared_key_heads(device, heads, kv_heads, causal):
    ql, kl = [45, 1, 300], [61, 77, 300]
    q, k, v, do, mask = _make(ql, kl, heads, kv_heads, 32, torch.bfloat16, device, heads, masked=0.2)
    _check(q, k, v, do, ql, kl, causal, 50, 4, mask)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [2, 4])
def test_many_short_segments(device, causal, dtype, heads):
    """Tiles of one wave (of keys; of rows without shared key heads), and the steps of 32 keys that it takes."""
    ql = [1, 17, 32, 33, 5, 90, 31, 0, 64, 2, 96] * 12
    kl = [9, 17, 32, 1, 70, 90, 0, 3, 65, 2, 96] * 12
    q, k, v, do, mask = _make(ql, kl, heads, 2, 32, dtype, device, 18, masked=0.1)
    segs = AttentionSegments(ql, kl, device=device)
    tiles = [segs._plan(w, heads // 2, 2, causal, 32 * q.element_size(), q.element_size(), 10, 2).tile for w in "qk"]
    assert tiles == [32 if heads == 2 else 128, 32]
    for window, sinks in ((10, 2), (20, 0), (4, 33)):
        _check(q, k, v, do, ql, kl, causal, window, sinks, mask)


@pytest.mark.gpu
@pytest.mark.parametrize("ql,kl,window,sinks,causal", [
    ([1], [20_000], 4096, 4, True), ([1, 1, 2], [5000, 1, 9000], 2500, 130, True), ([3], [9001], 3000, 64, False),
    ([4000], [4000], 300, 70, True), ([4000], [4000], 40, 1, False), ([6000], [500], 100, 20, False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_work_split_over_the_long_side(device, ql, kl, window, sinks, causal, dtype):
    q, k, v, do, mask = _make(ql, kl, 4, 2, 64, dtype, device, 3, masked=0.1)
    segs = AttentionSegments(ql, kl, device=device)
    plans = [segs._plan(w, 2, 2, causal, 64 * q.element_size(), q.element_size(), window, sinks) for w in "qk"]
    assert any(p.n_joins for p in plans)
    _check(q, k, v, do, ql, kl, causal, window, sinks, mask)


@pytest.mark.gpu
def test_drawn_cases(device):
    rng = random.Random(5)
    for i in range(40):
        segs = rng.randint(1, 4)
        ql = [rng.choice([0, 1, rng.randint(1, 500)]) for _ in range(segs)]
        kl = ql if rng.random() < 0.4 else [rng.choice([0, 1, n, rng.randint(1, 700)]) for n in ql]
        kv_heads, group = rng.choice([1, 2, 3]), rng.choice([1, 2, 4, 5])
        dim, dtype = rng.choice([16, 32, 64, 80, 128]), rng.choice(list(UNIT))
        window, sinks, causal = int(np.exp(rng.uniform(0, np.log(600)))), rng.choice([0, 0, 1, 4, 64, 100]), rng.random() < 0.5
        print(i, ql, kl, kv_heads, group, dim, dtype, window, sinks, causal, flush=True)
        q, k, v, do, mask = _make(ql, kl, kv_heads * group, kv_heads, dim, dtype, device, i, masked=rng.choice([0.0, 0.5]))
        _check(q, k, v, do, ql, kl, causal, window, sinks, mask)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
def test_a_wide_window_changes_no_bit(device, causal):
    ql, kl = [200, 31], [300, 31]
    q, k, v, do, _ = _make(ql, kl, 4, 2, 64, torch.bfloat16, device, 2)
    segs = AttentionSegments(ql, kl, device=device)
    want = _run(q, k, v, do, segs, causal=causal)
    for window, sinks in ((300, 0), (2 ** 40, 5), (1, 300)):
        got = _run(q, k, v, do, segs, causal=causal, window=window, sinks=sinks)
        assert all(torch.equal(got[n], want[n]) for n in want)


# ------------------------------------------------------------------ masks, and what is not finite


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
def test_rows_whose_window_is_masked_see_the_sinks_or_nothing(device, causal):
    ql = [400]
    q, k, v, do, _ = _make(ql, ql, 4, 2, 64, torch.bfloat16, device, 6)
    mask = torch.ones(400, dtype=torch.bool, device=device)
    mask[150:260] = False
    for sinks in (0, 3):
        got = _check(q, k, v, do, ql, ql, causal, 20, sinks, mask)
        if not sinks:
            assert not got["o"][175:235].any() and not got["dq"][175:235].any()
        assert not got["dk"][150:260].any() and not got["dv"][150:260].any()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 32), (torch.bfloat16, 32)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("at", [2, 130, 201])
def test_a_row_that_is_not_finite_stays_in_its_windows(device, bad, dtype, dim, causal, at):
    ql, window, sinks = [300, 20], 30, 4
    q, k, v, do, _ = _make(ql, ql, 4, 2, dim, dtype, device, 8)
    segs = AttentionSegments(ql, device=device)
    kw = dict(causal=causal, window=window, sinks=sinks)
    clean = _run(q, k, v, do, segs, **kw)
    see = torch.zeros((320, 320), dtype=torch.bool, device=device)
    see[:300, :300] = _sees(300, 300, causal, window, sinks, device)
    rows, keys = see[:, at], see[at]
    for which in ("v", "k"):  # the rows that do not see it keep theirs
        t = {"q": q, "k": k, "v": v, which: (k if which == "k" else v).clone()}
        t[which][at, :, 3] = bad
        got = _run(t["q"], t["k"], t["v"], do, segs, **kw)
        assert torch.equal(got["o"][~rows], clean["o"][~rows]) and torch.equal(got["dq"][~rows], clean["dq"][~rows])
        if which == "v":  # an infinity stays one in the column
            col = got["o"][rows][..., 3].float()
            assert torch.isnan(col).all() if bad != bad else (col == bad).all()
    for which in ("q", "do"):  # the keys that it does not see
        t = {"q": q.clone(), "do": do.clone()}
        t[which][at, :, 3] = bad
        got = _run(t["q"], k, v, t["do"], segs, **kw)
        assert torch.equal(got["dk"][~keys], clean["dk"][~keys]) and torch.equal(got["dv"][~keys], clean["dv"][~keys])


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ql,kl,window,sinks,causal,split", [([3], [9001], 3000, 64, False, "q"), ([2], [9000], 2500, 7, True, "q"),
                                                            ([4000], [4000], 300, 70, True, "k"), ([3000], [3000], 200, 5, False, "k")])
def test_not_finite_in_a_tile_in_parts(device, bad, dtype, ql, kl, window, sinks, causal, split):
    """Rows that do not see an element that is not finite keep their bits where a tile's work is split and joined too."""
    q, k, v, do, _ = _make(ql, kl, 4, 2, 64, dtype, device, 9)
    segs = AttentionSegments(ql, kl, device=device)
    assert segs._plan(split, 2, 2, causal, 64 * q.element_size(), q.element_size(), window, sinks).n_joins
    kw = dict(causal=causal, window=window, sinks=sinks)
    clean = _run(q, k, v, do, segs, **kw)
    nq, nk = ql[0], kl[0]
    see = _sees(nq, nk, causal, window, sinks, device)
    for at in (sinks - 1, nk - window // 2, nk - 1):
        rows = see[:, at]
        for which in ("v", "k"):
            t = {"k": k.clone(), "v": v.clone()}
            t[which][at, :, 3] = bad
            got = _run(q, t["k"], t["v"], do, segs, **kw)
            assert torch.equal(got["o"][~rows], clean["o"][~rows]) and torch.equal(got["dq"][~rows], clean["dq"][~rows])
            if which == "v":
                col = got["o"][rows][..., 3].float()
                assert torch.isnan(col).all() if bad != bad else (col == bad).all()
                assert torch.equal(got["o"][..., 4:], clean["o"][..., 4:])
    for at in (0, nq // 2, nq - 1):
        keys = see[at]
        for which in ("q", "do"):
            t = {"q": q.clone(), "do": do.clone()}
            t[which][at, :, 3] = bad
            got = _run(t["q"], k, v, t["do"], segs, **kw)
            assert torch.equal(got["dk"][~keys], clean["dk"][~keys]) and torch.equal(got["dv"][~keys], clean["dv"][~keys])


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_masked_keys_hold_does_not_matter(device, bad):
    ql = [290, 40]
    q, k, v, do, mask = _make(ql, ql, 4, 2, 64, torch.bfloat16, device, 7, masked=0.4)
    segs = AttentionSegments(ql, device=device)
    kw = dict(key_mask=mask, window=50, sinks=9, causal=True)
    clean = _run(q, k, v, do, segs, **kw)
    k[~mask], v[~mask] = bad, bad
    got = _run(q, k, v, do, segs, **kw)
    assert all(torch.equal(got[n], clean[n]) for n in got)


# ------------------------------------------------------------------ calls


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
def test_gradients_against_differences(device, causal):
    """Along random directions in fp32: central differences with e = 2^-6 (curvature e^2, rounding 2^-22 / e)."""
    ql, kl = [20, 9], [20, 30]
    q, k, v, do, mask = _make(ql, kl, 4, 2, 16, torch.float32, device, 12, masked=0.2)
    segs = AttentionSegments(ql, kl, device=device)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    f = lambda ts: (sparse_attention(*ts, segs, causal=causal, key_mask=mask, window=6, sinks=2).double()  # noqa: E731
                    * do.double()).sum()
    grads = torch.autograd.grad(f(leaves), leaves)
    e = 2.0 ** -6
    for i in range(3):
        d = torch.randn_like(leaves[i])
        with torch.no_grad():
            up, down = (f([t + s * e * d if j == i else t for j, t in enumerate(leaves)]) for s in (1, -1))
        slope, got = (up - down) / (2 * e), (grads[i].double() * d.double()).sum()
        assert (slope - got).abs() <= 1e-2 * (grads[i].double() * d.double()).norm(), (i, slope.item(), got.item())


@pytest.mark.gpu
def test_offsets_past_32_bits(device):
    """Sinks and a window more than 2^32 bytes apart: rows 16 KB apart."""
    n, dim = 400_000, 64
    cache = torch.empty((n, 128, dim), dtype=torch.bfloat16, device=device)
    g = torch.Generator(device=device).manual_seed(11)
    k, v = cache[:, 3:4], cache[:, 77:78]
    k.copy_(torch.randn((n, 1, dim), generator=g, device=device))
    v.copy_(torch.randn((n, 1, dim), generator=g, device=device))
    q = torch.randn((2, 4, dim), generator=g, device=device).to(torch.bfloat16)
    at = torch.cat((torch.arange(5), torch.arange(n - 1001, n))).to(device)
    got = sparse_attention(q, k, v, AttentionSegments([2], [n], device=device), causal=True, window=1000, sinks=5)
    see = _sees(2, n, True, 1000, 5)[:, at.cpu()].to(device)
    for h in range(4):
        s = (q[:, h].double() @ k[at, 0].double().T * dim ** -0.5).masked_fill(~see, float("-inf"))
        p = torch.softmax(s, 1)
        want = p @ v[at, 0].double()
        bound = (2.0 ** -8 + W) * (p @ v[at, 0].double().abs()) + 2.0 ** -8 * want.abs()
        assert ((got[:, h].double() - want).abs() <= bound).all()


@pytest.mark.gpu
def test_strides(device):
    n = 300
    segs = AttentionSegments([100, 200], device=device)
    g = torch.Generator().manual_seed(10)
    qkv = torch.randn((n, 3, 4, 32), generator=g).to(device, torch.bfloat16).requires_grad_(True)
    kw = dict(causal=True, window=17, sinks=2)
    o = sparse_attention(*qkv.unbind(1), segs, **kw)
    leaves = [t.detach().contiguous().requires_grad_(True) for t in qkv.unbind(1)]
    ref = sparse_attention(*leaves, segs, **kw)
    do = torch.randn(ref.shape, generator=g).to(device, torch.bfloat16)
    assert torch.equal(o, ref)
    o.backward(do)
    grads = torch.autograd.grad(ref, leaves, do)
    assert all(torch.equal(qkv.grad[:, i], d) for i, d in enumerate(grads))
    apart = [torch.empty((n, 4, 32, 2), dtype=torch.bfloat16, device=device)[..., 1].copy_(t.detach()) for t in leaves]
    assert torch.equal(sparse_attention(*apart, segs, **kw), ref)


@pytest.mark.gpu
def test_the_same_bits_on_every_run_and_stream(device):
    ql = [1000, 37, 600]
    q, k, v, do, mask = _make(ql, ql, 8, 2, 64, torch.bfloat16, device, 13, masked=0.1)
    segs = AttentionSegments(ql, device=device)
    kw = dict(key_mask=mask, window=100, sinks=4)
    first = _run(q, k, v, do, segs, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = _run(q, k, v, do, segs, **kw)
    torch.cuda.current_stream().wait_stream(side)
    for other in (second, _run(q, k, v, do, segs, **kw)):
        assert all(torch.equal(first[n], other[n]) for n in first)


@pytest.mark.gpu
def test_graph_capture_and_replay(device):
    ql, kl = [1, 1], [3000, 500]
    q, k, v, _, _ = _make(ql, kl, 8, 2, 64, torch.bfloat16, device, 15)
    segs = AttentionSegments(ql, kl, device=device)
    kw = dict(causal=True, window=1200, sinks=4)
    sparse_attention(q, k, v, segs, **kw)  # the tile lists are built by an eager call
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sparse_attention(q, k, v, segs, **kw)
    for _ in range(3):
        q.copy_(torch.randn(q.shape, device=device))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, sparse_attention(q, k, v, segs, **kw))


@pytest.mark.gpu
def test_refusals(device):
    segs = AttentionSegments([4, 2], device=device)
    q = torch.zeros((6, 4, 16), device=device)
    for window, sinks in ((0, 0), (-3, 0), (4, -1), (None, 2)):
        with pytest.raises(ValueError, match="window"):
            sparse_attention(q, q, q, segs, window=window, sinks=sinks)
    for window, sinks in ((1.5, 0), (4, 2.0), (True, 0), (4, True), ("4", 0)):
        with pytest.raises(TypeError):
            sparse_attention(q, q, q, segs, window=window, sinks=sinks)
    assert torch.equal(sparse_attention(q, q, q, segs, window=np.int64(2), sinks=torch.tensor(1)), q)
