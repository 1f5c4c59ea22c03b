"""sparse_qk_norm_rotary (st_qk_norm_rotary and its backward) against the formulas in float64.

Tolerances (f = 2^-24, and half a unit of the result's type for its rounding): the mean square is a sum of at most
256 squares, 2 V or fewer on a lane and six steps across them, so 1 / sqrt of it is within 20 f; with the products, the
cosine and sine 64 f of |a| + |b| of the normalised pair.  dx is the difference of two such terms, each
within 64 f of its own size.  dw adds n h terms, some hundred on a lane, then lanes, waves and workgroups: 512 f of
the sum of their sizes.
"""

import pytest
import torch

from sparsetriton_amd import SparseTensor, _lib
from sparsetriton_amd.nn.functional import RotaryAxes, sparse_qk_norm_rotary, sparse_rotary

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F = 2.0 ** -24


def _turn(x, pos, axes, sign=1.0):
    """(rotated, |a| + |b| at every channel) in float64."""
    x, size, p, pair = x.clone(), x.abs(), axes.pairs, 0
    size = size.clone()
    for a, dims in enumerate(axes.axes):
        for i in range(dims // 2):
            f = float(torch.tensor(axes.base ** (-2.0 * i / dims), dtype=torch.float64).float())
            t = pos[:, a].double().cpu()[:, None] * f
            u, v = (2 * pair, 2 * pair + 1) if axes.interleaved else (pair, pair + p)
            c, s = torch.cos(t), sign * torch.sin(t)
            xa, xb = x[:, :, u].clone(), x[:, :, v].clone()
            x[:, :, u], x[:, :, v] = xa * c - xb * s, xa * s + xb * c
            size[:, :, u] = size[:, :, v] = xa.abs() + xb.abs()
            pair += 1
    return x, size


def _formula(x, w, dy, pos, axes, eps):
    """{name: (value, bound)} of one tensor, in float64 on the host."""
    x, dy = x.detach().double().cpu(), dy.double().cpu()
    w = torch.ones(x.shape[2], dtype=torch.float64) if w is None else w.detach().double().cpu()
    s = 1 / torch.sqrt((x * x).mean(2, keepdim=True) + eps)
    y, size = _turn(x * s * w, pos, axes)
    g, gsize = _turn(dy, pos, axes, -1.0)
    along = (g * w * x).mean(2, keepdim=True)
    dx = s * (g * w - x * s * s * along)
    dsize = s * (gsize * w.abs() + x.abs() * s * s * (gsize * (w * x).abs()).mean(2, keepdim=True))
    terms, tsize = g * x * s, gsize * (x * s).abs()
    return {"y": (y, 64 * F * size), "dx": (dx, 64 * F * dsize),
            "dw": (terms.sum((0, 1)), 512 * F * tsize.sum((0, 1)))}


def _close(got, ref, bound, what):
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 1e-40
    off = (got.detach().double().cpu() - ref).abs() - (UNIT[got.dtype] * ref.abs() + bound + tiny)
    assert got.shape == ref.shape and got.is_contiguous() and not torch.isnan(got).any(), what
    assert off.numel() == 0 or off.max().item() <= 0, (what, off.max().item())


def _check(q, k, pos, axes, wq=None, wk=None, eps=1e-6):
    with torch.no_grad():
        plain = sparse_qk_norm_rotary(q, k, pos, axes, wq, wk, eps)
    leaves = [t.requires_grad_(True) for t in (q, k, wq, wk) if t is not None]
    out = sparse_qk_norm_rotary(q, k, pos, axes, wq, wk, eps)
    g = torch.Generator().manual_seed(99)
    dys = [None if t is None else torch.randn(t.shape, generator=g).to(t.device, t.dtype) for t in (q, k)]
    grads = dict(zip(map(id, leaves), torch.autograd.grad([o for o in out if o is not None], leaves,
                                                          [d for d in dys if d is not None])))
    for x, w, y, p, dy in zip((q, k), (wq, wk), out, plain, dys):
        assert (x is None) == (y is None)
        if x is None:
            continue
        assert torch.equal(p, y) and y.dtype == x.dtype
        ref = _formula(x, w, dy, pos, axes, eps)
        _close(y, *ref["y"], "y")
        assert grads[id(x)].dtype == x.dtype
        _close(grads[id(x)].contiguous(), *ref["dx"], "dx")
        if w is not None:
            assert grads[id(w)].dtype == w.dtype
            _close(grads[id(w)], *ref["dw"], "dw")
    return out, grads


def _make(n, heads, kv, dim, axes, dtype, device, seed, wdtype=None):
    g = torch.Generator().manual_seed(seed)
    spread = 0.2 + 3 * torch.rand((dim,), generator=g)
    q = (torch.randn((n, heads, dim), generator=g) * spread).to(device, dtype)
    k = (torch.randn((n, kv, dim), generator=g) * spread).to(device, dtype)
    wq, wk = ((1 + 0.3 * torch.randn((dim,), generator=g)).to(device, wdtype or dtype) for _ in range(2))
    pos = torch.randint(-1440, 1440, (n, len(axes)), generator=g).to(device, torch.int16)
    return q, k, wq, wk, pos


@pytest.mark.gpu
@pytest.mark.parametrize("dim,axes", [(2, (2,)), (8, (4, 4)), (16, (6, 6, 4)), (24, (10, 6, 8)), (32, (12, 12, 8)), (48, (16, 16, 8)),
                                      (64, (24, 24, 16)), (80, (80,)), (96, (32, 32, 32)), (128, (48, 48, 32)),
                                      (100, (2, 0, 4)), (36, (14,)), (7, (2, 2)), (16, (0, 0)), (1, (0,)), (256, (96, 96, 64)),
                                      (250, (50, 32)), (255, (2,)), (130, (64, 66))])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_heads(device, dim, axes, interleaved, dtype):
    q, k, wq, wk, pos = _make(53, 6, 2, dim, axes, dtype, device, dim)
    _check(q, k, pos, RotaryAxes(dim, axes, interleaved=interleaved), wq, wk)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,axes", [(8, (2,)), (8, (6,)), (16, (2, 4)), (16, (14,)), (24, (10,)), (24, (2, 2, 2)), (32, (2,)), (40, (36,)),
                                      (48, (22, 24)), (64, (10, 14, 6)), (64, (62,)), (64, (20, 20)), (80, (26,)), (96, (2, 30, 26)),
                                      (128, (42, 42, 42)), (128, (2,)), (256, (254,)), (256, (10, 20)), (256, (4,)), (68, (6, 20))])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_any_number_of_pairs(device, dim, axes, interleaved, dtype):
    """Pairs that no vector divides: partners with other lanes, and vectors half of which turn."""
    q, k, wq, wk, pos = _make(131, 5, 3, dim, axes, dtype, device, dim + len(axes))
    _check(q, k, pos, RotaryAxes(dim, axes, interleaved=interleaved), wq, wk)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 31, 1023, 1025, 20_011])
@pytest.mark.parametrize("pdtype", [torch.int16, torch.int32, torch.int64, torch.float32])
def test_rows_and_position_types(device, n, pdtype):
    axes = (12, 12, 8)
    q, k, wq, wk, _ = _make(n, 4, 4, 32, axes, torch.bfloat16, device, n)
    top = 1440 if pdtype != torch.int32 else 3_000_000
    pos = torch.randint(-top, top, (n, 3), generator=torch.Generator().manual_seed(n))
    pos = (pos + 0.25 if pdtype == torch.float32 else pos).to(device, pdtype)
    _check(q, k, pos, RotaryAxes(32, axes, base=500.0), wq, wk)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv", [(1, 1), (40, 8), (3, 7), (1, 129)])
def test_head_counts(device, heads, kv):
    q, k, wq, wk, pos = _make(300, heads, kv, 24, (8, 8, 8), torch.float32, device, heads)
    _check(q, k, pos, RotaryAxes(24, (8, 8, 8)), wq, wk)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16),
                                          (torch.float32, torch.float16)])
def test_weight_types(device, dtype, wdtype):
    axes = RotaryAxes(64, (24, 24, 16))
    q, k, wq, wk, pos = _make(70, 4, 2, 64, (24, 24, 16), dtype, device, 1, wdtype)
    _check(q, k, pos, axes, wq, wk)
    _check(q.detach(), k.detach(), pos, axes, None, wk.detach().to(dtype))
    _check(q.detach(), k.detach(), pos, axes, wq.detach().float(), None)
    _check(q.detach(), k.detach(), pos, axes)
    _check(q.detach(), k.detach(), pos, axes, wq.detach().float(), wk.detach().to(dtype))  # of two types


@pytest.mark.gpu
def test_one_of_the_two_and_what_needs_a_gradient(device):
    axes = RotaryAxes(32, (12, 12, 8))
    q, k, wq, wk, pos = _make(90, 4, 2, 32, (12, 12, 8), torch.float32, device, 2)
    _check(q, None, pos, axes, wq)
    _check(None, k, pos, axes, None, wk)
    q, k, wq, wk = (t.detach() for t in (q, k, wq, wk))
    full, grads = _check(q, k, pos, axes, wq, wk)
    want = [grads[id(t)] for t in (q, k, wq, wk)]
    g = torch.Generator().manual_seed(99)
    dys = [torch.randn(t.shape, generator=g).to(device) for t in (q, k)]
    for keep in range(1, 16):
        leaves = [t.detach().requires_grad_(bool(keep >> i & 1)) for i, t in enumerate((q, k, wq, wk))]
        out = sparse_qk_norm_rotary(leaves[0], leaves[1], pos, axes, *leaves[2:])
        loss = sum((o * d).sum() for o, d in zip(out, dys) if o.requires_grad)
        loss.backward()
        for i, (t, w) in enumerate(zip(leaves, want)):
            assert torch.equal(t.grad, w) if keep >> i & 1 else t.grad is None
    leaves = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
    out = sparse_qk_norm_rotary(leaves[0], leaves[1], pos, axes, *leaves[2:])
    got = torch.autograd.grad(out[1], leaves, dys[1], allow_unused=True)  # nothing arrives at q's output
    assert got[0] is None and torch.equal(got[1], want[1]) and not got[2].any() and torch.equal(got[3], want[3])


@pytest.mark.gpu
def test_strides(device):
    """q and k as slices of one projection, off a 16-byte address, channels apart, heads first; one head given to four."""
    axes = RotaryAxes(16, (6, 6, 4))
    n, g = 70, torch.Generator().manual_seed(3)
    qkv = torch.randn((n, 3, 4, 16), generator=g).to(device, torch.bfloat16)
    coords = torch.randint(0, 500, (n, 4), generator=g).to(device, torch.int16)
    wide = torch.randn((32,), generator=g).to(device, torch.bfloat16)
    w, wc = wide[::2], wide[::2].contiguous()
    q, k = qkv[:, 0], qkv[:, 1]
    ref = sparse_qk_norm_rotary(q.contiguous(), k.contiguous(), coords[:, 1:].contiguous(), axes, wc, wc)
    x = SparseTensor(qkv.view(n, -1), coords, spatial_shape=(500, 500, 500))
    for pos in (coords[:, 1:], x):
        assert all(torch.equal(a, b) for a, b in zip(ref, sparse_qk_norm_rotary(q, k, pos, axes, w, w)))
    off = torch.empty((n * 64 + 1,), dtype=torch.bfloat16, device=device)[1:].view(n, 4, 16).copy_(q)
    half = torch.empty((n * 64 + 4,), dtype=torch.bfloat16, device=device)[4:].view(n, 4, 16).copy_(q)
    apart = torch.empty((n, 4, 16, 2), dtype=torch.bfloat16, device=device)[..., 0].copy_(q)
    heads_first = torch.empty((4, n, 16), dtype=torch.bfloat16, device=device).transpose(0, 1).copy_(q)
    f32 = sparse_qk_norm_rotary(q.float(), None, x, axes, w)[0]
    for t in (off, half, apart, heads_first):
        got = sparse_qk_norm_rotary(t, None, x, axes, w)[0]
        assert (got.float() - f32).abs().max().item() <= (2.0 ** -8 + 64 * F) * f32.abs().max().item()
        _check(t.detach(), k, coords[:, 1:], axes, wc.detach().clone(), wc.detach().clone())
    one = q[:, :1].expand(n, 4, 16)
    _check(one.detach(), k, coords[:, 1:], axes, wc.detach().clone())
    dy = torch.randn((n, 16, 4), device=device, dtype=torch.bfloat16).transpose(1, 2)  # the gradient's channels apart
    leaf = q.detach().clone().requires_grad_(True)
    y = sparse_qk_norm_rotary(leaf, None, x, axes, w)[0]
    a, = torch.autograd.grad(y, leaf, dy, retain_graph=True)
    b, = torch.autograd.grad(y, leaf, dy.contiguous())
    assert torch.equal(a, b)


@pytest.mark.gpu
def test_rows_past_the_reach_of_32_bit_offsets(device):
    """Rows and heads at any stride: heads first, with more than 2^31 bytes from a row's first head to its last, in
    the inputs and in the gradients at the outputs; one such row; a single row whose stride is past 2^31."""
    heads, n, dim, axes = 3, (1 << 20) * 3 + 5, 128, RotaryAxes(128, (48, 48, 32))
    g = torch.Generator(device=device).manual_seed(14)
    make = lambda: torch.randn((heads, n, dim), generator=g, device=device, dtype=torch.bfloat16).transpose(0, 1)  # noqa: E731
    q, dy = make(), make()
    assert q.stride(1) * q.element_size() * heads > 2 ** 31
    pos = torch.randint(-1440, 1440, (n, 3), generator=g, device=device)
    w = (1 + 0.1 * torch.randn((dim,), generator=g, device=device)).bfloat16()

    def step(x, d, p):
        x, wq = (t.detach().requires_grad_(True) for t in (x, w))
        y = sparse_qk_norm_rotary(x, None, p, axes, wq)[0]
        return (y.detach(),) + torch.autograd.grad(y, (x, wq), d)

    want = step(q.contiguous(), dy.contiguous(), pos)
    for a, b in ((q, dy), (q.contiguous(), dy), (q, dy.contiguous())):
        assert all(torch.equal(x, y) for x, y in zip(step(a, b, pos), want))
    _, none = sparse_qk_norm_rotary(q[:7], None, pos[:7], axes, w)
    assert none is None
    for rows in (slice(0, 7), slice(n - 1, n)):
        y, none = sparse_qk_norm_rotary(None, q[rows], pos[rows], axes, None, w)[::-1]
        assert none is None and torch.equal(y, want[0][rows])
    one = q[5:6].contiguous()
    far = torch.as_strided(one, one.shape, (2 ** 33, dim, 1))
    got = step(far, torch.as_strided(one, one.shape, (2 ** 33, dim, 1)), pos[5:6])
    assert all(torch.equal(x, y) for x, y in zip(got, step(one, one, pos[5:6])))


@pytest.mark.gpu
def test_gradients_against_differences(device):
    """fp32 with large steps: (f(x + h) - f(x - h)) / 2h of a smooth function, off by h^2 / 6 of its third derivative (of
    the size of its first here) and 2^-22 of f / h."""
    axes = RotaryAxes(24, (8, 8, 4))
    q, k, wq, wk, pos = (t.double().cpu() for t in _make(5, 2, 1, 24, (8, 8, 4), torch.float32, device, 4))
    pos = pos.to(device, torch.int16)
    leaves = [t.float().to(device).requires_grad_(True) for t in (q, k, wq, wk)]
    g = torch.Generator().manual_seed(5)
    dys = [torch.randn(t.shape, generator=g).to(device) for t in leaves[:2]]

    def f(ts):
        return sum((o * d).sum(dtype=torch.float64) for o, d in zip(sparse_qk_norm_rotary(ts[0], ts[1], pos, axes, *ts[2:]), dys))

    grads = torch.autograd.grad(f(leaves), leaves)
    h = 2.0 ** -7
    for i, t in enumerate(leaves):
        along = torch.randn(t.shape, generator=g).to(device)
        up, down = ([(u + s * h * along if j == i else u).detach() for j, u in enumerate(leaves)] for s in (1, -1))
        want = (f(up) - f(down)).item() / (2 * h)
        got = (grads[i] * along).sum(dtype=torch.float64).item()
        assert abs(got - want) <= 2e-3 * grads[i].double().norm().item() * along.double().norm().item()


@pytest.mark.gpu
def test_small_large_and_empty_heads(device):
    axes = RotaryAxes(32, (12, 12, 8))
    q, k, wq, wk, pos = _make(40, 4, 2, 32, (12, 12, 8), torch.float32, device, 6)
    for scale in (1e-6, 1e-3, 1e3, 1e15):
        _check(q.detach() * scale, k.detach() * scale, pos, axes, wq.detach(), wk.detach())
    zero = q.detach().clone()
    zero[3] = 0
    out, grads = _check(zero, k.detach(), pos, axes, wq.detach(), wk.detach())
    assert not out[0][3].any()
    _check(q.detach(), k.detach(), pos, axes, wq.detach(), wk.detach(), eps=0.0)
    half = (q.detach() * 2000).half()
    _check(half, None, pos, axes, wq.detach().half())  # squares past float16's range
    w = wq.detach().requires_grad_(True)
    e = q.detach()[:0].requires_grad_(True)
    y, none = sparse_qk_norm_rotary(e, None, pos[:0], axes, w)
    de, dw = torch.autograd.grad(y.sum(), (e, w))
    assert y.shape == (0, 4, 32) and none is None and de.shape == e.shape and not dw.any()


@pytest.mark.gpu
def test_not_finite_stays_in_its_head(device):
    axes = RotaryAxes(16, (6, 6, 4))
    q, _, wq, _, pos = _make(30, 3, 1, 16, (6, 6, 4), torch.float32, device, 7)
    dy = torch.randn_like(q)
    leaf = q.clone().requires_grad_(True)
    clean = sparse_qk_norm_rotary(leaf, None, pos, axes, wq)[0]
    dclean, = torch.autograd.grad(clean, leaf, dy)
    for bad in (float("nan"), float("inf")):
        leaf = q.clone()
        leaf[2, 1, 5] = bad
        leaf.requires_grad_(True)
        got = sparse_qk_norm_rotary(leaf, None, pos, axes, wq)[0]
        d, = torch.autograd.grad(got, leaf, dy)
        keep = torch.ones((30, 3), dtype=torch.bool, device=device)
        keep[2, 1] = False
        assert torch.equal(got[keep], clean[keep]) and torch.equal(d[keep], dclean[keep])
        assert torch.isnan(got[2, 1]).any() and torch.isnan(d[2, 1]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dim,axes,dtype", [(16, (6, 6), torch.float32), (16, (4, 4), torch.float32), (15, (2, 4), torch.float32),
                                            (18, (4, 4), torch.float32), (16, (6, 6), torch.bfloat16), (48, (16, 16), torch.bfloat16),
                                            (20, (10,), torch.float16), (256, (90, 102), torch.float32), (255, (2, 4), torch.bfloat16)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_not_finite_stays_in_its_pair(device, dim, axes, dtype, interleaved, bad):
    """Channels past the pairs turn by nothing: what is not finite in one channel of a weight, an input or a gradient
    reaches the channel that turns with it and what the head's sums make of it, nothing else."""
    n, axes = 37, RotaryAxes(dim, axes, interleaved=interleaved)
    q, _, wq, _, pos = _make(n, 3, 1, dim, axes.axes, dtype, device, dim + interleaved)
    dy = torch.randn((n, 3, dim), generator=torch.Generator().manual_seed(dim)).to(device, dtype)

    def step(x, w, d):
        x, w = (t.clone().requires_grad_(True) for t in (x, w))
        y = sparse_qk_norm_rotary(x, None, pos, axes, w)[0]
        return (y.detach(),) + torch.autograd.grad(y, (x, w), d)

    clean = step(q, wq, dy)
    p = axes.pairs
    for c in sorted({0, 2 * p - 1, 2 * p, 2 * p + 1, dim - 2, dim - 1}):
        partner = c if c >= 2 * p else c ^ 1 if interleaved else (c + p) % (2 * p)
        others = torch.tensor([i for i in range(dim) if i not in (c, partner)], device=device)
        w = wq.clone()
        w[c] = bad
        y = step(q, w, dy)[0]
        assert torch.equal(y[..., others], clean[0][..., others]) and not torch.isfinite(y[..., c]).any(), c
        x = q.clone()
        x[2, 1, c] = bad
        y = step(x, wq, dy)[0]
        assert torch.isnan(y[2, 1, c])
        assert torch.isnan(y[2, 1]).all() if bad != bad else not y[2, 1, others].any(), c  # (divided by an infinity)
        keep = torch.ones((n, 3), dtype=torch.bool, device=device)
        keep[2, 1] = False
        assert torch.equal(y[keep], clean[0][keep])
        d = dy.clone()
        d[2, 1, [c, partner]] = 0
        zero = step(q, wq, d)
        d[2, 1, c] = bad
        _, dx, dw = step(q, wq, d)
        assert torch.equal(dw[others], zero[2][others]) and not torch.isfinite(dw[c]), c
        assert torch.equal(dx[keep], clean[1][keep])


@pytest.mark.gpu
def test_same_as_the_rotation_of_normalised_heads(device):
    """Heads whose mean square is one already, no weight and eps = 0: sparse_rotary, to a few roundings."""
    axes = RotaryAxes(64, (24, 24, 16))
    q, k, _, _, pos = _make(500, 8, 2, 64, (24, 24, 16), torch.float32, device, 8)
    q, k = (t / t.square().mean(2, keepdim=True).sqrt() for t in (q, k))
    for a, b in zip(sparse_qk_norm_rotary(q, k, pos, axes, eps=0.0), sparse_rotary(q, k, pos, axes)):
        assert (a - b).abs().max().item() <= 128 * F * b.abs().max().item()


@pytest.mark.gpu
def test_repeats_and_graph(device, own_random):
    """The same bits at every call, on another stream, and at every replay of a captured step."""
    axes = RotaryAxes(64, (24, 24, 16))
    q, k, wq, wk, pos = _make(4001, 8, 2, 64, (24, 24, 16), torch.bfloat16, device, 9)
    dys = [torch.randn_like(t) for t in (q, k)]

    def step():  # (leaves of its own: a captured backward must not meet those of an eager graph that lives)
        leaves = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
        out = sparse_qk_norm_rotary(leaves[0], leaves[1], pos, axes, *leaves[2:])
        return [o.detach() for o in out] + list(torch.autograd.grad(out, leaves, dys))

    want = step()
    assert all(torch.equal(a, b) for a, b in zip(want, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    del other
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        q.mul_(1.5)
        pos.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step(), got))


@pytest.mark.gpu
def test_more_workgroups_than_one_launch_takes(device):
    """A grid has fewer than 2^32 threads: 2^24 workgroups, each of one row where its heads have odd sizes."""
    n, small, axes = (1 << 24) + 3, 4099, RotaryAxes(53, (2, 4))
    q, k, wq, wk, pos = _make(small, 5, 2, 53, (2, 4), torch.bfloat16, device, 13)
    want = sparse_qk_norm_rotary(q, k, pos, axes, wq, wk)
    got = sparse_qk_norm_rotary(*[t.repeat(-(-n // small), *[1] * (t.dim() - 1))[:n] for t in (q, k, pos)], axes, wq, wk)
    for at in range(0, n, 1 << 20):
        rows = torch.arange(at, min(n, at + (1 << 20)), device=device) % small
        assert all(torch.equal(a[at:at + (1 << 20)], b[rows]) for a, b in zip(got, want))


@pytest.mark.gpu
def test_a_second_launch_begins_where_the_first_ends(device):
    """A grid has fewer than 2^32 threads: 2^24 - 1 workgroups.  9 heads of 64 lanes (35 channels with one pair: 34 of a
    channel or a pair) are more than half of the 1,024 lanes' worth that a workgroup takes, so each has one row."""
    n, small, axes = (1 << 24) + 3, 4099, RotaryAxes(35, (2,))
    q, k, wq, wk, pos = _make(small, 6, 3, 35, (2,), torch.bfloat16, device, 15)
    assert (6 + 3) * 64 * 2 > 1024
    want = sparse_qk_norm_rotary(q, k, pos, axes, wq, wk)
    got = sparse_qk_norm_rotary(*[t.repeat(-(-n // small), *[1] * (t.dim() - 1))[:n] for t in (q, k, pos)], axes, wq, wk)
    for at in list(range(0, n, 1 << 20)) + [n - 100]:
        rows = torch.arange(at, min(n, at + (1 << 20)), device=device) % small
        assert all(torch.equal(a[at:at + (1 << 20)], b[rows]) for a, b in zip(got, want))


def test_refusals_before_any_launch():
    with pytest.raises(ValueError, match="needs"):
        sparse_qk_norm_rotary(None, None, torch.zeros((1, 1)), RotaryAxes(16, (8,)))
    with pytest.raises(RuntimeError, match="GPU"):
        sparse_qk_norm_rotary(torch.zeros((1, 1, 16)), None, torch.zeros((1, 1)), RotaryAxes(16, (8,)))
    lib, args = _lib.lib(), _lib.QkNormArgs()
    for f in (lib.st_qk_norm_rotary, lib.st_qk_norm_rotary_backward):
        assert f(None, None) == -1
        args.n, args.dim, args.pairs, args.eps = 4, 16, 9, 0.0
        assert f(args, None) == -1  # more pairs than the head has
        args.pairs, args.eps = 4, -1.0
        assert f(args, None) == -1
        args.eps, args.dim = 0.0, 257
        assert f(args, None) == -3
        args.dim, args.dtype = 16, 7
        assert f(args, None) == -3
        args.dtype = 0
        assert f(args, None) == -1  # neither q nor k
        args.n = 0
        assert f(args, None) == 0


@pytest.mark.gpu
def test_refusals(device):
    axes = RotaryAxes(16, (8, 4))
    q, pos = torch.zeros((5, 2, 16), device=device), torch.zeros((5, 2), device=device, dtype=torch.int32)
    w = torch.ones((16,), device=device)
    for bad in (q[:, :, :8], q[0], q[:, :0]):
        with pytest.raises(ValueError, match="expected"):
            sparse_qk_norm_rotary(bad, None, pos, axes)
    for k in (q[:4], q.half()):
        with pytest.raises(ValueError, match="same"):
            sparse_qk_norm_rotary(q, k, pos, axes)
    for p in (pos[:4], pos[:, :1], pos[0]):
        with pytest.raises(ValueError, match="positions"):
            sparse_qk_norm_rotary(q, None, p, axes)
    for bad in (w[:8], w.cpu(), w[None]):
        with pytest.raises(ValueError, match="q_weight"):
            sparse_qk_norm_rotary(q, None, pos, axes, bad)
        with pytest.raises(ValueError, match="k_weight"):
            sparse_qk_norm_rotary(q, q, pos, axes, w, bad)
    with pytest.raises(ValueError, match="without"):
        sparse_qk_norm_rotary(q, None, pos, axes, w, w)
    for eps in (-1e-6, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            sparse_qk_norm_rotary(q, None, pos, axes, w, eps=eps)
    with pytest.raises(ValueError, match="at most 256"):
        sparse_qk_norm_rotary(torch.zeros((5, 1, 264), device=device), None, pos, RotaryAxes(264, (8, 4)))
    with pytest.raises(ValueError, match="32,767"):
        sparse_qk_norm_rotary(torch.zeros((5, 1 << 15, 16), device=device), None, pos, axes)
    with pytest.raises(TypeError, match="feature dtype"):
        sparse_qk_norm_rotary(q, None, pos, axes, w.double())
    with torch.autograd.forward_ad.dual_level():
        for which in range(3):
            ts = [q, q.clone(), w]
            ts[which] = torch.autograd.forward_ad.make_dual(ts[which], torch.ones_like(ts[which]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                sparse_qk_norm_rotary(ts[0], ts[1], pos, axes, ts[2])
