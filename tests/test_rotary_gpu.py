"""sparse_rotary (st_rotary) against the rotation in float64.

Tolerances: one rounding to the result's type plus a cosine, a sine and two products in fp32:
8 * 2^-24 of |a| + |b|.  The angle's own error (64-bit turns, one rounding to fp32 of a value
below half a turn) is 2^-24 * pi, in the same bound.
"""

import math

import pytest
import torch

from sparsetriton_amd import SparseTensor, _lib
from sparsetriton_amd.nn.functional import RotaryAxes, sparse_rotary

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _formula(x, pos, axes, sign=1.0):
    """(rotated, |a| + |b| at every channel) in float64."""
    x = x.detach().double().cpu().clone()
    size = x.abs().clone()
    p, pair = axes.pairs, 0
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


def _close(got, ref, size):
    off = (got.double().cpu() - ref).abs() - (UNIT[got.dtype] * ref.abs() + 16 * 2.0 ** -24 * size)
    assert got.shape == ref.shape and off.max().item() <= 0, off.max().item()


def _check(q, k, pos, axes):
    leaves = [t for t in (q, k) if t is not None]
    out = sparse_rotary(q, k, pos, axes)
    assert (out[0] is None) == (q is None) and (out[1] is None) == (k is None)
    gs = [torch.randn(t.shape, device=t.device).to(t.dtype) for t in leaves]
    leaves = [t.requires_grad_(True) for t in leaves]
    tracked = [t for t in sparse_rotary(q, k, pos, axes) if t is not None]
    grads = torch.autograd.grad(tracked, leaves, gs)
    for t, plain, y, g, d in zip(leaves, [o for o in out if o is not None], tracked, gs, grads):
        assert torch.equal(plain, y) and y.is_contiguous() and y.dtype == t.dtype
        _close(y.detach(), *_formula(t, pos, axes))
        _close(d, *_formula(g, pos, axes, -1.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dim,axes", [(2, (2,)), (16, (6, 6, 4)), (24, (10, 6, 8)), (32, (12, 12, 8)), (48, (16, 16, 8)),
                                      (64, (24, 24, 16)), (80, (80,)), (128, (48, 48, 32)), (100, (2, 0, 4)), (36, (14,)),
                                      (7, (2, 2)), (16, (0, 0))])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_heads(device, dim, axes, interleaved, dtype):
    g = torch.Generator().manual_seed(dim)
    n, heads, kv = 53, 6, 2
    q = torch.randn((n, heads, dim), generator=g).to(device, dtype)
    k = torch.randn((n, kv, dim), generator=g).to(device, dtype)
    pos = torch.randint(-1440, 1440, (n, len(axes)), generator=g).to(device, torch.int16)
    _check(q, k, pos, RotaryAxes(dim, axes, interleaved=interleaved))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 1023, 20_011])
@pytest.mark.parametrize("pdtype", [torch.int16, torch.int32, torch.int64, torch.float32])
def test_rows_and_position_types(device, n, pdtype):
    g = torch.Generator().manual_seed(n)
    q = torch.randn((n, 4, 32), generator=g).to(device, torch.bfloat16)
    top = 1440 if pdtype != torch.int32 else 3_000_000
    pos = torch.randint(-top, top, (n, 3), generator=g)
    pos = (pos + 0.25 if pdtype == torch.float32 else pos).to(device, pdtype)
    _check(q, q.clone(), pos, RotaryAxes(32, (12, 12, 8), base=500.0))


@pytest.mark.gpu
def test_one_of_the_two(device):
    q = torch.randn((30, 4, 32), device=device)
    pos = torch.randint(0, 100, (30, 3), device=device)
    axes = RotaryAxes(32, (12, 12, 8))
    _check(q, None, pos, axes)
    _check(None, q.detach(), pos, axes)


@pytest.mark.gpu
def test_strides(device):
    """q and k as slices of one projection, off a 16-byte address, channels apart; positions as columns of the coordinates."""
    axes = RotaryAxes(16, (6, 6, 4))
    n, g = 70, torch.Generator().manual_seed(3)
    qkv = torch.randn((n, 3, 4, 16), generator=g).to(device, torch.bfloat16)
    coords = torch.randint(0, 500, (n, 4), generator=g).to(device, torch.int16)
    q, k = qkv[:, 0], qkv[:, 1]
    ref = sparse_rotary(q.contiguous(), k.contiguous(), coords[:, 1:].contiguous(), axes)
    got = sparse_rotary(q, k, coords[:, 1:], axes)
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    x = SparseTensor(qkv.view(n, -1), coords, spatial_shape=(500, 500, 500))
    assert all(torch.equal(a, b) for a, b in zip(ref, sparse_rotary(q, k, x, axes)))
    off = torch.empty((n * 64 + 1,), dtype=torch.bfloat16, device=device)[1:].view(n, 4, 16).copy_(q)
    apart = torch.empty((n, 4, 16, 2), dtype=torch.bfloat16, device=device)[..., 0].copy_(k)
    heads_first = torch.empty((4, n, 16), dtype=torch.bfloat16, device=device).transpose(0, 1).copy_(q)
    for t, r in ((off, ref[0]), (heads_first, ref[0]), (apart, ref[1])):
        assert torch.equal(sparse_rotary(t, None, coords[:, 1:], axes)[0], r)
    one = q[:, :1].expand(n, 4, 16)  # one head given to four: the gradient adds over them
    _check(one.detach(), k, coords[:, 1:], axes)


@pytest.mark.gpu
def test_turning_back_and_lengths(device):
    q = torch.randn((100, 8, 64), device=device)
    pos = torch.randint(-30000, 30000, (100, 3), device=device).short()
    axes = RotaryAxes(64, (24, 24, 16))
    there, _ = sparse_rotary(q, None, pos, axes)
    back, _ = sparse_rotary(there, None, -pos.int(), axes)
    assert (back - q).abs().max().item() < 1e-5
    assert (there.norm(dim=2) / q.norm(dim=2) - 1).abs().max().item() < 1e-6


@pytest.mark.gpu
def test_empty_and_not_finite(device):
    axes = RotaryAxes(16, (6, 6, 4))
    out = sparse_rotary(torch.zeros((0, 2, 16), device=device), None, torch.zeros((0, 3), device=device), axes)
    assert out[0].shape == (0, 2, 16)
    q = torch.randn((6, 2, 16), device=device)
    pos = torch.randint(0, 9, (6, 3), device=device)
    clean = sparse_rotary(q, None, pos, axes)[0]
    q[2, 1, 5] = float("nan")
    got = sparse_rotary(q, None, pos, axes)[0]
    bad = torch.isnan(got)
    assert bad.nonzero().tolist() == [[2, 1, 5], [2, 1, 13]] and torch.equal(got[~bad], clean[~bad])


def test_refusals_before_any_launch():
    with pytest.raises(ValueError, match="even"):
        RotaryAxes(16, (3, 4))
    with pytest.raises(ValueError, match="turn"):
        RotaryAxes(16, (12, 6))
    with pytest.raises(ValueError, match="base"):
        RotaryAxes(16, (8,), base=0)
    with pytest.raises(ValueError, match="needs"):
        sparse_rotary(None, None, torch.zeros((1, 1)), RotaryAxes(16, (8,)))
    with pytest.raises(RuntimeError, match="GPU"):
        sparse_rotary(torch.zeros((1, 1, 16)), None, torch.zeros((1, 1)), RotaryAxes(16, (8,)))
    axes = RotaryAxes(16, (8, 4))
    assert axes.pairs == 6 and axes.frequencies.tolist() == pytest.approx(
        [1, 10000 ** -0.25, 10000 ** -0.5, 10000 ** -0.75, 1, 10000 ** -0.5])
    args = _lib.RotaryArgs()
    assert _lib.lib().st_rotary(None, None) == -1
    args.n, args.dim, args.pairs = 4, 16, 9
    assert _lib.lib().st_rotary(args, None) == -1  # more pairs than the head has


@pytest.mark.gpu
def test_refusals(device):
    axes = RotaryAxes(16, (8, 4))
    q, pos = torch.zeros((5, 2, 16), device=device), torch.zeros((5, 2), device=device, dtype=torch.int32)
    for bad in (q[:, :, :8], q[0], q[:, :0]):
        with pytest.raises(ValueError, match="expected"):
            sparse_rotary(bad, None, pos, axes)
    for k in (q[:4], q.half()):
        with pytest.raises(ValueError, match="same"):
            sparse_rotary(q, k, pos, axes)
    for p in (pos[:4], pos[:, :1], pos[0]):
        with pytest.raises(ValueError, match="positions"):
            sparse_rotary(q, None, p, axes)
    with pytest.raises(ValueError, match="positions are on"):
        sparse_rotary(q, None, pos.cpu(), axes)
    with pytest.raises(TypeError, match="position dtype"):
        sparse_rotary(q, None, pos.double(), axes)
    with pytest.raises(TypeError, match="feature dtype"):
        sparse_rotary(q.double(), None, pos, axes)
    assert math.isclose(RotaryAxes(16, (8,)).frequencies[1].item(), 10000 ** -0.25, rel_tol=1e-7)


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(2))
@pytest.mark.parametrize("recorded", [False, True])
def test_forward_mode_is_refused(device, own_random, which, recorded):
    """No forward-mode derivative: a tangent on q or k raises, where it is not to be dropped, with or without a graph."""
    t = [torch.randn((5, 2, 16), device=device, requires_grad=recorded) for _ in range(2)]
    pos, axes = torch.zeros((5, 2), dtype=torch.int32, device=device), RotaryAxes(16, (8, 4))
    with torch.autograd.forward_ad.dual_level():
        sparse_rotary(*t, pos, axes)
        t[which] = torch.autograd.forward_ad.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            sparse_rotary(*t, pos, axes)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            sparse_rotary(*t, pos, axes)


@pytest.mark.gpu
def test_tables_outlive_their_owner_on_another_stream(device, own_random):
    """The frequencies' memory, made on one stream, is not handed out again while another stream's kernel may read it."""
    q, pos = torch.randn((4000, 4, 32), device=device), torch.randint(0, 500, (4000, 3), device=device)
    want = sparse_rotary(q, None, pos, RotaryAxes(32, (12, 12, 8)))[0]
    axes, busy = RotaryAxes(32, (12, 12, 8)), torch.randn((4096, 4096), device=device)
    sparse_rotary(q, None, pos, axes)
    held = [t.data_ptr() for t in axes.on(q.device)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):  # (some milliseconds for the call below to wait behind)
            other = busy @ busy
        got = sparse_rotary(q, None, pos, axes)[0]
    sizes = [(t.numel(), t.dtype) for t in axes.on(q.device)]
    del axes
    new = [torch.empty((n,), dtype=d, device=device) for n, d in sizes for _ in range(4)]
    done = side.query()
    torch.cuda.current_stream().wait_stream(side)
    other.record_stream(torch.cuda.current_stream())
    got.record_stream(torch.cuda.current_stream())
    assert torch.equal(got, want)
    assert done or not set(held) & {t.data_ptr() for t in new}


@pytest.mark.gpu
def test_more_workgroups_than_one_launch_takes(device):
    """A grid has fewer than 2^32 threads: 2^24 workgroups, each of one row where its heads have odd sizes."""
    n, small, axes = (1 << 24) + 3, 4099, RotaryAxes(53, (2, 4))
    g = torch.Generator().manual_seed(13)
    q = torch.randn((small, 9, 53), generator=g).to(device, torch.bfloat16)
    k = torch.randn((small, 2, 53), generator=g).to(device, torch.bfloat16)
    pos = torch.randint(-500, 500, (small, 2), generator=g).to(device, torch.int16)
    want = sparse_rotary(q, k, pos, axes)
    got = sparse_rotary(*[t.repeat(-(-n // small), *[1] * (t.dim() - 1))[:n] for t in (q, k, pos)], axes)
    for at in range(0, n, 1 << 20):
        rows = torch.arange(at, min(n, at + (1 << 20)), device=device) % small
        assert all(torch.equal(a[at:at + (1 << 20)], b[rows]) for a, b in zip(got, want))
