"""sparse_layer_norm (st_ln_forward / st_ln_backward) against the formula in float64.

Tolerances: one rounding to the result's type (half a unit: 2^-24, 2^-11, 2^-8 relative) plus fp32
arithmetic on the way: a normalised value carries a few fp32 roundings of the largest |h| of its
row, scaled by 1 / std; a row gradient a few of the largest |dy w|, scaled alike; a column sum
adds its terms' errors (a few 2^-24 each, chains of at most some hundred) to theirs.
"""

import pytest
import torch

from sparsetriton_amd import SparseTensor, _lib
from sparsetriton_amd.nn.functional import sparse_layer_norm

pytestmark = pytest.mark.gpu
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F32 = 2.0 ** -24
EPS = 1e-5


def _formula(h, w, b, dy, dh):
    h, dy = h.double(), dy.double()
    w = torch.ones(h.shape[1], dtype=torch.float64, device=h.device) if w is None else w.double()
    mu = h.mean(1, keepdim=True)
    rs = 1 / torch.sqrt(((h - mu) ** 2).mean(1, keepdim=True) + EPS)
    xh = (h - mu) * rs
    y = xh * w + (0 if b is None else b.double())
    g = dy * w
    dx = rs * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    if dh is not None:
        dx = dx + dh.double()
    return y, dx, (dy * xh).sum(0), dy.sum(0), rs, xh, g


def _close(got, ref, bound, what):
    assert got.shape == ref.shape, what
    off = (got.double() - ref).abs() - (UNIT[got.dtype] * ref.abs() + bound)
    assert not torch.isnan(got).any() and off.max().item() <= 0, (what, off.max().item())


def _check(x, w, b, res, dy, dh):
    leaves = [t.requires_grad_(True) for t in (x, w, b, res) if t is not None]
    out = sparse_layer_norm(x, w, b, eps=EPS, residual=res)
    y, h = out if res is not None else (out, x)
    if res is not None:
        assert torch.equal(h, (x.detach().float() + res.detach().float()).to(x.dtype))
    grads = dict(zip(map(id, leaves), torch.autograd.grad([y] + ([h] if res is not None else []), leaves,
                                                          [dy] + ([dh] if res is not None else []))))
    ry, rdx, rdw, rdb, rs, xh, g = _formula(h.detach(), w, b, dy, dh)
    wmax = 1.0 if w is None else w.detach().abs().max().item()
    top = h.detach().double().abs().amax(1, keepdim=True)
    _close(y.detach(), ry, 16 * F32 * (top * rs * wmax + (0 if b is None else b.detach().abs().max().item())), "y")
    slack = 32 * F32 * rs * g.abs().amax(1, keepdim=True) * (1 + xh.abs().amax(1, keepdim=True)) * \
        (1 + top * rs)
    _close(grads[id(x)], rdx, slack + 4 * F32 * rdx.abs(), "dx")
    if res is not None:
        assert torch.equal(grads[id(res)], grads[id(x)])
    if w is not None:
        terms = dy.double().abs() * (xh.abs() + 16 * top * rs)
        _close(grads[id(w)], rdw, 64 * F32 * terms.sum(0), "dw")
    if b is not None:
        _close(grads[id(b)], rdb, 64 * F32 * dy.double().abs().sum(0), "db")
    # without a gradient to compute the same output
    with torch.no_grad():
        again = sparse_layer_norm(x, w, b, eps=EPS, residual=res)
    assert torch.equal(again if res is None else again[0], y)


def _make(n, C, dtype, wdtype, residual, affine, seed, device):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((n, C), generator=g) + 0.5).to(device, dtype)
    res = torch.randn((n, C), generator=g).to(device, dtype) if residual else None
    w = (1 + 0.3 * torch.randn((C,), generator=g)).to(device, wdtype) if affine else None
    b = (0.3 * torch.randn((C,), generator=g)).to(device, wdtype) if affine else None
    dy = torch.randn((n, C), generator=g).to(device, dtype)
    dh = torch.randn((n, C), generator=g).to(device, dtype) if residual else None
    return x, w, b, res, dy, dh


# channels: one lane pair to whole workgroups a row, vector and element forms, and rows past the registers
@pytest.mark.parametrize("C", [1, 2, 7, 8, 16, 40, 64, 100, 129, 512, 520, 1000, 1001, 2048, 4096, 4100, 8200, 4099])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_widths(device, C, dtype):
    _check(*_make(37, C, dtype, dtype, C % 2 == 0, True, C, device))


@pytest.mark.parametrize("n,C", [(1, 64), (3, 512), (20_001, 64), (5003, 256), (9001, 24), (2100, 2048)])
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                          (torch.float16, torch.float16)])
@pytest.mark.parametrize("residual", [False, True])
def test_rows(device, n, C, dtype, wdtype, residual):
    _check(*_make(n, C, dtype, wdtype, residual, True, n + C, device))


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
def test_affine_parts(device, weight, bias):
    x, w, b, res, dy, dh = _make(50, 96, torch.bfloat16, torch.bfloat16, True, True, 5, device)
    _check(x, w if weight else None, b if bias else None, res, dy, dh)


def test_parameter_dtypes_that_differ(device):
    x, w, b, _, dy, _ = _make(33, 64, torch.bfloat16, torch.float32, False, True, 6, device)
    _check(x, w, b.to(torch.bfloat16), None, dy, None)
    x, w, b, _, dy, _ = _make(33, 64, torch.float32, torch.float16, False, True, 7, device)
    _check(x, w, b, None, dy, None)


def test_strides_and_offsets(device):
    """Rows out of a wider tensor, transposed storage, storage that starts off a 16-byte address."""
    g = torch.Generator().manual_seed(8)
    wide = torch.randn((40, 200), generator=g).to(device, torch.bfloat16)
    w, b = torch.ones(64, device=device), torch.zeros(64, device=device)
    off = torch.randn((40 * 64 + 3,), generator=g).to(device, torch.bfloat16)[3:].view(40, 64)
    assert off.data_ptr() % 16
    for x in (wide[:, 5:69], torch.randn((64, 40), generator=g).to(device, torch.bfloat16).t(), off):
        dy = torch.randn((40, 64), generator=g).to(device, torch.bfloat16)
        _check(x.detach(), w.clone(), b.clone(), None, dy, None)


def test_more_dimensions_and_empty(device):
    x = torch.randn((2, 3, 5, 32), device=device)
    y = sparse_layer_norm(x)
    assert y.shape == x.shape and torch.equal(y.view(-1, 32), sparse_layer_norm(x.view(-1, 32)))
    x = torch.zeros((0, 32), device=device, requires_grad=True)
    w = torch.ones(32, device=device, requires_grad=True)
    dx, dw = torch.autograd.grad(sparse_layer_norm(x, w), [x, w], torch.zeros((0, 32), device=device))
    assert dx.shape == (0, 32) and torch.equal(dw, torch.zeros(32, device=device))


def test_sparse_tensors_share_their_coordinates(device):
    coords = torch.stack([torch.zeros(20), torch.arange(20), torch.arange(20), torch.arange(20)], 1).int().to(device)
    x = SparseTensor(torch.randn((20, 32), device=device), coords, spatial_shape=(20, 20, 20), batch_size=1)
    r = x.replace(torch.randn((20, 32), device=device))
    y, h = sparse_layer_norm(x, residual=r)
    assert isinstance(y, SparseTensor) and y._cache is x._cache and h._cache is x._cache
    assert torch.equal(h.F, x.F + r.F) and torch.equal(y.F, sparse_layer_norm(h.F))


@pytest.mark.parametrize("C", [64, 1000, 1001, 4100])
def test_a_row_that_is_not_finite_stays_alone(device, C):
    x = torch.randn((9, C), device=device)
    clean = sparse_layer_norm(x)
    x[4, 3], x[6, 0] = float("nan"), float("inf")
    got = sparse_layer_norm(x)
    rest = [0, 1, 2, 3, 5, 7, 8]
    assert torch.equal(got[rest], clean[rest]) and torch.isnan(got[4]).all() and torch.isnan(got[6]).any()


@pytest.mark.parametrize("C", [64, 1001])
def test_large_offset_keeps_its_digits(device, C):
    """The variance is a sum of squared differences: a mean of 1000 standard deviations costs three digits, not six."""
    x = torch.randn((16, C), device=device) + 1000.0
    ref = _formula(x, None, None, x, None)[0]
    assert (sparse_layer_norm(x).double() - ref).abs().max().item() < 16 * F32 * 1010 * 2


def test_gradients_against_differences(device):
    """Along random directions: (f(p + e d) - f(p - e d)) / 2e; e = 2^-7 leaves e^2 of curvature and 2^-24 / e of rounding."""
    x, w, b, res, dy, dh = _make(11, 48, torch.float32, torch.float32, True, True, 9, device)
    leaves = [t.requires_grad_(True) for t in (x, w, b, res)]

    def value(ts):
        y, h = sparse_layer_norm(ts[0], ts[1], ts[2], eps=EPS, residual=ts[3])
        return (y.double() * dy.double()).sum() + (h.double() * dh.double()).sum()

    grads = torch.autograd.grad(value(leaves), leaves)
    e = 2.0 ** -7
    for i in range(4):
        d = torch.randn_like(leaves[i])
        with torch.no_grad():
            up = value([t + e * d if k == i else t for k, t in enumerate(leaves)])
            down = value([t - e * d if k == i else t for k, t in enumerate(leaves)])
        slope, got = (up - down) / (2 * e), (grads[i].double() * d.double()).sum()
        scale = (grads[i].double() * d.double()).norm()
        assert (slope - got).abs() <= 2e-3 * scale + 1e-3, (i, slope.item(), got.item())


def test_gradients_are_the_same_bits_on_every_run(device):
    x, w, b, res, dy, dh = _make(30_000, 256, torch.bfloat16, torch.float32, True, True, 10, device)
    leaves = [t.requires_grad_(True) for t in (x, w, b, res)]
    runs = [torch.autograd.grad(sparse_layer_norm(x, w, b, residual=res), leaves, [dy, dh]) for _ in range(3)]
    for other in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(runs[0], other))


def test_only_one_output_is_used(device):
    x, w, b, res, dy, dh = _make(12, 64, torch.float32, torch.float32, True, True, 11, device)
    leaves = [t.requires_grad_(True) for t in (x, w, b, res)]
    y, h = sparse_layer_norm(*leaves[:3], residual=res)
    dx, dw, db, dr = torch.autograd.grad(h, leaves, dh, allow_unused=True, retain_graph=True)
    assert torch.equal(dx, dh) and torch.equal(dr, dh) and not dw.any() and not db.any()
    dx, _, _, dr = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(dx, dr)


def test_another_stream(device):
    x = torch.randn((4000, 256), device=device)
    ref = sparse_layer_norm(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sparse_layer_norm(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, ref)


def test_refusals(device):
    x = torch.randn((4, 8), device=device)
    with pytest.raises(RuntimeError, match="GPU"):
        sparse_layer_norm(torch.randn(4, 8))
    with pytest.raises(TypeError):
        sparse_layer_norm(x.double())
    with pytest.raises(ValueError, match="weight"):
        sparse_layer_norm(x, torch.ones(7, device=device))
    with pytest.raises(ValueError, match="weight"):
        sparse_layer_norm(x, torch.ones(8))
    with pytest.raises(ValueError, match="bias"):
        sparse_layer_norm(x, None, torch.ones(9, device=device))
    with pytest.raises(TypeError):
        sparse_layer_norm(x, torch.ones(8, device=device, dtype=torch.float64))
    with pytest.raises(ValueError, match="residual"):
        sparse_layer_norm(x, residual=x.half())
    with pytest.raises(ValueError, match="residual"):
        sparse_layer_norm(x, residual=x[:3])
    with pytest.raises(ValueError, match="channel"):
        sparse_layer_norm(torch.zeros((4, 0), device=device))
    lib, p = _lib.lib(), x.data_ptr()
    s = _lib.stream_of(x.device)
    assert lib.st_ln_forward(p, None, 4, 0, 0, None, None, 0, 1e-5, None, p, None, None, s) == -1
    assert lib.st_ln_forward(p, p, 4, 8, 0, None, None, 0, 1e-5, None, p, None, None, s) == -1  # residual without H
    assert lib.st_ln_forward(p, None, 4, 8, 7, None, None, 0, 1e-5, None, p, None, None, s) == -3
    assert lib.st_ln_forward(p, None, 4, 8, 1, p, None, 2, 1e-5, None, p, None, None, s) == -3
    assert lib.st_ln_backward(p, p, None, 4, 8, 0, None, 0, p, p, None, 0, p, p, None, s) == -1  # no workspace


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("recorded", [False, True])
def test_forward_mode_is_refused(device, own_random, which, recorded):
    """No forward-mode derivative: a tangent on an input raises, where it is not to be dropped, with or without a graph."""
    t = [torch.randn(s, device=device, requires_grad=recorded) for s in ((5, 16), (16,), (16,), (5, 16))]
    with torch.autograd.forward_ad.dual_level():
        sparse_layer_norm(*t[:3], residual=t[3])
        t[which] = torch.autograd.forward_ad.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            sparse_layer_norm(*t[:3], residual=t[3])
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            sparse_layer_norm(*t[:3], residual=t[3])


def test_more_workgroups_than_one_launch_takes(device):
    """A grid has fewer than 2^32 threads: 2^24 workgroups, each of one row where a row takes all of its lanes."""
    n, C, small = (1 << 24) + 5, 257, 4099
    g = torch.Generator().manual_seed(12)
    part = torch.randn((small, C), generator=g).to(device, torch.bfloat16)
    w = (1 + 0.2 * torch.randn((C,), generator=g)).to(device)
    want, stream = sparse_layer_norm(part, w, residual=part)
    whole = part.repeat(-(-n // small), 1)[:n]
    got, sums = sparse_layer_norm(whole, w, residual=whole)
    for at in range(0, n, 1 << 20):
        rows = torch.arange(at, min(n, at + (1 << 20)), device=device) % small
        assert torch.equal(got[at:at + (1 << 20)], want[rows]) and torch.equal(sums[at:at + (1 << 20)], stream[rows])
