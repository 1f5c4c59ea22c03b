"""sparse_dropout (st_dropout) against its definition: the generator's words in 64-bit integers on the host, the
values in float64.

Tolerances: one rounding to the result's type (half a unit: 2^-24, 2^-11, 2^-8 relative; float16 also 2^-25 of its
smallest numbers) and on the way three in fp32, the scale's, the product's and the sum's: 4 * 2^-24 of |x| scale + |r|.
"""

import copy

import numpy as np
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from sparsetriton_amd import SparseTensor, _lib, nn as snn
from sparsetriton_amd.nn.functional import sparse_dropout

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LOW = np.uint64(0xFFFFFFFF)


def _block(counter, key):
    """Philox 4 x 32, ten rounds: counter (.., 4) and key (2) of 32-bit words."""
    x = [np.asarray(counter[..., i], dtype=np.uint64) for i in range(4)]
    k = [np.uint64(int(w)) for w in key]
    for _ in range(10):
        a, b = np.uint64(0xD2511F53) * x[0], np.uint64(0xCD9E8D57) * x[2]
        x = [(b >> np.uint64(32)) ^ x[1] ^ k[0], b & LOW, (a >> np.uint64(32)) ^ x[3] ^ k[1], a & LOW]
        k = [(k[0] + np.uint64(0x9E3779B9)) & LOW, (k[1] + np.uint64(0xBB67AE85)) & LOW]
    return np.stack(x, -1)


def _kept(numbers, first, count, p):
    """Which of elements first .. first + count - 1 stay."""
    key, call = (int(n) % 2 ** 64 for n in numbers.tolist())
    i = np.arange(first // 4, (first + count + 3) // 4, dtype=np.uint64)
    counter = np.stack([i & LOW, i >> np.uint64(32), np.full_like(i, call & 0xFFFFFFFF), np.full_like(i, call >> 32)], 1)
    words = _block(counter, (key & 0xFFFFFFFF, key >> 32)).reshape(-1)[first % 4:][:count]
    kept = words >= np.uint64(min(2 ** 32 - 1, round(p * 2.0 ** 32)))
    return torch.from_numpy(kept if p < 1 else np.zeros_like(kept))


def _numbers(seed, device="cuda"):
    return torch.from_numpy(np.random.default_rng(seed).integers(-2 ** 63, 2 ** 63 - 1, 2)).to(device)


def _close(y, x, r, kept, p):
    scale = 1.0 / (1.0 - p) if p < 1 else 0.0
    x = torch.where(kept.to(x.device).view(x.shape), x.double(), 0.0) * scale
    want = x if r is None else x + r.double()
    size = x.abs() if r is None else x.abs() + r.double().abs()
    tiny = 2.0 ** -25 if y.dtype == torch.float16 else 0.0
    off = (y.double() - want).abs() - (UNIT[y.dtype] * want.abs() + 4 * 2.0 ** -24 * size + tiny)
    assert y.shape == x.shape and not torch.isnan(y).any() and (off.numel() == 0 or off.max().item() <= 0)


def test_generator_known_answers():
    """The published test vectors of the generator: this file's oracle is the generator that it names."""
    def words(*w):
        return [int(x) for x in w]

    for counter, key, want in (
            ([0] * 4, [0] * 2, [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
            ([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2, [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]),
            ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0],
             [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1])):
        assert words(*_block(np.array(counter, dtype=np.uint64), key)) == want


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1,), (3,), (4, 1), (7, 33), (256, 8), (2049,), (16, 512), (5, 3, 70), (4099, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("p", [0.1, 0.5])
def test_values_and_gradients(device, shape, dtype, residual, p):
    g = torch.Generator().manual_seed(sum(shape))
    rand = lambda: torch.randn(shape, generator=g).to(device, dtype)  # noqa: E731
    x, r, dy, numbers = rand(), rand() if residual else None, rand(), _numbers(len(shape))
    plain = sparse_dropout(x, p, residual=r, numbers=numbers)
    leaves = [t.requires_grad_(True) for t in (x, r) if t is not None]
    y = sparse_dropout(x, p, residual=r, numbers=numbers)
    grads = torch.autograd.grad(y, leaves, dy)
    kept = _kept(numbers, 0, x.numel(), p)
    assert torch.equal(plain, y) and y.dtype == dtype
    _close(y.detach(), x.detach(), None if r is None else r.detach(), kept, p)
    _close(grads[0], dy, None, kept, p)
    assert r is None or torch.equal(grads[1], dy)


@pytest.mark.gpu
@pytest.mark.parametrize("p", [2.0 ** -33, 2.0 ** -20, 0.999, 1.0 - 2.0 ** -40, 1.0])
def test_probabilities_at_the_ends(device, p):
    x, numbers = torch.randn((70_000,), device=device, requires_grad=True), _numbers(3)
    y = sparse_dropout(x, p, numbers=numbers)
    kept = _kept(numbers, 0, x.numel(), p)
    _close(y.detach(), x.detach(), None, kept, p)
    dx, = torch.autograd.grad(y.sum(), x)
    _close(dx, torch.ones_like(x), None, kept, p)
    r = torch.randn_like(x)
    assert p < 1 or torch.equal(sparse_dropout(x, p, residual=r, numbers=numbers), r)


@pytest.mark.gpu
def test_share_kept(device):
    """470,532 x 64 elements: the share kept is p within five standard deviations, and no two calls share a mask."""
    x = torch.ones((470_532, 64), device=device, dtype=torch.bfloat16)
    for p in (0.1, 0.5, 0.9):
        a, b = (sparse_dropout(x, p) != 0 for _ in range(2))
        n = x.numel()
        assert abs(a.float().mean(dtype=torch.float64).item() - (1 - p)) < 5 * (p * (1 - p) / n) ** 0.5
        both = (a & b).float().mean(dtype=torch.float64).item()
        assert abs(both - (1 - p) ** 2) < 5 * ((1 - p) ** 2 * (1 - (1 - p) ** 2) / n) ** 0.5
        assert abs((a[:, 1:] & a[:, :-1]).float().mean(dtype=torch.float64).item() - (1 - p) ** 2) < 1e-3


@pytest.mark.gpu
def test_strides_and_alignment(device):
    numbers = _numbers(5)
    for dtype in (torch.float32, torch.bfloat16):
        flat = torch.randn((4 * 70 + 8,), device=device).to(dtype)
        want = sparse_dropout(flat[:280].clone().view(4, 70), 0.3, residual=flat[8:].clone().view(4, 70), numbers=numbers)
        off = torch.empty((281,), dtype=dtype, device=device)[1:].copy_(flat[:280]).view(4, 70)
        assert torch.equal(sparse_dropout(off, 0.3, residual=flat[8:].view(4, 70), numbers=numbers), want)
        across = torch.empty((70, 4), dtype=dtype, device=device).t().copy_(off)
        got = sparse_dropout(across, 0.3, residual=flat[8:].view(4, 70), numbers=torch.stack((numbers, numbers), 1)[:, 0])
        assert torch.equal(got, want) and got.is_contiguous()
        one = torch.randn((1, 70), device=device).to(dtype).requires_grad_(True)  # a row given to four: its gradient adds over them
        d, = torch.autograd.grad(sparse_dropout(one.expand(4, 70), 0.3, numbers=numbers).sum().float(), one)
        kept = _kept(numbers, 0, 280, 0.3).view(4, 70).to(device).double()
        assert (d.double() - kept.sum(0) / 0.7).abs().max().item() <= 8 * 4 * UNIT[dtype] / 0.7


@pytest.mark.gpu
def test_dropped_values_do_not_matter(device):
    numbers = _numbers(6)
    kept = _kept(numbers, 0, 4000, 0.4).to(device)
    x = torch.randn((4000,), device=device)
    clean = sparse_dropout(x, 0.4, numbers=numbers)
    for bad in (float("nan"), float("inf")):
        y = sparse_dropout(torch.where(kept, x, bad), 0.4, numbers=numbers)
        assert torch.equal(y, clean)
    assert torch.isnan(sparse_dropout(torch.full_like(x, float("nan")), 0.4, numbers=numbers)).equal(kept)


@pytest.mark.gpu
def test_off_and_empty(device, own_random):
    x, r = torch.randn((20, 8), device=device), torch.randn((20, 8), device=device)
    before = torch.cuda.get_rng_state()
    for kw in ({"training": False}, {"p": 0.0}):
        assert torch.equal(sparse_dropout(x, **kw), x) and torch.equal(sparse_dropout(x, residual=r, **kw), r + x)
    assert torch.equal(torch.cuda.get_rng_state(), before)  # nothing drawn
    empty = torch.zeros((0, 8), device=device, requires_grad=True)
    y = sparse_dropout(empty, 0.5, residual=empty)
    assert y.shape == (0, 8) and torch.autograd.grad(y.sum(), empty)[0].shape == (0, 8)


@pytest.mark.gpu
def test_numbers_come_from_torch(device, own_random):
    x = torch.randn((100, 64), device=device)
    torch.manual_seed(7)
    a, b = sparse_dropout(x, 0.5), sparse_dropout(x, 0.5)
    torch.manual_seed(7)
    assert torch.equal(sparse_dropout(x, 0.5), a) and torch.equal(sparse_dropout(x, 0.5), b) and not torch.equal(a, b)


@pytest.mark.gpu
def test_checkpointed_and_differentiated_twice(device, own_random):
    x = torch.randn((300, 40), device=device, requires_grad=True)
    drop = lambda t: sparse_dropout(t.tanh(), 0.5, residual=t)  # noqa: E731
    torch.manual_seed(3)
    y = drop(x)
    want, = torch.autograd.grad(y.square().sum(), x)
    torch.manual_seed(3)
    y2 = checkpoint(drop, x, use_reentrant=False)
    torch.rand((10,), device=device)
    got, = torch.autograd.grad(y2.square().sum(), x)
    assert torch.equal(y, y2) and torch.equal(got, want)
    numbers = _numbers(8)
    y = sparse_dropout(x, 0.25, numbers=numbers)
    v = torch.randn_like(x).requires_grad_(True)
    d, = torch.autograd.grad(y, x, v, create_graph=True)  # what is kept of v, scaled: linear in v
    assert torch.equal(d, sparse_dropout(v, 0.25, numbers=numbers))
    dd, = torch.autograd.grad(d, v, x.detach())
    assert torch.equal(dd, y)


@pytest.mark.gpu
def test_changed_numbers_are_noticed(device):
    x, numbers = torch.randn((10, 8), device=device, requires_grad=True), _numbers(9)
    y = sparse_dropout(x, 0.5, numbers=numbers)
    numbers.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


@pytest.mark.gpu
def test_captured_steps_draw_anew(device, own_random):
    """Forward and backward in a graph: every replay has a mask of its own, the same one in both directions."""
    x, dy = torch.randn((500, 64), device=device), torch.ones((500, 64), device=device)
    given = _numbers(10)

    def step():
        t = x.detach().requires_grad_(True)
        y = sparse_dropout(t, 0.5)
        z = sparse_dropout(t, 0.5, numbers=given)
        return y, z, torch.autograd.grad((y, z), t, (dy, torch.zeros_like(dy)))[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, z, dx = step()
    seen = []
    for i in range(4):
        given.add_(i)
        graph.replay()
        torch.cuda.synchronize()
        kept = dx != 0
        assert torch.equal(y, torch.where(kept, x * 2, 0.0)) and torch.equal(dx, kept * 2.0)
        assert torch.equal(z, sparse_dropout(x, 0.5, numbers=given))
        assert 0.45 < kept.float().mean().item() < 0.55 and not any(torch.equal(kept, k) for k in seen)
        seen.append(kept.clone())


@pytest.mark.gpu
def test_on_another_stream(device):
    x, numbers = torch.randn((3000, 64), device=device), _numbers(11)
    want = sparse_dropout(x, 0.5, numbers=numbers)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sparse_dropout(x, 0.5, numbers=numbers)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_indexes_past_32_bits(device):
    """More elements than 2^32: the mask goes by the 64-bit index (and takes more than one launch's counters)."""
    n, numbers = (1 << 32) + 4100, _numbers(12)
    x = torch.ones((n,), dtype=torch.bfloat16, device=device)
    y = sparse_dropout(x, 0.5, numbers=numbers)
    for first in (0, (1 << 31) - 1000, (1 << 32) - 2000, n - 2001):
        assert torch.equal(y[first:first + 2001].cpu() != 0, _kept(numbers, first, 2001, 0.5))


@pytest.mark.gpu
def test_counters_past_32_bits_and_a_second_launch(device):
    """A grid has fewer than 2^32 threads, 2^24 - 1 workgroups of 2,048 elements: the elements behind those are another launch's,
    and past 2^34 a counter, an index / 4, has a second word."""
    launch = ((1 << 24) - 1) * 2048
    n, numbers = launch + 4100, _numbers(13)
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 4 * n + (8 << 30):
        pytest.skip("needs two tensors of 69 GB")
    x = torch.ones((n,), dtype=torch.bfloat16, device=device)
    y = sparse_dropout(x, 0.5, numbers=numbers)
    try:
        for first in (0, (1 << 34) - 1000, launch - 2048, launch - 1001, n - 2001):
            kept = _kept(numbers, first, 2001, 0.5)
            assert torch.equal(y[first:first + 2001].cpu(), kept.bfloat16() * 2)
    finally:
        del x, y
        torch.cuda.empty_cache()


@pytest.mark.gpu
def test_module(device, own_random):
    drop = snn.SparseDropout(0.5)
    feats = torch.randn((60, 16), device=device)
    x = SparseTensor(feats, torch.randint(0, 9, (60, 4), device=device).int(), spatial_shape=(9, 9, 9))
    y = drop(x)
    assert isinstance(y, SparseTensor) and y._cache is x._cache
    kept = y.F != 0
    assert torch.equal(y.F, torch.where(kept, feats * 2, 0.0)) and not kept.all()
    torch.manual_seed(1)
    a = drop(x, residual=y).F
    torch.manual_seed(1)
    assert torch.equal(drop(feats, residual=y.F), a)
    assert torch.equal(copy.deepcopy(drop).eval()(x).F, feats) and not drop.state_dict()
    assert "p=0.5" in repr(drop)


def test_refusals_before_any_launch():
    with pytest.raises(RuntimeError, match="GPU"):
        sparse_dropout(torch.zeros((3,)))
    with pytest.raises(ValueError, match="probability"):
        snn.SparseDropout(1.5)
    lib = _lib.lib()
    assert lib.st_dropout(None, None, 5, 0, None, 0.5, None, None) == -1
    assert lib.st_dropout(None, None, -1, 0, None, 0.5, None, None) == -1
    for p in (-0.1, 1.1, float("nan")):
        assert lib.st_dropout(None, None, 0, 0, None, p, None, None) == -1
    assert lib.st_dropout(None, None, 0, 0, None, 0.5, None, None) == 0


@pytest.mark.gpu
def test_refusals(device, own_random):
    x = torch.zeros((5, 8), device=device)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="probability"):
            sparse_dropout(x, p)
    for r in (x[:4], x.half(), x.cpu()):
        with pytest.raises(ValueError, match="residual"):
            sparse_dropout(x, residual=r)
    with pytest.raises(TypeError, match="feature dtype"):
        sparse_dropout(x.double())
    with pytest.raises(TypeError, match="int64"):
        sparse_dropout(x, numbers=torch.zeros((2,), dtype=torch.int32, device=device))
    for numbers in (torch.zeros((3,), dtype=torch.int64, device=device), torch.zeros((2,), dtype=torch.int64)):
        with pytest.raises(ValueError, match="numbers"):
            sparse_dropout(x, numbers=numbers)
    with torch.autograd.forward_ad.dual_level():
        t = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for kw in ({}, {"training": False}):
            with pytest.raises(RuntimeError, match="forward-mode"):
                sparse_dropout(t, **kw)
