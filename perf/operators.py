"""Performance cases of the transformer operators over voxel features.

Layer norm with the residual add, rotary positions over the voxel axes, and
attention over segments of packed rows (samples, windows or patches of a
serialised scene), each as a block of a voxel transformer calls them.
``listed()`` names the cases, ``draw(rng)`` gives further ones of the same
ranges, ``prepare`` builds what the program has in hand before the call,
``run`` is one pass -- through the framework's operators where ``own`` is
true, in plain float32 torch otherwise -- and ``exact`` the same pass in
float64 from the definitions.

Case fields
  op         "norm", "rotary" or "attention"
  dtype      "f32", "bf16", "f16": features, gradients and outputs
  train      forward and backward (outputs and all gradients), or forward only
  n          norm, rotary: rows
  c          norm: channels;  residual  the stream's add is part of the pass
  heads, kv_heads, dim    rotary, attention: query heads, key heads, head size
  axes       rotary: "x+y+z" rotated dims of each axis; interleaved: pairs (2p, 2p + 1)
             in place of (p, p + half)
  segs       attention: segments;  q_min..q_max, k_min..k_max their lengths, spread
             over the logarithm (k_max = 0: the keys are the queries' own rows)
  total      attention: rows cut in patches of q_max in place of random lengths
  causal     attention: a query sees keys up to its own place, counted from the end
  masked     attention: share of the keys that a mask leaves out
"""

import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ESZ = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5
BASE = 10000.0
LIDAR_SHAPE = (1440, 1440, 41)


def _norm(name=None, **kw):
    c = {"op": "norm", "dtype": "bf16", "train": True, "n": 0, "c": 64, "residual": False}
    c.update(kw)
    return dict(c, name=name) if name else c


def _rotary(name=None, **kw):
    c = {"op": "rotary", "dtype": "bf16", "train": False, "n": 0, "heads": 8, "kv_heads": 8, "dim": 32,
         "axes": "12+12+8", "interleaved": False}
    c.update(kw)
    return dict(c, name=name) if name else c


def _attention(name=None, **kw):
    c = {"op": "attention", "dtype": "bf16", "train": False, "segs": 1, "total": 0, "q_min": 1, "q_max": 1,
         "k_min": 0, "k_max": 0, "heads": 8, "kv_heads": 8, "dim": 64, "causal": False, "masked": 0.0}
    c.update(kw)
    return dict(c, name=name) if name else c


def listed():
    return [
        # One token for each of 16 scenes on its way through a block at inference: latency.
        _norm("norm_16x512_res", n=16, c=512, residual=True, train=False),
        # A 64-channel stage over four LiDAR sweeps, the benchmark's set, trained in fp32.
        _norm("norm_lidar_64_f32_train", n=470_532, c=64, dtype="f32"),
        # A 512-channel transformer stage with its residual stream, trained in bf16.
        _norm("norm_65537x512_res_train", n=65_537, c=512, residual=True),
        # The same 16 tokens' queries and keys: latency.
        _rotary("rotary_16", n=16, heads=32, kv_heads=8, dim=128, axes="48+48+32"),
        # Queries and keys of a wide first stage over four LiDAR sweeps.
        _rotary("rotary_lidar_8x32", n=470_532),
        # An odd head size with unrotated dims, interleaved pairs, trained in fp32.
        _rotary("rotary_60001_f32_train", n=60_001, heads=6, kv_heads=6, dim=48, axes="16+16+8", interleaved=True,
                dtype="f32", train=True),
        # Window attention: many windows of a few voxels each, inference.
        _attention("attn_windows", segs=2000, q_min=1, q_max=96, heads=4, kv_heads=4, dim=32),
        # A serialised scene cut in patches of 1,024 rows (the last one holds a single row), training.
        _attention("attn_patches_train", total=65_537, q_max=1024, segs=65, dim=64, train=True),
        # One summary token for each scene over all of its voxels, shared key heads: a pass over the keys.
        _attention("attn_one_query", segs=12, q_min=1, q_max=1, k_min=1, k_max=40_000, heads=32, kv_heads=8, dim=128),
        # An autoregressive order over one long scene, shared key heads, training.
        _attention("attn_causal_train", segs=1, q_min=8191, q_max=8191, heads=16, kv_heads=4, dim=128, causal=True,
                   train=True),
        # A detector's 300 queries over the voxels of four scenes, some of them masked out.
        _attention("attn_cross_f16", segs=4, q_min=300, q_max=300, k_min=1000, k_max=20_000, dim=32, dtype="f16",
                   masked=0.2),
        # Samples of very different sizes, padding masked, odd head size, trained in fp32.
        _attention("attn_samples_f32_train", segs=24, q_min=1, q_max=1500, heads=6, kv_heads=6, dim=48, dtype="f32",
                   masked=0.1, train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "rotary", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    train = rng.random() < 0.5
    if op == "norm":
        c = _log_int(rng, 8, 4096)
        if rng.random() < 0.8:
            c = max(8, c // 8 * 8)
        n = _log_int(rng, 1, min(470_532, 33_000_000 // c))
        return _norm(n=n, c=c, dtype=dtype, train=train, residual=rng.random() < 0.5)
    kv_heads = rng.choice([1, 2, 4, 6, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    dim = rng.choice([16, 24, 32, 48, 64, 64, 80, 96, 128])
    if op == "rotary":
        a = [max(2, 2 * rng.randint(1, dim // 6)) for _ in range(rng.choice([1, 2, 3]))]
        n = _log_int(rng, 1, min(470_532, 120_000_000 // ((heads + kv_heads) * dim)))
        return _rotary(n=n, heads=heads, kv_heads=kv_heads, dim=dim, axes="+".join(map(str, a)), dtype=dtype, train=train,
                       interleaved=rng.random() < 0.5)
    kind = rng.choice(["windows", "patches", "query", "long", "cross"])
    c = _attention(dtype=dtype, train=train, heads=heads, kv_heads=kv_heads, dim=dim, causal=rng.random() < 0.3,
                   masked=rng.choice([0.0, 0.0, 0.1, 0.5]))
    if kind == "windows":
        c.update(segs=_log_int(rng, 20, 2000), q_max=_log_int(rng, 8, 128))
    elif kind == "patches":
        size = rng.choice([128, 256, 500, 1024])
        total = _log_int(rng, 1000, 65_537)
        c.update(total=total, q_max=size, segs=-(-total // size))
    elif kind == "query":
        c.update(segs=_log_int(rng, 1, 32), q_max=rng.choice([1, 1, 4]), k_min=1, k_max=_log_int(rng, 100, 40_000),
                 train=False)
    elif kind == "long":
        n = _log_int(rng, 500, 8191)
        c.update(segs=1, q_min=n, q_max=n)
    else:
        c.update(segs=_log_int(rng, 1, 8), q_min=10, q_max=_log_int(rng, 20, 1000), k_min=100,
                 k_max=_log_int(rng, 200, 20_000))
    # no more than the largest listed case: products, and the scores that the plain form holds
    while True:
        lq, lk = c["q_max"], c["k_max"] or c["q_max"]
        scores = c["segs"] * lq * lk * c["heads"]
        most = 2.7e11 if dtype != "f32" else 5e10
        if scores <= 1.0e9 and 4.0 * scores * c["dim"] <= most:
            return c
        if c["heads"] > c["kv_heads"]:
            c["heads"] = c["kv_heads"]
        elif c["kv_heads"] > 1:
            c["kv_heads"] = c["heads"] = c["kv_heads"] // 2
        elif c["total"]:
            c["total"] = max(1000, c["total"] // 2)
            c["segs"] = -(-c["total"] // c["q_max"])
        elif c["segs"] > 1:
            c["segs"] //= 2
        else:
            c["q_max"] = max(1, c["q_max"] // 2)
            c["q_min"] = min(c["q_min"], c["q_max"])


def _lengths(case, seed):
    """Rows of each segment: (queries, keys).  They go by the case alone: seeds change the values."""
    rng = random.Random(case["segs"] * 7919 + case["q_max"] * 31 + case["k_max"])
    if case["total"]:
        q = [case["q_max"]] * (case["total"] // case["q_max"])
        if case["total"] % case["q_max"]:
            q.append(case["total"] % case["q_max"])
        return q, q
    q = [_log_int(rng, case["q_min"], case["q_max"]) for _ in range(case["segs"])]
    if not case["k_max"]:
        return q, q
    k = [_log_int(rng, case["k_min"], case["k_max"]) for _ in range(case["segs"])]
    k[-1] = case["k_max"]
    return q, k


def _axes(case):
    return [int(a) for a in case["axes"].split("+")]


def _frequencies(axes):
    """(axis, frequency in fp32) of each rotated pair."""
    at = [a for a, d in enumerate(axes) for _ in range(d // 2)]
    f = [BASE ** (-2.0 * i / d) for d in axes for i in range(d // 2)]
    return at, f


class State:
    pass


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 17)
    dt = DTYPES[case["dtype"]]
    s = State()
    s.case = case

    def randn(*shape, grad=False, scale=1.0, dtype=dt):
        t = (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)
        return t.requires_grad_(True) if grad else t

    train = case["train"]
    if case["op"] == "norm":
        n, c = case["n"], case["c"]
        # features: a shared offset and a spread for each channel, as after a projection
        with torch.no_grad():
            s.x = (randn(n, c, dtype=torch.float32) * (0.5 + torch.rand((c,), generator=g, device="cuda"))
                   + 0.3 * randn(c, dtype=torch.float32)).to(dt).requires_grad_(train)
        s.res = randn(n, c, grad=train) if case["residual"] else None
        s.w = (1 + 0.2 * randn(c, dtype=torch.float32)).to(dt).requires_grad_(train)
        s.b = (0.2 * randn(c, dtype=torch.float32)).to(dt).requires_grad_(train)
        s.dy = randn(n, c)
        s.dh = randn(n, c) if case["residual"] else None
    elif case["op"] == "rotary":
        n, dim, axes = case["n"], case["dim"], _axes(case)
        s.q, s.k = randn(n, case["heads"], dim, grad=train), randn(n, case["kv_heads"], dim, grad=train)
        s.dq, s.dk = randn(n, case["heads"], dim), randn(n, case["kv_heads"], dim)
        s.pos = torch.stack([torch.randint(0, LIDAR_SHAPE[a], (n,), generator=g, device="cuda") for a in range(len(axes))],
                            1).to(torch.int16)
        at, f = _frequencies(axes)
        s.axis = torch.tensor(at, device="cuda")
        s.freq = torch.tensor(f, dtype=torch.float64).float().cuda()
        if own:  # the handle that a program keeps beside its weights
            from sparsetriton_amd.nn.functional import RotaryAxes
            s.rotary = RotaryAxes(dim, axes, base=BASE, interleaved=case["interleaved"])
    else:
        ql, kl = _lengths(case, seed)
        nq, nk, d = sum(ql), sum(kl), case["dim"]
        s.q = randn(nq, case["heads"], d, grad=train)
        s.k, s.v = randn(nk, case["kv_heads"], d, grad=train), randn(nk, case["kv_heads"], d, grad=train)
        s.do = randn(nq, case["heads"], d)
        s.mask = torch.rand((nk,), generator=g, device="cuda") >= case["masked"] if case["masked"] else None
        s.ql, s.kl = torch.tensor(ql, device="cuda"), torch.tensor(kl, device="cuda")
        s.lq, s.lk = max(ql), max(kl)
        if own:  # the plan of the scene's row groups, which all blocks of a stage share
            from sparsetriton_amd.nn.functional import AttentionSegments
            s.segments = AttentionSegments(ql, None if ql is kl else kl, device="cuda")
    return s


# ------------------------------------------------------------------ plain forms


def _plain_norm(s):
    x = s.x.detach().float()
    if s.res is not None:
        h = (x + s.res.detach().float()).to(s.x.dtype)
        x = h.float()
    w, b = s.w.detach().float(), s.b.detach().float()
    mu = x.mean(1, keepdim=True)
    rs = torch.rsqrt(((x - mu) ** 2).mean(1, keepdim=True) + EPS)
    xh = (x - mu) * rs
    y = (xh * w + b).to(s.x.dtype)
    out = [y] if s.res is None else [y, h]
    if not s.case["train"]:
        return out
    dy = s.dy.float()
    gw = dy * w
    dx = rs * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
    if s.res is not None:
        dx = dx + s.dh.float()
    dx = dx.to(s.x.dtype)
    return out + [dx] + ([dx] if s.res is not None else []) + [(dy * xh).sum(0).to(s.w.dtype), dy.sum(0).to(s.b.dtype)]


def _turn(t, cos, sin, interleaved):
    """The rotation of t (N, H, D) in fp32, rounded to its type."""
    x = t.detach().float()
    p = cos.shape[1]
    c, s = cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0:2 * p:2], x[..., 1:2 * p:2]
        turned = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    else:
        a, b = x[..., :p], x[..., p:2 * p]
        turned = torch.cat((a * c - b * s, a * s + b * c), -1)
    return torch.cat((turned, x[..., 2 * p:]), -1).to(t.dtype)


def _plain_rotary(s):
    angle = s.pos.float()[:, s.axis] * s.freq
    cos, sin, il = torch.cos(angle), torch.sin(angle), s.case["interleaved"]
    out = [_turn(s.q, cos, sin, il), _turn(s.k, cos, sin, il)]
    if s.case["train"]:
        out += [_turn(s.dq, cos, -sin, il), _turn(s.dk, cos, -sin, il)]
    return out


def _places(lens):
    """(segment, place in it) of each packed row."""
    seg = torch.repeat_interleave(torch.arange(lens.numel(), device=lens.device), lens)
    return seg, torch.arange(seg.numel(), device=lens.device) - (torch.cumsum(lens, 0) - lens)[seg]


def _padded(t, seg, at, segs, length):
    """(segments, heads, length, D) in fp32, zeros where a segment is shorter."""
    p = torch.zeros((segs, length) + t.shape[1:], device=t.device)
    p[seg, at] = t.detach().float()
    return p.transpose(1, 2).contiguous()


def _plain_attention(s):
    hk, d = s.case["kv_heads"], s.case["dim"]
    r, segs, scale = s.case["heads"] // hk, s.ql.numel(), d ** -0.5
    sq, aq = _places(s.ql)
    sk, ak = _places(s.kl)
    group = lambda t: t.reshape(segs, hk, r * s.lq, d)  # noqa: E731  (the query heads that share a key head)
    q = group(_padded(s.q, sq, aq, segs, s.lq))
    k, v = _padded(s.k, sk, ak, segs, s.lk), _padded(s.v, sk, ak, segs, s.lk)
    seen = torch.zeros((segs, s.lk), dtype=torch.bool, device=q.device)
    seen[sk, ak] = True if s.mask is None else s.mask
    seen = seen[:, None, :]
    if s.case["causal"]:
        i, j = torch.arange(s.lq, device=q.device), torch.arange(s.lk, device=q.device)
        seen = seen & (j[None, None, :] <= i[None, :, None] + (s.kl - s.ql)[:, None, None])
    seen = seen[:, None, None]
    p = torch.matmul(q, k.transpose(2, 3)).mul_(scale).view(segs, hk, r, s.lq, s.lk)
    p.masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = torch.exp_(p.sub_(torch.where(torch.isfinite(top), top, 0.0)))
    total = p.sum(-1, keepdim=True)
    p = p.mul_(torch.where(total > 0, 1.0 / total, 0.0)).view(segs, hk, r * s.lq, s.lk)
    back = lambda t, seg, at: t.transpose(1, 2)[seg, at].to(s.q.dtype)  # noqa: E731
    heads = lambda t: t.view(segs, hk * r, s.lq, d)  # noqa: E731
    o = torch.matmul(p, v)
    out = [back(heads(o), sq, aq)]
    if not s.case["train"]:
        return out
    do = group(_padded(s.do, sq, aq, segs, s.lq))
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = torch.matmul(do, v.transpose(2, 3)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(2, 3), q)
    return out + [back(heads(dq), sq, aq), back(dk, sk, ak), back(dv, sk, ak)]


# ------------------------------------------------------------------ the framework's operators


def _own_norm(s):
    from sparsetriton_amd.nn.functional import sparse_layer_norm
    out = sparse_layer_norm(s.x, s.w, s.b, eps=EPS, residual=s.res)
    out = [out] if s.res is None else list(out)
    if not s.case["train"]:
        return out
    ins = [s.x] + ([s.res] if s.res is not None else []) + [s.w, s.b]
    return out + list(torch.autograd.grad(out, ins, [s.dy] if s.res is None else [s.dy, s.dh]))


def _own_rotary(s):
    from sparsetriton_amd.nn.functional import sparse_rotary
    out = list(sparse_rotary(s.q, s.k, s.pos, s.rotary))
    return out + list(torch.autograd.grad(out, [s.q, s.k], [s.dq, s.dk])) if s.case["train"] else out


def _own_attention(s):
    from sparsetriton_amd.nn.functional import sparse_attention
    out = sparse_attention(s.q, s.k, s.v, s.segments, causal=s.case["causal"], key_mask=s.mask)
    return [out] + list(torch.autograd.grad(out, [s.q, s.k, s.v], s.do)) if s.case["train"] else [out]


def run(state):
    op = state.case["op"]
    if own:
        return _own_norm(state) if op == "norm" else _own_rotary(state) if op == "rotary" else _own_attention(state)
    return _plain_norm(state) if op == "norm" else _plain_rotary(state) if op == "rotary" else _plain_attention(state)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    e = ESZ[case["dtype"]]
    if case["op"] == "norm":
        n, c, r = case["n"], case["c"], case["residual"]
        # forward: x (and the residual) in, y (and the stream) out; backward: the stream, dy (and its gradient) in, dx out
        passes = (4 if r else 2) + ((4 if r else 3) if case["train"] else 0)
        return {"bytes": passes * n * c * e + 4 * c * e, "flops": n * c * (8 + (14 if case["train"] else 0))}
    if case["op"] == "rotary":
        size = case["n"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        both = 2 if case["train"] else 1
        return {"bytes": both * (2 * size * e + 2 * case["n"] * len(_axes(case))), "flops": both * 3 * size}
    ql, kl = _lengths(case, 0)
    if case["causal"]:  # query i of nq sees i + 1 + nk - nq keys
        pairs = sum(sum(min(k, max(0, i + 1 + k - q)) for i in range(q)) for q, k in zip(ql, kl))
    else:
        pairs = sum(q * k for q, k in zip(ql, kl))
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    qb, kb = sum(ql) * h * d * e, sum(kl) * hk * d * e
    if not case["train"]:
        return {"bytes": 2 * qb + 2 * kb, "flops": 4 * pairs * h * d}
    return {"bytes": (2 + 4) * qb + (2 + 4) * kb, "flops": 14 * pairs * h * d}


# ------------------------------------------------------------------ the definitions in 64 bits


def _exact_norm(s):
    f = lambda t: t.detach().double()  # noqa: E731
    h = f(s.x)
    if s.res is not None:
        h = (h + f(s.res)).to(s.x.dtype).double()  # the stream goes on in its own type
    var, mu = torch.var_mean(h, dim=1, correction=0, keepdim=True)
    sd = torch.sqrt(var + EPS)
    z = (h - mu) / sd
    out = [z * f(s.w) + f(s.b)] + ([h] if s.res is not None else [])
    if s.case["train"]:
        t, c = f(s.dy) * f(s.w), s.x.shape[1]
        d = (c * t - t.sum(1, keepdim=True) - z * (t * z).sum(1, keepdim=True)) / (c * sd)
        if s.res is not None:
            d = d + f(s.dh)
        out += [d] * (1 if s.res is None else 2) + [torch.einsum("nc,nc->c", f(s.dy), z), f(s.dy).sum(0)]
    return out


def _exact_rotary(s):
    # each pair as a complex number, turned by exp(i angle)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       torch.stack([s.pos[:, int(a)].double() * s.freq[p].double() for p, a in enumerate(s.axis.tolist())], 1))
    p = s.freq.numel()
    even = torch.arange(p, device="cuda") * 2 if s.case["interleaved"] else torch.arange(p, device="cuda")
    odd = even + (1 if s.case["interleaved"] else p)

    def at(t, z):
        x = t.detach().double().clone()
        w = torch.complex(x[..., even], x[..., odd]) * z[:, None]
        x[..., even], x[..., odd] = w.real, w.imag
        return x

    out = [at(s.q, turn), at(s.k, turn)]
    return out + [at(s.dq, turn.conj()), at(s.dk, turn.conj())] if s.case["train"] else out


def _exact_attention(s):
    q, k, v, do = (t.detach().double().transpose(0, 1).contiguous() for t in (s.q, s.k, s.v, s.do))
    r, scale = s.case["heads"] // s.case["kv_heads"], s.case["dim"] ** -0.5
    o, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    q0 = k0 = 0
    for nq, nk in zip(s.ql.tolist(), s.kl.tolist()):
        Q, K = slice(q0, q0 + nq), slice(k0, k0 + nk)
        drop = torch.zeros((nq, nk), dtype=torch.bool, device="cuda")
        if s.mask is not None:
            drop |= ~s.mask[K]
        if s.case["causal"]:
            drop |= torch.ones((nq, nk), dtype=torch.bool, device="cuda").triu(1 + nk - nq)
        none = drop.all(1, keepdim=True)
        for h0 in range(0, q.shape[0], r if nq * nk > 4_000_000 else q.shape[0]):
            hs = range(h0, h0 + (r if nq * nk > 4_000_000 else q.shape[0]))
            kv = [h // r for h in hs]
            H = slice(hs[0], hs[-1] + 1)
            z = (q[H, Q] @ k[kv, K].transpose(1, 2)) * scale
            p = torch.softmax(z.masked_fill(drop, -math.inf), -1).masked_fill(none, 0.0)
            del z
            o[H, Q] = p @ v[kv, K]
            if s.case["train"]:
                dp = do[H, Q] @ v[kv, K].transpose(1, 2)
                dz = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
                dq[H, Q] = dz @ k[kv, K]
                part = torch.stack((dz.transpose(1, 2) @ q[H, Q], p.transpose(1, 2) @ do[H, Q]))
                part = part.view(2, len(kv) // r, r, nk, -1).sum(2)
                dk[kv[0]:kv[-1] + 1, K], dv[kv[0]:kv[-1] + 1, K] = part[0], part[1]
        q0, k0 = q0 + nq, k0 + nk
    out = [o] + ([dq, dk, dv] if s.case["train"] else [])
    return [t.transpose(0, 1) for t in out]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s)
    return _exact_rotary(s) if case["op"] == "rotary" else _exact_attention(s)
