"""Performance cases of a transformer block's further operators over voxel features.

Norms of queries and keys for each head with the position rotation in the same
pass, attention with a sliding window and a few first rows that stay visible,
and dropout (with the residual add) whose mask comes from a counter and is
never stored.  ``listed()`` names the cases, ``draw(rng)`` gives further ones
of the same ranges, ``prepare`` builds what the program has in hand before the
call, ``run`` is one pass -- through the framework's operators where ``own`` is
true, in plain float32 torch otherwise -- and ``exact`` the same pass in
float64 from the definitions.

Case fields
  op         "qk", "window" or "dropout"
  dtype      "f32", "bf16", "f16": features, weights, gradients and outputs
  train      forward and backward (outputs and all gradients), or forward only
  heads, kv_heads, dim    qk, window: query heads, key heads, head size
  n          qk, dropout: rows
  axes       qk: "x+y+z" rotated dims of each axis; interleaved: pairs (2p, 2p + 1)
             in place of (p, p + half)
  segs       window: segments;  q_min..q_max, k_min..k_max their lengths, spread over
             the logarithm (k_max = 0: the keys are the queries' own rows)
  window     window: keys at places less than so many from the row's own place
             (counted from the end), before it (causal) or on both sides
  sinks      window: first keys of the segment that stay visible
  masked     window: share of the keys that a mask leaves out
  c          dropout: channels;  p  share dropped;  residual  the stream's add is
             part of the pass
"""

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ESZ = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6
BASE = 10000.0
LIDAR_SHAPE = (1440, 1440, 41)


def _qk(name=None, **kw):
    c = {"op": "qk", "dtype": "bf16", "train": False, "n": 0, "heads": 8, "kv_heads": 8, "dim": 32,
         "axes": "12+12+8", "interleaved": False}
    c.update(kw)
    return dict(c, name=name) if name else c


def _window(name=None, **kw):
    c = {"op": "window", "dtype": "bf16", "train": False, "segs": 1, "q_min": 1, "q_max": 1, "k_min": 0, "k_max": 0,
         "heads": 8, "kv_heads": 8, "dim": 64, "causal": True, "window": 1024, "sinks": 4, "masked": 0.0}
    c.update(kw)
    return dict(c, name=name) if name else c


def _dropout(name=None, **kw):
    c = {"op": "dropout", "dtype": "bf16", "train": True, "n": 0, "c": 64, "p": 0.1, "residual": False}
    c.update(kw)
    return dict(c, name=name) if name else c


def listed():
    return [
        # One token for each of 16 scenes on its way through a block at inference: latency.
        _qk("qk_16", n=16, heads=32, kv_heads=8, dim=128, axes="48+48+32"),
        # Queries and keys of a wide first stage over four LiDAR sweeps, the benchmark's set.
        _qk("qk_lidar_8x32", n=470_532),
        # A block with shared key heads, trained in bf16.
        _qk("qk_65537_train", n=65_537, heads=16, kv_heads=4, dim=128, axes="48+48+32", train=True),
        # An odd head size with unrotated dims, interleaved pairs, trained in fp32.
        _qk("qk_60001_f32_train", n=60_001, heads=6, kv_heads=6, dim=48, axes="16+16+8", interleaved=True, dtype="f32",
            train=True),
        # One new row for each of 16 scenes, generated row by row, over the rows so far: latency.
        _window("window_one_query", segs=16, q_min=1, q_max=1, k_min=500, k_max=40_000, heads=32, kv_heads=8, dim=128),
        # The order of generation over one long scene, shared key heads, training.
        _window("window_causal_train", q_min=16_383, q_max=16_383, heads=16, kv_heads=4, dim=128, train=True),
        # Serialised scenes of different sizes, each row and its neighbours on both sides, training.
        _window("window_scenes_train", segs=4, q_min=2000, q_max=20_000, causal=False, window=256, sinks=0, train=True),
        # Scenes read in before the generation of further rows, an odd window and head size, inference.
        _window("window_prompts_f16", segs=6, q_min=1, q_max=8191, kv_heads=2, dim=80, window=500, sinks=16, dtype="f16"),
        # Samples of very different sizes, padding masked, summary rows at their head, trained in fp32.
        _window("window_samples_f32_train", segs=24, q_min=1, q_max=1500, heads=6, kv_heads=6, dim=48, causal=False,
                window=100, sinks=3, masked=0.1, dtype="f32", train=True),
        # The 16 tokens' branch back into their stream: latency.
        _dropout("dropout_16x512_res", n=16, c=512, residual=True, train=False),
        # A 64-channel stage over four LiDAR sweeps, trained in fp32.
        _dropout("dropout_lidar_64_f32_train", n=470_532, c=64, p=0.3, dtype="f32"),
        # A 512-channel stage's branch back into its stream, trained in bf16.
        _dropout("dropout_65537x512_res_train", n=65_537, c=512, residual=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["qk", "window", "window", "dropout"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    train = rng.random() < 0.5
    if op == "dropout":
        c = _log_int(rng, 8, 4096)
        if rng.random() < 0.7:
            c = max(8, c // 8 * 8)
        n = _log_int(rng, 1, min(470_532, 33_000_000 // c))
        return _dropout(n=n, c=c, p=rng.choice([0.05, 0.1, 0.3, 0.5]), dtype=dtype, train=train, residual=rng.random() < 0.5)
    kv_heads = rng.choice([1, 2, 4, 6, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    dim = rng.choice([16, 24, 32, 48, 64, 64, 80, 96, 128])
    if op == "qk":
        a = [max(2, 2 * rng.randint(1, dim // 6)) for _ in range(rng.choice([1, 2, 3]))]
        n = _log_int(rng, 1, min(470_532, 80_000_000 // ((heads + kv_heads) * dim)))
        return _qk(n=n, heads=heads, kv_heads=kv_heads, dim=dim, axes="+".join(map(str, a)), dtype=dtype, train=train,
                   interleaved=rng.random() < 0.5)
    kind = rng.choice(["query", "long", "samples", "next"])
    c = _window(dtype=dtype, train=train, heads=heads, kv_heads=kv_heads, dim=dim, causal=rng.random() < 0.6,
                window=_log_int(rng, 16, 4096), sinks=rng.choice([0, 0, 1, 4, 64, 130]), masked=rng.choice([0.0, 0.0, 0.1]))
    if kind == "query":  # single rows over the rows so far
        c.update(segs=_log_int(rng, 1, 32), q_max=1, k_min=1, k_max=_log_int(rng, 100, 40_000), train=False, causal=True)
    elif kind == "long":
        n = _log_int(rng, 500, 16_383)
        c.update(segs=1, q_min=n, q_max=n)
    elif kind == "samples":
        c.update(segs=_log_int(rng, 2, 24), q_max=_log_int(rng, 20, 8191))
    else:  # some further rows of each scene over all of it
        c.update(segs=_log_int(rng, 1, 8), q_min=2, q_max=_log_int(rng, 20, 1000), k_min=1000, k_max=_log_int(rng, 2000, 20_000),
                 causal=True)
    # no more than the largest listed case: products of the visible pairs
    while True:
        most = 4.0e11 if dtype != "f32" else 5.0e10
        if 4.0 * _pairs(c) * c["heads"] * c["dim"] * (3.5 if c["train"] else 1.0) <= most:
            return c
        if c["window"] > 64:
            c["window"] //= 2
        elif c["heads"] > c["kv_heads"]:
            c["heads"] = c["kv_heads"]
        elif c["segs"] > 1:
            c["segs"] //= 2
        else:
            c["q_max"] = max(1, c["q_max"] // 2)
            c["q_min"] = min(c["q_min"], c["q_max"])


def _lengths(case):
    """Rows of each segment: (queries, keys).  They go by the case alone: seeds change the values."""
    rng = random.Random(case["segs"] * 7919 + case["q_max"] * 31 + case["k_max"])
    q = [_log_int(rng, case["q_min"], case["q_max"]) for _ in range(case["segs"])]
    if not case["k_max"]:
        q[-1] = case["q_max"]
        return q, q
    k = [_log_int(rng, case["k_min"], case["k_max"]) for _ in range(case["segs"])]
    k[-1] = case["k_max"]
    return q, k


def _reach(case, nq, nk, i0, i1):
    """Keys (lo, hi) that the windows of queries i0 .. i1 - 1 of a segment cover, sinks aside."""
    off, w = nk - nq, case["window"]
    hi = i1 - 1 + off + (1 if case["causal"] else w)
    hi = max(0, min(nk, hi))
    return max(0, min(hi, i0 + off - w + 1)), hi


def _pairs(case):
    """Visible (query, key) pairs of one head."""
    total = 0
    for nq, nk in zip(*_lengths(case)):
        i = np.arange(nq, dtype=np.int64)
        p, w = i + nk - nq, case["window"]
        hi = np.clip(p + (1 if case["causal"] else w), 0, nk)
        lo = np.clip(p - w + 1, 0, hi)
        sinks = np.minimum(min(case["sinks"], nk), np.maximum(hi, 0) if case["causal"] else nk)
        total += int((hi - lo + np.where(lo < hi, np.minimum(sinks, lo), sinks)).sum())
    return total


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
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 29)
    dt = DTYPES[case["dtype"]]
    s = State()
    s.case = case
    train = case["train"]

    def randn(*shape, grad=False, dtype=dt):
        t = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)
        return t.requires_grad_(True) if grad else t

    if case["op"] == "qk":
        n, dim, axes = case["n"], case["dim"], _axes(case)
        # projections of different sizes for each channel
        spread = 0.3 + 2 * torch.rand((dim,), generator=g, device="cuda")
        with torch.no_grad():
            s.q = (randn(n, case["heads"], dim, dtype=torch.float32) * spread).to(dt).requires_grad_(train)
            s.k = (randn(n, case["kv_heads"], dim, dtype=torch.float32) * spread).to(dt).requires_grad_(train)
        s.wq = (1 + 0.2 * randn(dim, dtype=torch.float32)).to(dt).requires_grad_(train)
        s.wk = (1 + 0.2 * randn(dim, dtype=torch.float32)).to(dt).requires_grad_(train)
        s.dq, s.dk = randn(n, case["heads"], dim), randn(n, case["kv_heads"], dim)
        s.pos = torch.stack([torch.randint(0, LIDAR_SHAPE[a], (n,), generator=g, device="cuda") for a in range(len(axes))],
                            1).to(torch.int16)
        at, f = _frequencies(axes)
        s.axis = torch.tensor(at, device="cuda")
        s.freq = torch.tensor(f, dtype=torch.float64).float().cuda()
        if own:  # the handle that a program keeps beside its weights
            from sparsetriton_amd.nn.functional import RotaryAxes
            s.rotary = RotaryAxes(dim, axes, base=BASE, interleaved=case["interleaved"])
    elif case["op"] == "window":
        ql, kl = _lengths(case)
        nq, nk, d = sum(ql), sum(kl), case["dim"]
        s.q = randn(nq, case["heads"], d, grad=train)
        s.k, s.v = randn(nk, case["kv_heads"], d, grad=train), randn(nk, case["kv_heads"], d, grad=train)
        s.do = randn(nq, case["heads"], d)
        s.mask = torch.rand((nk,), generator=g, device="cuda") >= case["masked"] if case["masked"] else None
        s.lengths, s.kl = (ql, kl), torch.tensor(kl, device="cuda")
        if own:  # the plan of the scenes' rows, which all blocks of a stage share
            from sparsetriton_amd.nn.functional import AttentionSegments
            s.segments = AttentionSegments(ql, None if ql is kl else kl, device="cuda")
    else:
        n, c = case["n"], case["c"]
        s.x = randn(n, c, grad=train)
        s.res = randn(n, c, grad=train) if case["residual"] else None
        s.dy = randn(n, c)
        s.numbers = torch.randint(0, 2 ** 62, (2,), generator=g, device="cuda")
    return s


# ------------------------------------------------------------------ plain forms


def _turn(x, cos, sin, interleaved):
    """The rotation of x (N, H, D) in fp32."""
    p = cos.shape[1]
    c, s = cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0:2 * p:2], x[..., 1:2 * p:2]
        turned = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    else:
        a, b = x[..., :p], x[..., p:2 * p]
        turned = torch.cat((a * c - b * s, a * s + b * c), -1)
    return torch.cat((turned, x[..., 2 * p:]), -1)


def _plain_qk(s):
    angle = (s.pos.double()[:, s.axis] * s.freq.double())
    cos, sin, il = torch.cos(angle).float(), torch.sin(angle).float(), s.case["interleaved"]
    out, grads, weights = [], [], []
    for x, w, dy in ((s.q, s.wq, s.dq), (s.k, s.wk, s.dk)):
        x, w = x.detach().float(), w.detach().float()
        rs = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        xh = x * rs
        out.append(_turn(xh * w, cos, sin, il).to(s.q.dtype))
        if s.case["train"]:
            g = _turn(dy.float(), cos, -sin, il)
            gw = g * w
            grads.append((rs * (gw - xh * (gw * xh).mean(-1, keepdim=True))).to(s.q.dtype))
            weights.append((g * xh).sum((0, 1)).to(s.wq.dtype))
    return out + grads + weights


def _plain_query(s):
    """Single queries: each one's sinks and last keys gathered side by side."""
    c, hk, d = s.case, s.case["kv_heads"], s.case["dim"]
    segs, r, w = s.kl.numel(), c["heads"] // hk, c["window"]
    first = torch.cumsum(s.kl, 0) - s.kl
    at = torch.cat((torch.arange(c["sinks"], device="cuda").expand(segs, -1),
                    (s.kl - w)[:, None] + torch.arange(w, device="cuda")), 1)
    seen = (at >= 0) & (at < s.kl[:, None])
    seen[:, :c["sinks"]] &= at[:, :c["sinks"]] < (s.kl - w)[:, None]  # (the others are in the window)
    rows = first[:, None] + at.clamp_min(0).minimum((s.kl - 1)[:, None])
    if s.mask is not None:
        seen = seen & s.mask[rows]
    k, v = (t.detach()[rows].float().transpose(1, 2).contiguous() for t in (s.k, s.v))  # (segs, hk, keys, d)
    q = s.q.detach().float().view(segs, hk, r, d)
    p = torch.matmul(q, k.transpose(2, 3)).mul_(d ** -0.5).masked_fill_(~seen[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p = torch.exp_(p.sub_(torch.where(torch.isfinite(top), top, 0.0)))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) * torch.where(total > 0, 1.0 / total, 0.0)
    return [o.view(segs, hk * r, d).to(s.q.dtype)]


def _plain_window(s):
    """Blocks of a segment's queries over the sinks and the keys that their windows cover."""
    c, hk, d = s.case, s.case["kv_heads"], s.case["dim"]
    if c["q_max"] == 1:
        return _plain_query(s)
    r, scale, block = c["heads"] // hk, d ** -0.5, 1024
    f = lambda t: t.detach().float().transpose(0, 1).contiguous()  # noqa: E731  (heads first)
    q, k, v, do = f(s.q), f(s.k), f(s.v), f(s.do)
    o = torch.zeros_like(q)
    if c["train"]:
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    q0 = k0 = 0
    for nq, nk in zip(*s.lengths):
        for i0 in range(0, nq, block):
            i1 = min(nq, i0 + block)
            lo, hi = _reach(c, nq, nk, i0, i1)
            n0 = min(c["sinks"], nk) if hi <= lo else min(c["sinks"], lo)
            at = torch.cat((torch.arange(n0, device="cuda"), torch.arange(lo, max(lo, hi), device="cuda")))
            if not at.numel():
                continue
            place = torch.arange(i0, i1, device="cuda")[:, None] + (nk - nq)
            seen = at > place - c["window"]
            if not c["causal"]:
                seen &= at < place + c["window"]
            seen |= at < c["sinks"]
            if c["causal"]:
                seen &= at <= place
            rows, Q = at + k0, slice(q0 + i0, q0 + i1)
            if s.mask is not None:
                seen &= s.mask[rows]
            kb, vb = k[:, rows], v[:, rows]
            b = i1 - i0
            qb = q[:, Q].view(hk, r, b, d).reshape(hk, r * b, d)
            p = torch.matmul(qb, kb.transpose(1, 2)).mul_(scale).view(hk, r, b, -1).masked_fill_(~seen, -math.inf)
            top = p.amax(-1, keepdim=True)
            p = torch.exp_(p.sub_(torch.where(torch.isfinite(top), top, 0.0)))
            total = p.sum(-1, keepdim=True)
            p = p.mul_(torch.where(total > 0, 1.0 / total, 0.0)).view(hk, r * b, -1)
            ob = torch.matmul(p, vb)
            o[:, Q] = ob.view(hk * r, b, d)
            if c["train"]:
                gb = do[:, Q].view(hk, r, b, d).reshape(hk, r * b, d)
                dv[:, rows] += torch.matmul(p.transpose(1, 2), gb)
                ds = torch.matmul(gb, vb.transpose(1, 2)).sub_((gb * ob).sum(-1, keepdim=True)).mul_(p).mul_(scale)
                dq[:, Q] = torch.matmul(ds, kb).view(hk * r, b, d)
                dk[:, rows] += torch.matmul(ds.transpose(1, 2), qb)
        q0, k0 = q0 + nq, k0 + nk
    back = lambda t: t.transpose(0, 1).to(s.q.dtype).contiguous()  # noqa: E731
    return [back(o)] + ([back(dq), back(dk), back(dv)] if c["train"] else [])


# Philox 4 x 32 with ten rounds (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; 2011):
# element e of the tensor takes word e % 4 of the block that the counter (e / 4, numbers[1]) has under the key numbers[0].
PHILOX_M = (0xD2511F53, 0xCD9E8D57)
PHILOX_W = (0x9E3779B9, 0xBB67AE85)


def _threshold(p):
    """An element stays where its 32-bit word is not below this."""
    return min(2 ** 32 - 1, int(round(p * 2.0 ** 32)))


def _plain_words(numbers, count):
    """The first ``count`` elements' words, as int64."""
    low = 0xFFFFFFFF
    i = torch.arange(-(-count // 4), device=numbers.device)
    c = [i & low, i >> 32, (numbers[1] & low).expand_as(i), ((numbers[1] >> 32) & low).expand_as(i)]
    key = [numbers[0] & low, (numbers[0] >> 32) & low]

    def product(m, b):  # (high, low) 32 bits of m * b
        high = (m * (b >> 16) + ((m * (b & 0xFFFF)) >> 16)) >> 16
        return high, (m * b) & low

    for _ in range(10):
        h0, l0 = product(PHILOX_M[0], c[0])
        h1, l1 = product(PHILOX_M[1], c[2])
        c = [h1 ^ c[1] ^ key[0], l1, h0 ^ c[3] ^ key[1], l0]
        key = [(k + w) & low for k, w in zip(key, PHILOX_W)]
    return torch.stack(c, 1).flatten()[:count]


def _plain_dropout(s):
    p = s.case["p"]
    kept = (_plain_words(s.numbers, s.x.numel()) >= _threshold(p)).view(s.x.shape)
    drop = lambda t: torch.where(kept, t.detach().float() * (1.0 / (1.0 - p)), 0.0)  # noqa: E731
    y = drop(s.x)
    if s.res is not None:
        y = s.res.detach().float() + y
    out = [y.to(s.x.dtype)]
    if s.case["train"]:
        out.append(drop(s.dy).to(s.x.dtype))
        if s.res is not None:
            out.append(s.dy)
    return out


# ------------------------------------------------------------------ the framework's operators


def _own_qk(s):
    from sparsetriton_amd.nn.functional import sparse_qk_norm_rotary
    out = list(sparse_qk_norm_rotary(s.q, s.k, s.pos, s.rotary, s.wq, s.wk, eps=EPS))
    return out + list(torch.autograd.grad(out, [s.q, s.k, s.wq, s.wk], [s.dq, s.dk])) if s.case["train"] else out


def _own_window(s):
    from sparsetriton_amd.nn.functional import sparse_attention
    c = s.case
    out = sparse_attention(s.q, s.k, s.v, s.segments, causal=c["causal"], key_mask=s.mask, window=c["window"], sinks=c["sinks"])
    return [out] + list(torch.autograd.grad(out, [s.q, s.k, s.v], s.do)) if c["train"] else [out]


def _own_dropout(s):
    from sparsetriton_amd.nn.functional import sparse_dropout
    out = sparse_dropout(s.x, s.case["p"], residual=s.res, numbers=s.numbers)
    if not s.case["train"]:
        return [out]
    return [out] + list(torch.autograd.grad(out, [s.x] + ([s.res] if s.res is not None else []), s.dy))


def run(state):
    op = state.case["op"]
    if own:
        return _own_qk(state) if op == "qk" else _own_window(state) if op == "window" else _own_dropout(state)
    return _plain_qk(state) if op == "qk" else _plain_window(state) if op == "window" else _plain_dropout(state)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    e = ESZ[case["dtype"]]
    if case["op"] == "qk":
        size = case["n"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        where = 2 * case["n"] * len(_axes(case))
        # forward: q and k in and out; backward: the inputs and the outputs' gradients in, the inputs' gradients out
        return {"bytes": 2 * size * e + where + ((3 * size * e + where) if case["train"] else 0),
                "flops": size * (7 + (14 if case["train"] else 0))}
    if case["op"] == "dropout":
        size, r = case["n"] * case["c"], case["residual"]
        return {"bytes": size * e * ((3 if r else 2) + (2 if case["train"] else 0)),
                "flops": size * ((2 if r else 1) + (1 if case["train"] else 0))}
    ql, kl = _lengths(case)
    h, hk, d, keys = case["heads"], case["kv_heads"], case["dim"], 0
    for nq, nk in zip(ql, kl):  # the keys that any query sees
        lo, hi = _reach(case, nq, nk, 0, nq)
        keys += hi - lo + (min(case["sinks"], lo) if lo < hi else min(case["sinks"], nk) * (not case["causal"]))
    qb, kb = sum(ql) * h * d * e, keys * hk * d * e
    if not case["train"]:
        return {"bytes": 2 * qb + 2 * kb, "flops": 4 * _pairs(case) * h * d}
    # q, k, v and o once more and the output's gradient in, three gradients out
    return {"bytes": (2 + 4) * qb + (2 + 2) * kb + 2 * sum(kl) * hk * d * e, "flops": 14 * _pairs(case) * h * d}


# ------------------------------------------------------------------ the definitions in 64 bits


def _exact_qk(s):
    angle = torch.stack([s.pos[:, int(a)].double() * s.freq[p].double() for p, a in enumerate(s.axis.tolist())], 1)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), angle)
    p = s.freq.numel()
    even = torch.arange(p, device="cuda") * 2 if s.case["interleaved"] else torch.arange(p, device="cuda")
    odd = even + (1 if s.case["interleaved"] else p)

    def at(x, z):  # each pair as a complex number, turned by exp(i angle)
        x = x.clone()
        t = torch.complex(x[..., even], x[..., odd]) * z[:, None]
        x[..., even], x[..., odd] = t.real, t.imag
        return x

    outs, grads, weights = [], [], []
    for x, w, dy in ((s.q, s.wq, s.dq), (s.k, s.wk, s.dk)):
        x, w, dy = x.detach().double(), w.detach().double(), dy.double()
        size = torch.sqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / x.shape[-1] + EPS)
        outs.append(at(x * w / size, turn))
        if s.case["train"]:
            g = at(dy, turn.conj())
            # d (x / size) / dx = (1 - x x^T / (D size^2)) / size
            weights.append(torch.einsum("nhd,nhd->d", g, x / size))
            along = torch.einsum("nhd,nhd->nh", g * w, x)[..., None]
            grads.append((g * w - x * along / (x.shape[-1] * size ** 2)) / size)
    return outs + grads + weights


def _exact_window(s):
    c, scale = s.case, s.case["dim"] ** -0.5
    r = c["heads"] // c["kv_heads"]
    q, k, v, do = (t.detach().double().transpose(0, 1).contiguous() for t in (s.q, s.k, s.v, s.do))
    o, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    q0 = k0 = 0
    for nq, nk in zip(*s.lengths):
        Q, K = slice(q0, q0 + nq), slice(k0, k0 + nk)
        away = torch.arange(nk, device="cuda")[None] - (torch.arange(nq, device="cuda") + (nk - nq))[:, None]
        drop = away <= -c["window"]
        if not c["causal"]:
            drop |= away >= c["window"]
        drop[:, :c["sinks"]] = False
        if c["causal"]:
            drop |= away > 0
        if s.mask is not None:
            drop |= ~s.mask[K]
        none = drop.all(1, keepdim=True)
        del away
        for h in range(c["heads"]):
            kh, vh = k[h // r, K], v[h // r, K]
            p = torch.softmax((q[h, Q] @ kh.T * scale).masked_fill_(drop, -math.inf), -1).masked_fill_(none, 0.0)
            o[h, Q] = p @ vh
            if c["train"]:
                dz = do[h, Q] @ vh.T
                dz -= (p * dz).sum(-1, keepdim=True)
                dz *= p * scale
                dq[h, Q] = dz @ kh
                dk[h // r, K] += dz.T @ q[h, Q]
                dv[h // r, K] += p.T @ do[h, Q]
        q0, k0 = q0 + nq, k0 + nk
    return [t.transpose(0, 1) for t in [o] + ([dq, dk, dv] if c["train"] else [])]


def _exact_kept(numbers, count, p):
    """Which elements stay, by 64-bit arithmetic on the host, some counters at a time."""
    key, call = (np.uint64(int(x)) for x in numbers.tolist())
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    kept = np.empty((-(-count // 4), 4), dtype=bool)
    for b in range(0, kept.shape[0], 1 << 16):
        e = min(kept.shape[0], b + (1 << 16))
        x0 = np.arange(b, e, dtype=np.uint64)
        x1, x0 = x0 >> half, x0 & low
        x2, x3 = np.full_like(x0, call & low), np.full_like(x0, call >> half)
        k0, k1 = key & low, key >> half
        for _ in range(10):
            a, c = np.uint64(PHILOX_M[0]) * x0, np.uint64(PHILOX_M[1]) * x2
            x0, x1, x2, x3 = (c >> half) ^ x1 ^ k0, c & low, (a >> half) ^ x3 ^ k1, a & low
            k0, k1 = (k0 + np.uint64(PHILOX_W[0])) & low, (k1 + np.uint64(PHILOX_W[1])) & low
        for j, x in enumerate((x0, x1, x2, x3)):
            kept[b:e, j] = x >= np.uint64(_threshold(p))
    return torch.from_numpy(kept.reshape(-1)[:count])


def _exact_dropout(s):
    p = s.case["p"]
    by = _exact_kept(s.numbers, s.x.numel(), p).to("cuda").view(s.x.shape).double() / (1.0 - p)
    y = s.x.detach().double() * by
    out = [y if s.res is None else y + s.res.detach().double()]
    if s.case["train"]:
        out += [s.dy.double() * by] + ([s.dy.double()] if s.res is not None else [])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "qk":
        return _exact_qk(s)
    return _exact_window(s) if case["op"] == "window" else _exact_dropout(s)
