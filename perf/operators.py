"""Performance cases of the operators on device tensors: rotary positions with several axes, differential
attention over ragged batches and over a cache, and the norms around a block with its gate and residual scale.

A case is a plain dict; `op` names the call:

  rotary        rotate the heads of every row by its position on several axes
  rotary_grad   its backward pass, with the gradient of the positions
  attend        differential attention of a ragged batch, forward only
  attend_train  the same, forward and backward
  attend_cache  one new row per sequence against a cache of earlier ones
  norm          block output normed, gated and added to the residual, and the sum normed for the next block
  norm_train    the same, forward and backward

`own` false computes the plain form (elementary torch operations in 32 bits); true calls mtpx.ops.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6


# ---- cases -------------------------------------------------------------------


def _attend(name, op, dtype, rows, seqs, heads, kv_heads, dim, causal=False, masked=0.0):
    c = dict(op=op, dtype=dtype, rows=rows, seqs=seqs, heads=heads, kv_heads=kv_heads, dim=dim, causal=causal, masked=masked)
    return dict(c, name=name) if name else c


def _cache(name, dtype, seqs, capacity, heads, kv_heads, dim):
    c = dict(op="attend_cache", dtype=dtype, seqs=seqs, capacity=capacity, heads=heads, kv_heads=kv_heads, dim=dim)
    return dict(c, name=name) if name else c


def _rotary(name, op, dtype, rows, heads, dim, rotated, coordinates, interleaved=False):
    c = dict(op=op, dtype=dtype, rows=rows, heads=heads, dim=dim, rotated=rotated, coordinates=coordinates, interleaved=interleaved)
    return dict(c, name=name) if name else c


def _norm(name, op, dtype, rows, width, kind, act, per_row_gate):
    c = dict(op=op, dtype=dtype, rows=rows, width=width, kind=kind, act=act, per_row_gate=per_row_gate)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a Monte-Carlo move: one atom against the 997 of its cell, the shortest call, where latency counts
        _cache("cache_1x997", "bf16", 1, 997, 8, 8, 32),
        # serving: 64 sequences of different lengths, heads sharing keys and values
        _cache("cache_64x8192_shared", "bf16", 64, 8192, 32, 4, 64),
        # a training step in 32 bits over a screening set of small structures, some atoms masked
        _attend("train_f32_200x84", "attend_train", "f32", 16800, 200, 8, 8, 32, masked=0.1),
        # a training step over the benchmark's training batch: 1,000 structures of about 160 atoms
        _attend("train_bf16_1000x160", "attend_train", "bf16", 160000, 1000, 8, 8, 64),
        # a training step over long ordered sequences with shared heads
        _attend("train_bf16_causal_8192", "attend_train", "bf16", 16384, 2, 16, 4, 64, causal=True),
        # evaluation of the benchmark's 32,000-atom cell: the largest map
        _attend("attend_bf16_32000", "attend", "bf16", 32000, 1, 8, 8, 64),
        # one row's queries and keys: latency
        _rotary("rotary_1x32", "rotary", "bf16", 1, 32, 64, 64, False),
        # queries and keys of the benchmark's training batch, by integer positions on three axes
        _rotary("rotary_160000x32", "rotary", "bf16", 160000, 32, 64, 64, False),
        # backward in 32 bits with forces: gradient of the coordinates, part of each head rotated
        _rotary("rotary_grad_f32_16801x32", "rotary_grad", "f32", 16801, 32, 40, 36, True, interleaved=True),
        # a serving step's residual glue: few rows
        _norm("norm_64x4096", "norm", "bf16", 64, 4096, "rms", "none", False),
        # an odd-sized structure in 32 bits, trained, a gate per row
        _norm("norm_train_f32_4001x1000", "norm_train", "f32", 4001, 1000, "layer", "sigmoid", True),
        # the training batch's rows at an ordinary width
        _norm("norm_train_bf16_160000x1024", "norm_train", "bf16", 160000, 1024, "rms", "tanh", False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend_train", "attend_train", "attend_cache", "attend_cache", "rotary", "rotary_grad", "norm", "norm_train"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 1, 2, 4, 8])
    dim = rng.choice([16, 32, 40, 64, 64, 96, 128])
    if kind in ("attend", "attend_train"):
        heads = min(16, kv_heads * group)
        kv_heads = min(kv_heads, heads)
        rows = _log_int(rng, 50, 60000)
        seqs = max(_log_int(rng, 1, 400), -(-rows // 6000))
        seqs = min(seqs, rows)
        # a drawn case costs no more than the largest listed one, also in 32 bits
        while rows * rows / seqs * heads * dim > 1.5e10:
            rows = rows * 2 // 3
        return _attend("", kind, dtype, rows, min(seqs, rows), heads, kv_heads, dim, rng.random() < 0.4, rng.choice([0.0, 0.0, 0.15]))
    if kind == "attend_cache":
        seqs, capacity = _log_int(rng, 1, 128), _log_int(rng, 30, 20000)
        while seqs * capacity * kv_heads * dim > 1.3e8:
            capacity = capacity * 2 // 3
        return _cache("", dtype, seqs, capacity, kv_heads * group, kv_heads, dim)
    if kind in ("rotary", "rotary_grad"):
        heads = rng.choice([4, 8, 20, 32])
        rows = _log_int(rng, 1, 100000)
        rotated = dim if rng.random() < 0.6 else dim - 4
        coordinates = True if kind == "rotary_grad" or dtype == "f32" else rng.random() < 0.5
        while rows * heads * dim > 2.0e8:
            rows = rows * 2 // 3
        return _rotary("", kind, dtype, rows, heads, dim, rotated, coordinates, rng.random() < 0.5)
    width = rng.choice([_log_int(rng, 64, 8192), 8 * _log_int(rng, 8, 1024)])
    rows = _log_int(rng, 1, 160000)
    while rows * width > 1.6e8:
        rows = rows * 2 // 3
    return _norm("", kind, dtype, rows, width, rng.choice(["rms", "layer"]), rng.choice(["none", "sigmoid", "tanh"]), rng.random() < 0.4)


def _lengths(case):
    """Rows of each sequence: of different sizes, summing to the case's rows."""
    rows, seqs = case["rows"], case["seqs"]
    w = np.random.RandomState(rows % 1000003 + seqs).uniform(0.25, 1.75, seqs) if seqs > 2 else np.ones(seqs)
    n = np.maximum(1, np.floor(w / w.sum() * rows)).astype(np.int64)
    while n.sum() > rows:
        n[n.argmax()] -= 1
    n[: rows - n.sum()] += 1
    return n


def _cache_lengths(case):
    """Valid rows of each cache: from half of the capacity up to all of it."""
    u = np.random.RandomState(case["capacity"] + case["seqs"]).uniform(0.5, 1.0, case["seqs"])
    n = np.maximum(1, np.round(u * case["capacity"])).astype(np.int64)
    n[0] = case["capacity"]
    return n


def work(case):
    op, size = case["op"], torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if op in ("attend", "attend_train"):
        n = _lengths(case).astype(float)
        pairs = float((n * (n + 1) / 2 if case["causal"] else n * n).sum())
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        q, kv = case["rows"] * h * 2 * d * size, case["rows"] * hk * 4 * d * size
        forward = dict(bytes=2 * q + kv, flops=8 * d * h * pairs)
        if op == "attend":
            return forward
        return dict(bytes=forward["bytes"] + 4 * q + 2 * kv, flops=forward["flops"] + 20 * d * h * pairs)
    if op == "attend_cache":
        n, h, hk, d = float(_cache_lengths(case).sum()), case["heads"], case["kv_heads"], case["dim"]
        return dict(bytes=(n * hk * 4 + case["seqs"] * h * 4) * d * size, flops=8 * d * h * n)
    if op in ("rotary", "rotary_grad"):
        e = case["rows"] * case["heads"] * case["dim"]
        if op == "rotary":
            return dict(bytes=2 * e * size + 12 * case["rows"], flops=3 * e)
        return dict(bytes=3 * e * size + 24 * case["rows"], flops=5 * e)
    e = case["rows"] * case["width"]
    g = 1 if case["per_row_gate"] else 0
    if op == "norm":
        return dict(bytes=(4 + g) * e * size, flops=12 * e)
    return dict(bytes=(4 + g + 6 + 2 * g) * e * size, flops=45 * e)


# ---- inputs ------------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _inputs(case, seed):
    g, dt, op = _gen(seed), DTYPES[case["dtype"]], case["op"]
    s = dict(case=case)
    if op in ("attend", "attend_train"):
        n, rows = _lengths(case), case["rows"]
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        s["offsets"] = np.concatenate([[0], np.cumsum(n)]).astype(np.int64)
        # the projections of a block, normed, with queries sharpened as trained ones are
        s["q"] = _randn(g, (rows, h, 2, d), dt, 1.7)
        s["k"] = _randn(g, (rows, hk, 2, d), dt)
        s["v"] = _randn(g, (rows, hk, 2 * d), dt)
        s["lam"] = 0.2 + 0.6 * torch.rand(h, generator=g, device="cuda")
        s["mask"] = None
        if case["masked"]:
            m = torch.rand(rows, generator=g, device="cuda") >= case["masked"]
            m[: int(n[0])] = False  # a structure whose atoms are all masked: rows without a key
            s["mask"] = m
        s["dout"] = _randn(g, (rows, h, 2 * d), dt) if op == "attend_train" else None
    elif op == "attend_cache":
        b, cap, h, hk, d = case["seqs"], case["capacity"], case["heads"], case["kv_heads"], case["dim"]
        s["q"] = _randn(g, (b, h, 2, d), dt, 1.7)
        s["k"] = _randn(g, (b, cap, hk, 2, d), dt)
        s["v"] = _randn(g, (b, cap, hk, 2 * d), dt)
        s["lam"] = 0.2 + 0.6 * torch.rand(h, generator=g, device="cuda")
        s["lengths"] = torch.from_numpy(_cache_lengths(case).astype(np.int32)).cuda()
    elif op in ("rotary", "rotary_grad"):
        rows, h, d, r = case["rows"], case["heads"], case["dim"], case["rotated"]
        s["x"] = _randn(g, (rows, h, d), dt)
        axis = np.arange(r // 2) % 3
        if case["coordinates"]:
            # fractional coordinates and whole numbers of turns over the cell
            s["positions"] = torch.rand((rows, 3), generator=g, device="cuda")
            freq = 2 * np.pi * (1 + np.arange(r // 2) // 3)
        else:
            # frames, lines and columns
            s["positions"] = torch.stack([torch.randint(0, m, (rows,), generator=g, device="cuda", dtype=torch.int32) for m in (512, 64, 96)], 1)
            freq = 10000.0 ** (-2.0 * np.arange(r // 2) / r)
        s["freq"] = torch.tensor(freq, dtype=torch.float32, device="cuda")
        s["axis"] = torch.tensor(axis, dtype=torch.int32, device="cuda")
        s["dy"] = _randn(g, (rows, h, d), dt) if op == "rotary_grad" else None
    else:
        rows, c = case["rows"], case["width"]
        s["x"] = _randn(g, (rows, c), dt, 2.0)
        s["y"] = _randn(g, (rows, c), dt, 0.7) + 0.1
        s["gate"] = _randn(g, (rows, c) if case["per_row_gate"] else (c,), dt, 0.5)
        s["w1"] = 1 + _randn(g, (c,), dt, 0.1)
        s["w2"] = 1 + _randn(g, (c,), dt, 0.1)
        s["scales"] = (0.9, 0.5)  # of the residual and of the block
        if op == "norm_train":
            s["ds"] = _randn(g, (rows, c), dt)
            s["dn"] = _randn(g, (rows, c), dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        path = os.path.abspath("imr-mlp_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        from mtpx import capi, ops

        s["ops"], s["ctx"] = ops, capi.Context(0)
        if case["op"] in ("attend", "attend_train"):
            s["seqs"] = ops.Sequences(s["ctx"], s["offsets"])
    return s


def run(s):
    return _run_own(s) if own else _PLAIN[s["case"]["op"]](s)


def _run_own(s):
    ops, ctx, case = s["ops"], s["ctx"], s["case"]
    op = case["op"]
    if op == "attend":
        return ops.diff_attention(ctx, s["q"], s["k"], s["v"], s["lam"], s["seqs"], causal=case["causal"], key_mask=s["mask"])
    if op == "attend_train":
        kw = dict(causal=case["causal"], key_mask=s["mask"])
        out, saved = ops.diff_attention(ctx, s["q"], s["k"], s["v"], s["lam"], s["seqs"], save=True, **kw)
        return (out, *ops.diff_attention_backward(ctx, s["dout"], s["q"], s["k"], s["v"], s["lam"], s["seqs"], out, saved, **kw))
    if op == "attend_cache":
        return ops.diff_attention_cache(ctx, s["q"], s["k"], s["v"], s["lam"], s["lengths"])
    if op == "rotary":
        return ops.rotary(ctx, s["x"], s["positions"], s["freq"], s["axis"], interleaved=case["interleaved"])
    if op == "rotary_grad":
        return ops.rotary_backward(ctx, s["dy"], s["positions"], s["freq"], s["axis"], interleaved=case["interleaved"], x=s["x"])
    kw = dict(kind=case["kind"], gate_act=case["act"], residual_scale=s["scales"][0], block_scale=s["scales"][1], eps=EPS)
    if op == "norm":
        return ops.norm_block(ctx, s["x"], s["y"], s["gate"], s["w1"], s["w2"], **kw)
    out, n, stats = ops.norm_block(ctx, s["x"], s["y"], s["gate"], s["w1"], s["w2"], save=True, **kw)
    return (out, n, *ops.norm_block_backward(ctx, s["ds"], s["dn"], s["x"], s["y"], s["gate"], s["w1"], s["w2"], stats, **kw))


# ---- plain forms ---------------------------------------------------------------


def _chunks(n, heads, causal):
    """Sequences that are computed together, padded to the longest: lists of indices, longest first."""
    order, out, i = np.argsort(-n), [], 0
    while i < len(order):
        m = int(n[order[i]])
        take = max(1, int(1.5e8 // (m * m * heads)))
        out.append(order[i : i + take])
        i += take
    return out


def _plain_attend(s):
    case = s["case"]
    train = s["dout"] is not None
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    off, n = s["offsets"], np.diff(s["offsets"])
    scale = d ** -0.5
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    out = torch.zeros((case["rows"], h, 2 * d), device="cuda")
    if train:
        dq, dk, dv, dlam = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros(h, device="cuda")
        dout = s["dout"].float()
    for ids in _chunks(n, h, case["causal"]):
        m = int(n[ids].max())
        at = torch.arange(m, device="cuda")
        first, count = torch.tensor(off[ids], device="cuda"), torch.tensor(n[ids], device="cuda")
        inside = at[None] < count[:, None]
        rows = torch.where(inside, first[:, None] + at[None], 0)
        seen = inside if s["mask"] is None else inside & s["mask"][rows]
        kept = rows[inside]
        # query rows at a time, so that a long sequence's maps fit
        step = max(1, min(m, int(3e8 // (m * len(ids)))))
        for head in range(h):
            g = head // (h // hk)
            kk, vv = k[rows, g].contiguous(), v[rows, g].contiguous()  # [b, m, 2, d], [b, m, 2 d]
            kt, vt = kk.permute(2, 0, 3, 1).contiguous(), vv.transpose(1, 2).contiguous()
            if train:
                dkk, dvv = torch.zeros_like(kk), torch.zeros_like(vv)
            for a in range(0, m, step):
                r, live = rows[:, a : a + step], inside[:, a : a + step]
                qq = q[r, head]  # [b, step, 2, d]
                see = seen[:, None, :] if not case["causal"] else seen[:, None, :] & (at[None, None, :] <= at[a : a + step][None, :, None])
                p = []
                for j in range(2):
                    x = torch.matmul(qq[:, :, j].contiguous(), kt[j]) * scale
                    x = torch.where(see, x, -math.inf)
                    top = x.amax(-1, keepdim=True)
                    x = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
                    total = x.sum(-1, keepdim=True)
                    p.append(x / torch.where(total == 0, 1.0, total))
                lam = s["lam"][head]
                both = p[0] - lam * p[1]
                out[r[live], head] = torch.matmul(both, vv)[live]
                if not train:
                    continue
                do = torch.where(live[:, :, None], dout[r, head], 0.0)
                dp = torch.matmul(do, vt)
                dvv += torch.matmul(both.transpose(1, 2).contiguous(), do)
                share = (p[1] * dp).sum(-1, keepdim=True)
                dlam[head] -= share.sum()
                for j in range(2):
                    delta = share if j else (p[0] * dp).sum(-1, keepdim=True)
                    ds = p[j] * (dp - delta) * (scale * (-lam if j else 1.0))
                    dq[r[live], head, j] = torch.matmul(ds, kk[:, :, j].contiguous())[live]
                    dkk[:, :, j] += torch.matmul(ds.transpose(1, 2).contiguous(), qq[:, :, j].contiguous())
            if train:
                dk[kept, g] += dkk[inside]
                dv[kept, g] += dvv[inside]
    dt = DTYPES[case["dtype"]]
    if not train:
        return out.to(dt)
    return out.to(dt), dq.to(dt), dk.to(dt), dv.to(dt), dlam


def _plain_cache(s):
    case = s["case"]
    h, hk, d, b = case["heads"], case["kv_heads"], case["dim"], case["seqs"]
    group = h // hk
    at = torch.arange(case["capacity"], device="cuda")
    out = torch.empty((b, h, 2 * d), device="cuda")
    step = max(1, int(1e8 // (case["capacity"] * hk * 2 * d)))
    for a in range(0, b, step):
        z = slice(a, a + step)
        see = at[None] < s["lengths"][z, None]
        q = s["q"][z].float().view(-1, hk, group, 2, d).permute(0, 1, 3, 2, 4)  # [b, hk, 2, group, d]
        k = s["k"][z].float().permute(0, 2, 3, 4, 1).contiguous()  # [b, hk, 2, d, n]
        v = torch.where(see[:, :, None, None], s["v"][z].float(), 0.0).permute(0, 2, 1, 3).contiguous()
        x = torch.matmul(q.contiguous(), k) * d ** -0.5
        x = torch.where(see[:, None, None, None, :], x, -math.inf)
        x = torch.exp(x - x.amax(-1, keepdim=True))
        p = x / x.sum(-1, keepdim=True)
        lam = s["lam"].view(1, hk, group, 1)
        out[z] = torch.matmul(p[:, :, 0] - lam * p[:, :, 1], v).reshape(-1, h, 2 * d)
    return out.to(DTYPES[case["dtype"]])


def _pairs(x, r, interleaved):
    return (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., : r // 2], x[..., r // 2 : r])


def _unpair(a, b, rest, interleaved):
    both = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([both, rest], -1)


def _plain_rotary(s):
    case = s["case"]
    r, inter = case["rotated"], case["interleaved"]
    angle = s["positions"].float()[:, s["axis"].long()] * s["freq"]
    c, sn = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    back = s["dy"] is not None
    x = (s["dy"] if back else s["x"]).float()
    a, b = _pairs(x, r, inter)
    if back:
        sn = -sn
    a, b = a * c - b * sn, a * sn + b * c
    y = _unpair(a, b, x[..., r:], inter).to(DTYPES[case["dtype"]])
    if not back:
        return y
    x1, x2 = _pairs(s["x"].float(), r, inter)
    t = ((b * x1 - a * x2).sum(1)) * s["freq"]
    dpos = torch.zeros_like(s["positions"])
    for k in range(3):
        dpos[:, k] = t[:, s["axis"] == k].sum(-1)
    return y, dpos


def _act(kind, g):
    """The gate's activation and its derivative."""
    if kind == "sigmoid":
        a = 1 / (1 + torch.exp(-g))
        return a, a * (1 - a)
    if kind == "tanh":
        a = torch.tanh(g)
        return a, 1 - a * a
    return g, torch.ones_like(g)


def _plain_norm(s):
    case = s["case"]
    alpha, beta = s["scales"]
    center = case["kind"] == "layer"
    dt = DTYPES[case["dtype"]]
    x, y, g, w1, w2 = (s[t].float() for t in ("x", "y", "gate", "w1", "w2"))

    def normed(t):
        if center:
            t = t - t.mean(-1, keepdim=True)
        r = 1 / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS)
        return t * r, r

    def back(d, u, r):
        d = d - u * (d * u).mean(-1, keepdim=True) - (d.mean(-1, keepdim=True) if center else 0.0)
        return r * d

    u, r1 = normed(y)
    a, da = _act(case["act"], g)
    z = u * w1
    t = alpha * x + beta * a * z
    v, r2 = normed(t)
    out, n = t.to(dt), (v * w2).to(dt)
    if case["op"] == "norm":
        return out, n
    ds, dn = s["ds"].float(), s["dn"].float()
    dw2 = (dn * v).sum(0)
    ds = ds + back(dn * w2, v, r2)
    dg = beta * da * z * ds
    if g.dim() == 1:
        dg = dg.sum(0)
    dz = beta * a * ds
    dw1 = (dz * u).sum(0)
    dy = back(dz * w1, u, r1)
    return out, n, (alpha * ds).to(dt), dy.to(dt), dg.to(dt), dw1.to(dt), dw2.to(dt)


_PLAIN = {"attend": _plain_attend, "attend_train": _plain_attend, "attend_cache": _plain_cache, "rotary": _plain_rotary,
          "rotary_grad": _plain_rotary, "norm": _plain_norm, "norm_train": _plain_norm}


# ---- the definitions in 64 bits ---------------------------------------------------


def _softmax64(x, see):
    x = x.masked_fill(~see, -math.inf)
    empty = ~see.any(-1, keepdim=True)
    return torch.softmax(x.masked_fill(empty, 0.0), -1).masked_fill(empty, 0.0)


def _attend64(case, q, k, v, lam, mask, head, a):
    """Query rows a.. of one head of a sequence; q, k, v are the sequence's."""
    kv = head // (case["heads"] // case["kv_heads"])
    see = torch.ones((len(q), len(k)), dtype=torch.bool, device="cuda")
    if mask is not None:
        see &= mask[None]
    if case["causal"]:
        see &= torch.arange(len(k), device="cuda")[None] <= torch.arange(a, a + len(q), device="cuda")[:, None]
    p1 = _softmax64(q[:, head, 0] @ k[:, kv, 0].T / math.sqrt(case["dim"]), see)
    p2 = _softmax64(q[:, head, 1] @ k[:, kv, 1].T / math.sqrt(case["dim"]), see)
    return (p1 - lam[head] * p2) @ v[:, kv]


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op in ("attend", "attend_train"):
        train, off = op == "attend_train", s["offsets"]
        n = np.diff(off).astype(float)
        # about 20 seconds: 64-bit products of 30 Tflop/s, and launches per sequence and head
        if float((n * n).sum()) * case["heads"] * case["dim"] * (40 if train else 8) > 2e14 or case["seqs"] * case["heads"] > 12000:
            return None
        outs, grads = [], []
        lam = s["lam"].double().requires_grad_(train)
        for i in range(case["seqs"]):
            z = slice(int(off[i]), int(off[i + 1]))
            q, k, v = (s[t][z].double().requires_grad_(train) for t in "qkv")
            mask = None if s["mask"] is None else s["mask"][z]
            out = torch.empty((len(q), case["heads"], 2 * case["dim"]), dtype=torch.float64, device="cuda")
            step = len(q) if train else 4000
            for head in range(case["heads"]):
                for a in range(0, len(q), step):
                    o = _attend64(case, q[a : a + step], k, v, lam, mask, head, a)
                    out[a : a + step, head] = o.detach()
                    if train:
                        (o * s["dout"][z][:, head].double()).sum().backward()
            outs.append(out)
            grads.append((q.grad, k.grad, v.grad))
        if not train:
            return torch.cat(outs)
        return (torch.cat(outs), *(torch.cat([g[j] for g in grads]) for j in range(3)), lam.grad)
    if op == "attend_cache":
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        out = torch.empty((case["seqs"], h, 2 * d), dtype=torch.float64, device="cuda")
        for i, m in enumerate(_cache_lengths(case)):
            k, v = s["k"][i, :m].double(), s["v"][i, :m].double()
            for head in range(h):
                kv = head // (h // hk)
                p = [torch.softmax(k[:, kv, j] @ s["q"][i, head, j].double() / math.sqrt(d), 0) for j in range(2)]
                out[i, head] = (p[0] - s["lam"][head].double() * p[1]) @ v[:, kv]
        return out
    if op in ("rotary", "rotary_grad"):
        r, back = case["rotated"], op == "rotary_grad"
        x = s["x"].double()

        turn = lambda t: t[:, s["axis"].long()] * s["freq"].double()  # noqa: E731
        first = slice(0, r, 2) if case["interleaved"] else slice(0, r // 2)
        second = slice(1, r, 2) if case["interleaved"] else slice(r // 2, r)
        if not back:
            y = x.clone()
            angle = turn(s["positions"].double())
            w = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.ones_like(angle), angle)[:, None]
            y[..., first], y[..., second] = w.real, w.imag
            return y
        # the gradient of sum(y dy) by the chain rule of the rotation, a part of the rows at a time
        dx, dpos = [], []
        for a in range(0, case["rows"], 20000):
            z = slice(a, a + 20000)
            xx = x[z].clone().requires_grad_(True)
            pp = s["positions"][z].double().requires_grad_(True)
            c, sn = turn(pp).cos()[:, None], turn(pp).sin()[:, None]
            dy = s["dy"][z].double()
            l = ((xx[..., first] * c - xx[..., second] * sn) * dy[..., first]).sum() + ((xx[..., first] * sn + xx[..., second] * c) * dy[..., second]).sum()
            l = l + (xx[..., r:] * dy[..., r:]).sum()
            l.backward()
            dx.append(xx.grad)
            dpos.append(pp.grad)
        return torch.cat(dx), torch.cat(dpos)
    train = op == "norm_train"
    alpha, beta = s["scales"]
    leaf = [s[t].double().requires_grad_(train) for t in ("gate", "w1", "w2")]
    outs, grads = [], []

    def norm64(t, w):
        if case["kind"] == "layer":
            t = t - t.mean(-1, keepdim=True)
        return t / torch.sqrt(t.pow(2).mean(-1, keepdim=True) + EPS) * w

    step = max(1, int(2e7 // case["width"]))
    for a in range(0, case["rows"], step):
        z = slice(a, a + step)
        x, y = (s[t][z].double().requires_grad_(train) for t in ("x", "y"))
        g = leaf[0][z] if case["per_row_gate"] else leaf[0]
        g = {"none": lambda t: t, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[case["act"]](g)
        t = alpha * x + beta * g * norm64(y, leaf[1])
        n = norm64(t, leaf[2])
        outs.append((t.detach(), n.detach()))
        if train:
            ((t * s["ds"][z].double()).sum() + (n * s["dn"][z].double()).sum()).backward()
            grads.append((x.grad, y.grad))
    out = tuple(torch.cat([o[j] for o in outs]) for j in range(2))
    if not train:
        return out
    return (*out, *(torch.cat([o[j] for o in grads]) for j in range(2)), *(t.grad for t in leaf))
