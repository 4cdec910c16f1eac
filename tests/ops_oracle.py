"""The operators on device tensors from their formulas, in 64 bits on the CPU,
with the size of what is added up to each element: a bound on an element's
error is a small multiple of a type's rounding times that size."""
import math

import torch

#: Largest relative error of one rounding to the type.
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
F32 = 2.0 ** -24


def turned(x, theta, interleaved):
    """x [rows][heads][dim] in float64 turned by theta [rows][pairs], and the
    size of each element's terms."""
    r = 2 * theta.shape[1]
    i = torch.arange(r // 2)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
    c, s = theta.cos()[:, None], theta.sin()[:, None]
    y, size = x.clone(), x.abs()
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., first] * s + x[..., second] * c
    both = x[..., first].abs() + x[..., second].abs()
    size = size.clone()
    size[..., first] = both
    size[..., second] = both
    return y, size


def attention(q, k, v, lam, scale, q_off, k_off, causal=False, mask=None, dout=None):
    """float64 results of differential attention: a dict of out, lse, (dq, dk,
    dv, dlam with dout) and of sizes `|...|` for their bounds."""
    rows, heads, _, d = q.shape
    kv = k.shape[1]
    r = dict(out=torch.zeros(rows, heads, 2 * d).double(),
             lse=torch.full((2, heads, rows), -math.inf).double(), scores=0.0)
    r["|out|"] = torch.zeros_like(r["out"])
    if dout is not None:
        for n, t in (("dq", q), ("dk", k), ("dv", v)):
            r[n], r["|%s|" % n] = torch.zeros_like(t), torch.zeros_like(t)
        r["dlam"], r["|dlam|"] = torch.zeros(heads).double(), torch.zeros(heads).double()
    for i in range(len(q_off) - 1):
        a, b = slice(q_off[i], q_off[i + 1]), slice(k_off[i], k_off[i + 1])
        nq, nk = a.stop - a.start, b.stop - b.start
        see = torch.ones(nq, nk, dtype=torch.bool)
        if mask is not None:
            see &= mask[b][None]
        if causal:
            see &= torch.arange(nk)[None] <= torch.arange(nq)[:, None] + nk - nq
        live = see.any(1)
        seen = see.any(0)  # a key that no row sees does not matter, NaN included
        for h in range(heads):
            g = h // (heads // kv)
            kk = torch.where(seen[:, None, None], k[b, g], 0.0)
            vv = torch.where(seen[:, None], v[b, g], 0.0)
            p = []
            for m in range(2):
                s = (q[a, h, m] @ kk[:, m].T) * scale
                r["scores"] = max(r["scores"], float(s[see].abs().max()) if see.any() else 0.0)
                s = s.masked_fill(~see, -math.inf)
                top = s.amax(1, keepdim=True).clamp_min(-1e300) if nk else torch.zeros(nq, 1).double()
                e = torch.where(see, torch.exp(s - top), 0.0)
                total = e.sum(1, keepdim=True)
                p.append(torch.where(live[:, None], e / total.clamp_min(1e-300), 0.0))
                r["lse"][m, h, a] = torch.where(live, (top + total.log())[:, 0], -math.inf)
            both = p[0] - lam[h] * p[1]
            apart = p[0] + lam[h].abs() * p[1]
            r["out"][a, h] = both @ vv
            r["|out|"][a, h] = apart @ vv.abs()
            if dout is None:
                continue
            do = dout[a, h]
            dp = do @ vv.T
            o = [p[m] @ vv for m in range(2)]
            dv = r["dv"], r["|dv|"]
            dv[0][b, g] += both.T @ do
            dv[1][b, g] += apart.T @ do.abs()
            share = (do * o[1]).sum(1, keepdim=True)
            r["dlam"][h] -= share.sum()
            r["|dlam|"][h] += (p[1] * (do.abs() @ vv.abs().T)).sum()
            # what roundings of out and of P_1 V leave in D_0 and D_1
            off1 = (do.abs() * o[1].abs()).sum(1, keepdim=True)
            off0 = (do.abs() * r["out"][a, h].abs()).sum(1, keepdim=True) + lam[h].abs() * off1
            for m in range(2):
                w = -lam[h] if m else 1.0
                ds = w * p[m] * (dp - (p[m] * dp).sum(1, keepdim=True))
                size = ds.abs() + abs(w) * p[m] * (off1 if m else off0)
                r["dq"][a, h, m] = scale * (ds @ kk[:, m])
                r["|dq|"][a, h, m] = scale * (size @ kk[:, m].abs())
                r["dk"][b, g, m] += scale * (ds.T @ q[a, h, m])
                r["|dk|"][b, g, m] += scale * (size.T @ q[a, h, m].abs())
    return r


def act(kind, g):
    return {"none": lambda t: t, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[kind](g)


def normed(t, kind, eps):
    if kind == "layer":
        t = t - t.mean(1, keepdim=True)
    return t / torch.sqrt((t * t).mean(1, keepdim=True) + eps)


def norm_block(x, y, gate, w1, w2, kind, gate_act, alpha, beta, eps):
    """(s, n) in the tensors' own precision, differentiable."""
    z = normed(y, kind, eps)
    if w1 is not None:
        z = z * w1
    if gate is not None:
        z = z * act(gate_act, gate)
    s = beta * z if x is None else alpha * x + beta * z
    n = normed(s, kind, eps)
    return s, n if w2 is None else n * w2
