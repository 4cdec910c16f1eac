"""Norms of heads with their rotation, and rows in pages, from their formulas
in 64 bits on the CPU, with the size of what is added up to each element."""
import numpy as np
import torch

import ops_oracle as OO


def heads_normed(x, w, kind, eps):
    """(u, z, inv, size of u, size of z) of x [rows][heads][maps][dim] in float64."""
    if kind == "none":
        return x, x, None, x.abs(), x.abs()
    t, size = x, x.abs()
    if kind == "layer":
        t, size = x - x.mean(-1, keepdim=True), x.abs() + x.abs().mean(-1, keepdim=True)
    inv = 1 / torch.sqrt((t * t).mean(-1, keepdim=True) + eps)
    w = torch.ones(x.shape[-1]).double() if w is None else w.double()
    return t * inv, t * inv * w, inv, size * inv, size * inv * w.abs()


def turned(x, theta, interleaved):
    """OO.turned of [rows][heads][maps][dim]."""
    y, size = OO.turned(x.flatten(1, 2), theta, interleaved)
    return y.view(x.shape), size.view(x.shape)


def pair_slices(pairs, interleaved):
    i = torch.arange(pairs)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)


def forward(x, w, theta, kind, eps, interleaved):
    """(y, size): the result and the size of its terms."""
    _, z, _, _, size = heads_normed(x.double(), w, kind, eps)
    return turned(z, theta, interleaved)[0], turned(size, theta, interleaved)[1]


def backward(x, w, dy, theta, freq, axis, axes, kind, eps, interleaved):
    """(dx, dw, dpositions), each with its size."""
    x, dy = x.double(), dy.double()
    u, z, inv, su, sz = heads_normed(x, w, kind, eps)
    dz, sd = turned(dy, -theta, interleaved)[0], turned(dy.abs(), theta, interleaved)[1]
    one = torch.ones(x.shape[-1]).double() if w is None else w.double()
    g, sg = dz * one, sd * one.abs()
    dx = g - u * (g * u).mean(-1, keepdim=True)
    sx = sg + su * (sg * su).mean(-1, keepdim=True)
    if kind == "layer":
        dx, sx = dx - g.mean(-1, keepdim=True), sx + sg.mean(-1, keepdim=True)
    a, b = pair_slices(theta.shape[1], interleaved)
    t = (dz[..., b] * z[..., a] - dz[..., a] * z[..., b]).sum((1, 2)) * freq
    st = (sd[..., b] * sz[..., a] + sd[..., a] * sz[..., b]).sum((1, 2)) * freq
    dpos, sp = torch.zeros(len(x), axes).double(), torch.zeros(len(x), axes).double()
    dpos.index_add_(1, axis.long(), t)
    sp.index_add_(1, axis.long(), st.abs())
    return (dx * inv, sx * inv), ((dz * u).sum((0, 1, 2)), (sd * su).sum((0, 1, 2))), (dpos, sp)


def pool(g, lengths, page, kv, dim, dtype, width=None, extra=3, fill=float("nan")):
    """A cache of sequences of so many rows in pages in any order: a dict of
    k_pages, v_pages (rows beyond a length, and pages of none, hold `fill`),
    table, and the rows k, v themselves, one sequence after the other."""
    n = np.asarray(lengths)
    each = -(-n // page)
    width = int(each.max(initial=0)) + 1 if width is None else width
    total = int(each.sum()) + extra
    order = torch.randperm(total, generator=g).tolist()
    k = torch.randn((int(n.sum()), kv, 2, dim), generator=g).to(dtype)
    v = torch.randn((int(n.sum()), kv, 2 * dim), generator=g).to(dtype)
    k_pages = torch.full((total, page, kv, 2, dim), fill, dtype=dtype)
    v_pages = torch.full((total, page, kv, 2 * dim), fill, dtype=dtype)
    table = torch.full((len(n), width), -7, dtype=torch.int32)
    row = 0
    for i, m in enumerate(n):
        for p in range(int(each[i])):
            at, c = order.pop(), min(page, int(m) - p * page)
            table[i, p] = at
            k_pages[at, :c], v_pages[at, :c] = k[row:row + c], v[row:row + c]
            row += c
    return dict(k_pages=k_pages, v_pages=v_pages, table=table, k=k, v=v)
