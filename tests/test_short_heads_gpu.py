"""Norms of heads and appends of more rows than a lane a row fills the device with:
heads so short that one lane has a vector, and a row."""
import pytest
import torch

import ops_oracle as OO
import paged_oracle as PO
from mtpx import ops

pytestmark = pytest.mark.gpu

ROWS = (1 << 21) + 5  # (a lane a row from 2^21 on)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype,dim,interleaved,heads,kv", [
    (torch.float32, 2, False, 0, 1), (torch.bfloat16, 16, False, 1, 1), (torch.float16, 8, True, 1, 2)])
@pytest.mark.parametrize("ends", [(3, ROWS - 2), (0, 5, 5, 40001, 40002, ROWS)])
def test_append(ctx, dtype, dim, interleaved, heads, kv, ends):
    """Few and several sequences, rows of none: every key turned, within its rounding
    and that of cos, sin and the products in 32 bits, every value as it was."""
    g = torch.Generator(device="cuda").manual_seed(dim)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    k, v = randn(ROWS, kv, 2, dim), randn(ROWS, kv, 2 * dim)
    q = randn(ROWS, heads, 2, dim) if heads else None
    pos = torch.arange(ROWS, device="cuda")[:, None]
    freq, axis = torch.rand(dim // 2, generator=g, device="cuda"), torch.zeros(dim // 2, dtype=torch.int32, device="cuda")
    new = [b - a for a, b in zip(ends, ends[1:])]
    page = 1024
    each = [-(-n // page) for n in new]
    table, at = torch.full((len(new), max(each)), -1, dtype=torch.int32), 0
    for i, n in enumerate(each):
        table[i, :n] = torch.arange(at, at + n).flip(0)
        at += n
    kp, vp = torch.full((at, page, kv, 2, dim), 7.0, dtype=dtype, device="cuda"), torch.full((at, page, kv, 2 * dim), 7.0, dtype=dtype, device="cuda")
    out = torch.full_like(q, 5.0) if heads else None
    ops.append_paged(ctx, k, v, kp, vp, table.cuda(), i32(*ends), i32(*new), pos, freq, axis, q=q, interleaved=interleaved, out=out)
    theta, u, f32 = pos.double() * freq.double(), OO.UNIT[dtype], OO.F32 * (32 + 2 * dim)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0  # float16 numbers below 2^-14 lie 2^-24 apart

    def turned(x):
        y, size = OO.turned(x.double().flatten(1, 2), theta, interleaved)
        return y.view(x.shape), (u * y.abs() + f32 * size + tiny).view(x.shape)

    want_k, want_v = torch.full(kp.shape, 7.0, dtype=torch.float64, device="cuda"), torch.full_like(vp, 7.0)
    bound, (y, b) = torch.zeros_like(want_k), turned(k)
    for i, (a, n) in enumerate(zip(ends, new)):
        row = torch.arange(n, device="cuda")
        p = table[i].cuda().long()[row // page]
        want_k[p, row % page], bound[p, row % page], want_v[p, row % page] = y[a:a + n], b[a:a + n], v[a:a + n]
    assert torch.equal(vp, want_v)
    assert float(((kp.double() - want_k).abs() - bound).max()) <= 0.0
    if heads:
        held, (y, b) = slice(ends[0], ends[-1]), turned(q)
        assert float(((out.double() - y).abs() - b)[held].max()) <= 0.0
        assert bool((out[:ends[0]] == 5.0).all()) and bool((out[ends[-1]:] == 5.0).all())


@pytest.mark.parametrize("dim,interleaved,heads,kv", [(2, True, 1, 0), (8, False, 1, 2)])
def test_norms(ctx, dim, interleaved, heads, kv):
    """Against the formulas in 64 bits on a sample of the rows, the weights' gradients
    on all.  Their 32-bit sums are off by 2^-24 times the additions that one term goes
    through: 17 rows of two vectors a lane with 512 workgroups or more, 256 lanes, 16
    parts and their runs, below 512 in all."""
    g = torch.Generator(device="cuda").manual_seed(dim)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    x = [randn(ROWS, h, 1, dim) if h else None for h in (heads, kv)]
    dy = [randn(ROWS, h, 1, dim) if h else None for h in (heads, kv)]
    w = [1 + 0.3 * randn(dim) for _ in range(2)]
    pos, pairs = torch.rand((ROWS, 3), generator=g, device="cuda"), dim // 2
    freq, axis = (6.2831853 * (1 + torch.arange(pairs))).float().cuda(), (torch.arange(pairs) % 3).int().cuda()
    kw = dict(kind="rms", eps=1e-3, interleaved=interleaved)
    out = ops.head_norm_rotary(ctx, *x, *w, pos, freq, axis, **kw)
    grads = ops.head_norm_rotary_backward(ctx, *dy, *x, *w, pos, freq, axis, dpositions=True, **kw)
    rows = torch.cat([torch.arange(2000), torch.randint(0, ROWS, (2000,)), torch.arange(ROWS - 2000, ROWS)])
    f32 = OO.F32 * (32 + 2 * dim)
    dpos, size = 0.0, 0.0
    for i in range(2):
        if x[i] is None:
            assert out[i] is None and grads[i] is None and float(grads[2 + i].abs().max()) == 0.0
            continue
        xs, ds, ws, theta = x[i].cpu()[rows], dy[i].cpu()[rows], w[i].cpu(), (pos.double()[:, axis.long()] * freq.double()).cpu()
        want, s = PO.forward(xs, ws, theta[rows], "rms", 1e-3, interleaved)
        assert float(((out[i].double().cpu()[rows] - want).abs() - OO.F32 * want.abs() - f32 * s).max()) <= 0.0
        (dx, sx), _, (dp, sp) = PO.backward(xs, ws, ds, theta[rows], freq.double().cpu(), axis.cpu(), 3, "rms", 1e-3, interleaved)
        assert float(((grads[i].double().cpu()[rows] - dx).abs() - OO.F32 * dx.abs() - 4 * f32 * sx).max()) <= 0.0
        dpos, size = dpos + dp, size + sp
        _, (dw, sw), _ = PO.backward(x[i].cpu(), ws, dy[i].cpu(), theta, freq.double().cpu(), axis.cpu(), 3, "rms", 1e-3, interleaved)
        assert float(((grads[2 + i].double().cpu() - dw).abs() - OO.F32 * dw.abs() - (4 * f32 + OO.F32 * 512) * sw).max()) <= 0.0
    assert float(((grads[4].double().cpu()[rows] - dpos).abs() - OO.F32 * dpos.abs() - (4 * f32 + OO.F32 * (heads + kv) * dim) * size).max()) <= 0.0
