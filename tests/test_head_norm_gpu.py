"""mtpx.ops.head_norm_rotary and its gradients against their formulas in 64
bits, element by element.  A 16-bit result takes one rounding; 32-bit values are
off by 2^-24 times the operations between the inputs and them: dim for a sum
over a head, as many for its reciprocal root's half, and a few for the rotation
(cos and sin of a 32-bit fraction of a turn: 2 pi 2^-25 and two units each) and
the products, each times the size of what is added up.  float16 numbers below
2^-14 lie 2^-24 apart: a rounding there is off by up to 2^-25."""
import math

import pytest
import torch

import ops_oracle as OO
import paged_oracle as PO
from mtpx import capi, ops
from test_ops_gpu import close, dtypes, rand

pytestmark = pytest.mark.gpu


TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def case(seed, dtype, rows, heads, kv, maps, dim, rotated, kind, real=True, weights=True):
    g = torch.Generator().manual_seed(seed)
    shape = lambda h: (rows, h, maps, dim)  # noqa: E731
    pairs = rotated // 2
    c = dict(q=rand(g, *shape(heads), dtype=dtype, scale=2.0), k=rand(g, *shape(kv), dtype=dtype) + 0.5 if kv else None,
             dq=rand(g, *shape(heads), dtype=dtype), dk=rand(g, *shape(kv), dtype=dtype) if kv else None, wq=None, wk=None,
             kind=kind, axis=(torch.arange(pairs) % 3).int())
    if weights:
        c["wq"], c["wk"] = (1 + 0.3 * torch.randn(dim, generator=g)).to(dtype), rand(g, dim, dtype=dtype)
    if real:
        c["pos"], c["freq"] = torch.rand((rows, 3), generator=g), (6.2831853 * (1 + torch.arange(pairs) // 3)).float()
    else:
        c["pos"] = torch.randint(-9000, 90000, (rows, 3), generator=g, dtype=torch.int32)
        c["freq"] = (10000.0 ** (-torch.arange(pairs) / max(1, pairs))).float()
    return c


def check(ctx, c, interleaved, eps=1e-3):
    dtype, dim, kind = c["q"].dtype, c["q"].shape[-1], c["kind"]
    on = lambda t: None if t is None else t.cuda()  # noqa: E731
    turn = [on(c[t]) for t in ("pos", "freq", "axis")]
    given = [on(c[t]) for t in ("q", "k", "wq", "wk")]
    kw = dict(kind=kind, eps=eps, interleaved=interleaved)
    real = c["pos"].is_floating_point()
    out = ops.head_norm_rotary(ctx, *given, *turn, **kw)
    grads = ops.head_norm_rotary_backward(ctx, on(c["dq"]), on(c["dk"]), *given, *turn, dpositions=real, **kw)
    theta = c["pos"].double()[:, c["axis"].long()] * c["freq"].double()
    u, tiny = OO.UNIT[dtype], TINY[dtype]
    f32 = OO.F32 * (32 + 2 * dim)
    dpos, size, terms = 0.0, 0.0, 0
    for i, (x, w, dy) in enumerate((("q", "wq", "dq"), ("k", "wk", "dk"))):
        if c[x] is None:
            assert out[i] is None and grads[i] is None
            continue
        want, s = PO.forward(c[x], c[w], theta, kind, eps, interleaved)
        over = (out[i].double().cpu() - want).abs() - u * want.abs() - f32 * s - tiny
        assert bool(torch.isfinite(out[i]).all()) and float(over.max() if over.numel() else 0.0) <= 0.0
        n = c[x].shape[0] * c[x].shape[1] * c[x].shape[2]
        (dx, sx), (dw, sw), (dp, sp) = PO.backward(c[x], c[w], c[dy], theta, c["freq"].double(), c["axis"], 3, kind, eps, interleaved)
        over = (grads[i].double().cpu() - dx).abs() - u * dx.abs() - 4 * f32 * sx - tiny
        assert bool(torch.isfinite(grads[i]).all()) and float(over.max() if over.numel() else 0.0) <= 0.0
        if c[w] is None:
            assert grads[2 + i] is None
        else:
            over = (grads[2 + i].double().cpu() - dw).abs() - u * dw.abs() - (4 * f32 + OO.F32 * n) * sw - tiny
            assert float(over.max()) <= 0.0
        dpos, size, terms = dpos + dp, size + sp, terms + c[x].shape[1] * c[x].shape[2]
    if real:
        close(grads[4], dpos, size, 4 * f32 + OO.F32 * terms * dim)
    else:
        assert grads[4] is None
    again = ops.head_norm_rotary_backward(ctx, on(c["dq"]), on(c["dk"]), *given, *turn, dpositions=real, **kw)
    assert all(a is None or torch.equal(a, b) for a, b in zip(grads, again))
    return out


@dtypes
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,heads,kv,maps,dim,rotated", [
    (1, 1, 1, 1, 2, 2), (3, 32, 4, 2, 64, 64), (17, 5, 5, 2, 40, 36), (5, 2, 1, 1, 7, 6), (130, 3, 3, 2, 128, 96),
    (2, 1, 1, 2, 256, 256), (9, 33, 0, 2, 16, 0), (4, 2, 2, 1, 200, 100), (6, 1, 2, 2, 1, 0), (70, 2, 1, 1, 127, 126),
    (3, 2, 2, 2, 255, 2)])
def test_heads(ctx, dtype, interleaved, kind, rows, heads, kv, maps, dim, rotated):
    """Every width of an access, several rows a wave and several lanes a row."""
    check(ctx, case(rows * dim + heads, dtype, rows, heads, kv, maps, dim, rotated, kind, dim % 2 == 0), interleaved)


@dtypes
def test_many_rows(ctx, dtype):
    """More rows than workgroups of the backward pass; weights' gradients over all of them."""
    check(ctx, case(5, dtype, 9001, 2, 1, 2, 32, 32, "rms"), False)
    check(ctx, case(6, dtype, 2500, 40, 8, 1, 16, 12, "layer", real=False, weights=False), True)


@dtypes
def test_projections_side_by_side(ctx, dtype):
    """q and k as views of one projection, at any alignment, as three-dimensional tensors."""
    g = torch.Generator().manual_seed(8)
    whole = rand(g, 12, 6 * 48 + 9, dtype=dtype).cuda()
    pos, freq, axis = torch.rand(3, 12, generator=g).cuda().T, torch.rand(24, generator=g).cuda(), (torch.arange(24) % 3).int().cuda()
    w = rand(g, 50, dtype=dtype).cuda()
    for a in (0, 1, 4):
        q, k = whole[:, a:a + 4 * 48].unflatten(1, (4, 48)), whole[:, a + 4 * 48:a + 6 * 48].unflatten(1, (2, 48))
        wq, wk = w[a % 2:48 + a % 2], w[:48]
        got = ops.head_norm_rotary(ctx, q, k, wq, wk, pos, freq, axis, kind="layer")
        theta = pos.double().cpu()[:, axis.long().cpu()] * freq.double().cpu()
        for x, weight, y in ((q, wq, got[0]), (k, wk, got[1])):
            want, s = PO.forward(x.cpu()[:, :, None], weight.cpu(), theta, "layer", 1e-6, False)
            over = (y.double().cpu()[:, :, None] - want).abs() - OO.UNIT[dtype] * want.abs() - OO.F32 * 160 * s - TINY[dtype]
            assert float(over.max()) <= 0.0


def test_a_zero_head_and_no_rows(ctx):
    """A head of zeros is normed to zeros, whose gradient is w dz / sqrt(eps); no
    rows give zero gradients of the weights."""
    q = torch.zeros(2, 1, 8, device="cuda")
    w, pos = torch.full((8,), 2.0, device="cuda"), torch.zeros(2, 1, device="cuda")
    freq, axis = torch.ones(4, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    out, none = ops.head_norm_rotary(ctx, q, None, w, None, pos, freq, axis, eps=0.25)
    assert none is None and float(out.abs().max()) == 0.0
    dq, _, dw, _, _ = ops.head_norm_rotary_backward(ctx, torch.ones_like(q), None, q, None, w, None, pos, freq, axis, eps=0.25)
    assert torch.equal(dq, torch.full_like(q, 4.0)) and float(dw.abs().max()) == 0.0
    empty = torch.zeros(0, 3, 2, 8, device="cuda")
    out = ops.head_norm_rotary(ctx, empty, empty, w, None, pos[:0], freq, axis)
    assert out[0].shape == out[1].shape == empty.shape
    grads = ops.head_norm_rotary_backward(ctx, empty, empty, empty, empty, w, w, pos[:0], freq, axis, dpositions=True)
    assert float(grads[2].abs().max()) == 0.0 and float(grads[3].abs().max()) == 0.0 and grads[4].shape == (0, 1)


def test_gradients_against_differences(ctx):
    """Along a direction in q, k, the weights and the positions, from 64-bit
    differences of the formula (h^2 third derivatives: about 1e-8, cancellation
    1e-16 / h), against the 32-bit autograd function's."""
    c = case(3, torch.float32, 40, 4, 2, 2, 24, 20, "layer")
    g = torch.Generator().manual_seed(4)
    names = ("q", "k", "wq", "wk", "pos")
    d = {n: torch.randn(c[n].shape, generator=g).double() for n in names}

    def loss(s):
        t = {n: c[n].double() + s * d[n] for n in names}
        theta = t["pos"][:, c["axis"].long()] * c["freq"].double()
        return sum(float((PO.forward(t[x], t[w], theta, "layer", 1e-3, True)[0] * c[dy].double()).sum())
                   for x, w, dy in (("q", "wq", "dq"), ("k", "wk", "dk")))

    leaf = {n: c[n].cuda().requires_grad_(True) for n in names}
    y = ops.HeadNormRotaryFn.apply(ctx, leaf["q"], leaf["k"], leaf["wq"], leaf["wk"], leaf["pos"], c["freq"].cuda(),
                                   c["axis"].cuda(), dict(kind="layer", eps=1e-3, interleaved=True))
    torch.autograd.backward(y, (c["dq"].cuda(), c["dk"].cuda()))
    got = sum(float((leaf[n].grad.double().cpu() * d[n]).sum()) for n in names)
    size = sum(float((leaf[n].grad.double().cpu() * d[n]).abs().sum()) for n in names)
    h = 1e-6
    assert abs(got - (loss(h) - loss(-h)) / (2 * h)) < 1e-5 * size


def test_one_gradient_alone_and_second_ones_refused(ctx):
    """A loss of k only leaves q a zero gradient; a frequency that wants one raises."""
    c = case(3, torch.float32, 6, 2, 1, 2, 8, 8, "rms")
    leaf = [c[n].cuda().requires_grad_(True) for n in ("q", "k", "wq", "wk", "pos")]
    freq, axis = c["freq"].cuda(), c["axis"].cuda()
    _, k = ops.HeadNormRotaryFn.apply(ctx, *leaf, freq, axis, {})
    k.square().sum().backward()
    assert float(leaf[0].grad.abs().max()) == 0.0 and float(leaf[1].grad.abs().max()) > 0.0
    q, _ = ops.HeadNormRotaryFn.apply(ctx, *leaf, freq, axis, {})
    force, = torch.autograd.grad(q.square().sum(), leaf[4], create_graph=True)
    with pytest.raises(capi.MtpxError, match="second derivative"):
        force.square().sum().backward()
    with pytest.raises(capi.MtpxError, match="freq"):
        ops.HeadNormRotaryFn.apply(ctx, *leaf, freq.clone().requires_grad_(True), axis, {})[0].sum().backward()


def test_large_positions_keep_their_phase(ctx):
    pos = torch.tensor([[2 ** 40 + 12345], [-(2 ** 37) - 77]])
    freq = torch.tensor([1.0, 0.37], dtype=torch.float32)
    x = torch.tensor([[[1.0, 1.0, 1.0, -1.0]]] * 2)
    y, _ = ops.head_norm_rotary(ctx, x.cuda(), None, None, None, pos.cuda(), freq.cuda(), torch.zeros(2, dtype=torch.int32).cuda(), eps=0.0)
    want, _ = OO.turned(x.double(), pos.double() * freq.double(), False)
    # turns of 2^38: their fraction in 64 bits is good to 2^-14
    assert float((y.double().cpu() - want).abs().max()) < 2 * math.pi * 2 ** -13


@pytest.mark.parametrize("rows", [0, 37])
def test_a_weight_without_keys(ctx, rows):
    """Its gradient is zero, whatever lay in its place."""
    q, w = torch.randn(rows, 2, 16).cuda(), torch.ones(16).cuda()
    pos, freq, axis = torch.rand(rows, 1).cuda(), torch.rand(8).cuda(), torch.zeros(8, dtype=torch.int32).cuda()
    torch.full((16,), float("nan")).cuda()
    got = ops.head_norm_rotary_backward(ctx, q, None, q, None, w, w, pos, freq, axis)
    assert got[1] is None and float(got[3].abs().max()) == 0.0
