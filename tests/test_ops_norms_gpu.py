"""The norms around a block, element by element within what 32-bit arithmetic
and one rounding may leave (tests/norm_oracle.py): widths of every number of
threads, and more rows than the launched groups take at once."""
import pytest
import torch

import norm_oracle as NO
import ops_oracle as OO
from mtpx import ops
from test_ops_norm_bounds_host import ARGS, inputs

pytestmark = pytest.mark.gpu
dtypes = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])


def check(ctx, dtype, kind, act, rows, width, gated):
    t = inputs(width + rows, rows, width, gated, dtype)
    x, y, gate, w1, w2, ds, dn = (None if a is None else a.cuda() for a in t)
    kw = dict(kind=kind, gate_act=act, residual_scale=ARGS["alpha"], block_scale=ARGS["beta"], eps=ARGS["eps"])
    s, n, stats = ops.norm_block(ctx, x, y, gate, w1, w2, save=True, **kw)
    grads = ops.norm_block_backward(ctx, ds, dn, x, y, gate, w1, w2, stats, **kw)
    # the scales reach the kernels in 32 bits
    args = {k: float(torch.tensor(v, dtype=torch.float32)) for k, v in ARGS.items()}
    val, size = NO.norm_block(*t, kind, act, **args)
    for name, got in zip(NO.NAMES, (s, n, *grads)):
        assert (got is not None) == (name in val)
        if got is not None:
            assert got.dtype == dtype and bool(torch.isfinite(got).all())
            off = NO.passed(got.cpu(), val[name], size[name], name, OO.UNIT[dtype])
            assert off <= 1.0, (name, off)


WIDTHS = [(1, 1), (3, 7), (70, 64), (33, 129), (9, 512), (5, 1000), (7, 1025), (4, 1536), (3, 2353), (5, 4096), (2, 5001),
          (3, 8192), (2, 8193), (2, 16384)]


@dtypes
@pytest.mark.parametrize("kind,act,gated", [("rms", "none", 0), ("layer", "sigmoid", 1), ("rms", "tanh", 2), ("layer", "none", 2)])
@pytest.mark.parametrize("rows,width", WIDTHS)
def test_widths(ctx, dtype, kind, act, gated, rows, width):
    check(ctx, dtype, kind, act, rows, width, gated)


# Groups of the forward pass: 16,384 of 16 threads, 8,192 of 32, 4,096 of 64,
# 2,048 of 128; fewer in the backward pass.
@dtypes
@pytest.mark.parametrize("kind,act,gated", [("layer", "sigmoid", 1), ("rms", "tanh", 2), ("layer", "tanh", 0)])
@pytest.mark.parametrize("rows,width", [(33000, 40), (17001, 39), (16500, 200), (9003, 201), (8300, 500), (4099, 499),
                                        (4200, 1000), (2051, 1001)])
def test_several_rows_a_group(ctx, dtype, kind, act, gated, rows, width):
    check(ctx, dtype, kind, act, rows, width, gated)


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_gradients_against_differences(ctx, kind):
    """The 32-bit gradients along a direction in all inputs against 64-bit
    differences of the formula: central differences err by h^2 times a third
    derivative (below 1e-6 of the sum of absolute terms at h = 1e-4)."""
    t = inputs(6, 40, 72, 2, torch.float32)
    x, y, gate, w1, w2, ds, dn = (a.cuda() for a in t)
    kw = dict(kind=kind, gate_act="sigmoid", residual_scale=0.5, block_scale=0.25, eps=1e-2)
    _, _, stats = ops.norm_block(ctx, x, y, gate, w1, w2, save=True, **kw)
    grads = ops.norm_block_backward(ctx, ds, dn, x, y, gate, w1, w2, stats, **kw)
    g = torch.Generator().manual_seed(8)
    d = [torch.randn(a.shape, generator=g).double() for a in t[:5]]

    def loss(h):
        s, n = OO.norm_block(*(a.double() + h * b for a, b in zip(t, d)), kind, "sigmoid", 0.5, 0.25, 1e-2)
        return float((s * t[5].double()).sum() + (n * t[6].double()).sum())

    terms = [a.double().cpu() * b for a, b in zip(grads, d)]
    slope, size = sum(float(a.sum()) for a in terms), sum(float(a.abs().sum()) for a in terms)
    assert abs(slope - (loss(1e-4) - loss(-1e-4)) / 2e-4) < 1e-5 * size
