"""The bounds of tests/test_ops_norms_gpu.py see mistakes (made in the oracle),
and the oracle agrees with differentiation."""
import pytest
import torch

import norm_oracle as NO
import ops_oracle as OO


def inputs(seed, rows, width, gated, dtype):
    g = torch.Generator().manual_seed(seed)

    def rand(*shape, scale=1.0):
        return (torch.randn(shape, generator=g) * scale).to(dtype)

    x = rand(rows, width, scale=2.0) if gated else None
    y = rand(rows, width) + 0.25
    gate = [None, rand(width), rand(rows, width)][gated]
    return x, y, gate, 1 + rand(width, scale=0.1), 1 + rand(width, scale=0.1), rand(rows, width), rand(rows, width)


ARGS = dict(alpha=0.8, beta=-0.6, eps=1e-2)


@pytest.mark.parametrize("kind,act", [("rms", "none"), ("layer", "sigmoid"), ("rms", "tanh"), ("layer", "none")])
@pytest.mark.parametrize("gated", [0, 1, 2])
def test_the_oracle_is_the_derivative(kind, act, gated):
    x, y, gate, w1, w2, ds, dn = inputs(3, 5, 12, gated, torch.float64)
    val, size = NO.norm_block(x, y, gate, w1, w2, ds, dn, kind, act, **ARGS)
    leaf = [None if t is None else t.requires_grad_(True) for t in (x, y, gate, w1, w2)]
    s, n = OO.norm_block(*leaf, kind, act, 0.8, -0.6, 1e-2)
    ((s * ds).sum() + (n * dn).sum()).backward()
    for name, t in zip(("dx", "dy", "dgate", "dw1", "dw2"), leaf):
        assert (name in val) == (t is not None)
        if t is not None:
            # 64-bit rounding of the same sums
            assert bool(((val[name] - t.grad).abs() <= 2.0 ** -44 * size[name]).all())


@pytest.mark.parametrize("rows,width", [(3, 7), (70, 64), (20, 1000), (5, 4096), (4, 16384), (1100, 1032)])
@pytest.mark.parametrize("kind,act,mistake", [(k, a, m) for k, a in (("layer", "sigmoid"), ("rms", "tanh"), ("layer", "none"))
                                              for m in ("mean1", "mean2", "slope", "half") if k == "layer" or m in ("slope", "half")])
def test_mistakes_pass_the_bounds_of_32_bits(rows, width, kind, act, mistake):
    t = inputs(width, rows, width, 2, torch.float32)
    val, size = NO.norm_block(*t, kind, act, **ARGS)
    bad, _ = NO.norm_block(*t, kind, act, **ARGS, mutate=mistake)
    over = {n: NO.passed(bad[n], val[n], size[n], n, 2.0 ** -24) for n in val}
    seen_in = {"mean1": ["dy"], "mean2": ["dx", "dy", "dgate", "dw1"], "slope": ["dgate"],
               "half": ["dx", "dy", "dgate", "dw1"]}[mistake]
    assert all(over[n] > 1.0 for n in seen_in), over
    # and rounding the exact results to 32 bits does not
    assert all(NO.passed(val[n].float(), val[n], size[n], n, 2.0 ** -24) <= 1.0 for n in val)
