"""Gradients of attention whose size is not 1.

Roundings are taken as independent, u / sqrt(3) each in the mean: a gradient of
q or k takes one of dS and, through D, one of each saved result, together u; a
gradient of v one of P.  Rounding the exact gradient to the type is measured,
not bounded: in float16 it is most of the error of small gradients."""
import math

import pytest
import torch

import ops_oracle as OO
from test_ops_few_keys_gpu import exact, gradients
from test_ops_gpu import DTYPES, IDS, attention_case, check_attention

pytestmark = pytest.mark.gpu
dtypes = pytest.mark.parametrize("dtype", DTYPES, ids=IDS)


def check_sizes(ctx, c, causal=False, scale=None):
    dtype, dim = c["q"].dtype, c["q"].shape[-1]
    u = OO.UNIT[dtype]
    got, r = gradients(ctx, c, causal, scale), exact(c, causal, scale)
    f32 = OO.F32 * (16 + 4 * dim + len(c["q"]) + 4 * r["scores"])
    for name, roundings in (("dq", 3), ("dk", 3), ("dv", 1)):
        assert bool(torch.isfinite(got[name]).all()), name
        own = float((r[name].to(dtype).double() - r[name]).norm())
        # (5 % above the mean of many thousand independent roundings)
        bound = 1.05 * math.hypot(own, (u * math.sqrt(roundings / 3) + f32) * float(r[name].norm()))
        off = float((got[name] - r[name]).norm())
        assert off <= bound, (name, off / bound)
    off = (got["dlam"] - r["dlam"]).abs()
    assert bool((off <= 4 * f32 * r["|dlam|"]).all()), "dlam"


@dtypes
@pytest.mark.parametrize("size", [1e-6, 1e-4, 1e-3, 1.0, 300.0])
@pytest.mark.parametrize("rows,heads,kv,dim", [([2048], 2, 1, 64), ([700, 40, 300], 4, 4, 32), ([600, 90], 2, 2, 128)])
def test_gradients_of_any_size(ctx, dtype, size, rows, heads, kv, dim):
    """As of a mean loss over many rows, or of a scaled one.  (float16 holds
    multiples of 6e-8: the incoming gradient is what it rounds to.)"""
    c = attention_case(dim, dtype, rows, rows, heads, kv, dim)
    c["dout"] = (c["dout"].double() * size).to(dtype)
    check_sizes(ctx, c, causal=len(rows) == 3)


@dtypes
@pytest.mark.parametrize("heads,kv,dim", [(2, 1, 64), (2, 2, 32), (2, 2, 128)])
@pytest.mark.parametrize("more", [0, 100])
def test_products_beyond_float16(ctx, dtype, heads, kv, dim, more):
    """Values and gradients whose products pass 65,504, while every input and
    every result is within it."""
    n = [6, 5, 4] * 10 + [more]
    c = attention_case(dim, dtype, n, n, heads, kv, dim)
    c["v"], c["dout"] = c["v"] * 16, c["dout"] * 2000
    check_sizes(ctx, c, scale=0.02)


@dtypes
def test_gradients_of_very_different_rows(ctx, dtype):
    """One row's gradient is 10^5 times the others': theirs keep their bits."""
    c = attention_case(11, dtype, [500], [500], 2, 2, 64)
    c["dout"] = c["dout"] * 1e-3
    c["dout"][7] *= 1e5
    got, r = gradients(ctx, c), exact(c)
    u = OO.UNIT[dtype]
    rest = torch.arange(500) != 7
    own = float((r["dq"][rest].to(dtype).double() - r["dq"][rest]).norm())
    off = float((got["dq"][rest] - r["dq"][rest]).norm())
    assert off <= 1.05 * math.hypot(own, (u + OO.F32 * 1000) * float(r["dq"][rest].norm()))


@dtypes
@pytest.mark.parametrize("lam", [3.0, -40.0, 900.0])
def test_large_lambda(ctx, dtype, lam):
    c = attention_case(12, dtype, [130, 70], [130, 70], 2, 1, 40)
    c["lam"] = torch.tensor([lam, 0.1])
    c["dout"] = c["dout"] * 0.01
    check_attention(ctx, c, False)


@dtypes
@pytest.mark.parametrize("size", [1e-4, 300.0])
@pytest.mark.parametrize("q_len,k_len,heads,kv,dim", [([1500], [60], 4, 1, 32), ([900], [300], 8, 2, 64), ([700], [130], 2, 1, 128)])
def test_gradients_of_any_size_of_a_shared_key_pass(ctx, dtype, size, q_len, k_len, heads, kv, dim):
    """Few keys and many rows: parts of the walk over the rows, each scaled by
    itself, are summed."""
    c = attention_case(dim, dtype, q_len, k_len, heads, kv, dim)
    c["dout"] = (c["dout"].double() * size).to(dtype)
    check_sizes(ctx, c)


@dtypes
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_identical_atoms(ctx, dtype, dim):
    """A perfect crystal: all rows are alike, dS is zero but for rounding."""
    c = attention_case(13, dtype, [200, 5, 64], [200, 5, 64], 2, 2, dim)
    for n in ("q", "k", "v", "dout"):
        c[n] = c[n][:1].expand_as(c[n]).contiguous()
    check_attention(ctx, c, False)
    c["dout"] = c["dout"] * 1e-3
    check_attention(ctx, c, True)


@dtypes
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_an_infinite_gradient_is_not_hidden(ctx, dtype, bad):
    """As a scaled loss that overflowed: the sequence it reaches is not finite,
    the others are."""
    c = attention_case(14, dtype, [150, 90], [150, 90], 2, 2, 64)
    c["dout"][20, :, 3] = bad
    got = gradients(ctx, c)
    for name in ("dq", "dk", "dv"):
        assert not bool(torch.isfinite(got[name][:150]).all()), name
        assert bool(torch.isfinite(got[name][150:]).all()), name


@dtypes
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_key_gradients_take_nothing_from_the_saved_results(ctx, dtype, dim):
    """k's gradient: the roundings of dS and of the result alone, each u /
    sqrt(3) of their own terms in the mean."""
    c = attention_case(dim + 3, dtype, [160, 90, 230, 75], [160, 90, 230, 75], 8, 8, dim)
    got, r = gradients(ctx, c), exact(c)
    own = float((r["dk"].to(dtype).double() - r["dk"]).norm() / r["dk"].norm())
    off = float((got["dk"] - r["dk"]).norm() / r["dk"].norm())
    # one rounding measured, the other as large; 3 % for the spread of many thousand elements
    assert off <= 1.03 * math.sqrt(2) * own + OO.F32 * (16 + 4 * dim + 4 * r["scores"]), off / own
