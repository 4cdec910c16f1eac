"""Gradients of rows that see few keys, whatever else is in their batch: dS is
a small difference there, of which D = dO . O from rounded results would lose
as much as its own rounding."""
import math

import pytest
import torch

import ops_oracle as OO
from mtpx import ops
from test_ops_gpu import DTYPES, IDS, attention_case

pytestmark = pytest.mark.gpu
dtypes = pytest.mark.parametrize("dtype", DTYPES, ids=IDS)


def gradients(ctx, c, causal=False, scale=None):
    dev = [c[n].cuda() for n in ("q", "k", "v", "lam")]
    seqs = ops.Sequences(ctx, c["q_off"], c["k_off"])
    out, saved = ops.diff_attention(ctx, *dev, seqs, causal=causal, scale=scale, save=True)
    got = ops.diff_attention_backward(ctx, c["dout"].cuda(), *dev, seqs, out, saved, causal=causal, scale=scale)
    return dict(zip(("dq", "dk", "dv", "dlam"), (t.double().cpu() for t in got)))


def exact(c, causal=False, scale=None):
    scale = c["q"].shape[-1] ** -0.5 if scale is None else scale
    return OO.attention(*(c[n].double() for n in ("q", "k", "v", "lam")), scale, c["q_off"], c["k_off"], causal,
                        c["mask"], c["dout"].double())


def few(ctx, dtype, lengths, short, heads, dim, causal):
    """dq (and dk) of the rows `short`: two roundings, of dS and of the result;
    nothing of the saved results'."""
    c = attention_case(dim + 1, dtype, lengths, lengths, heads, heads, dim)
    got, r = gradients(ctx, c, causal), exact(c, causal)
    bound = math.sqrt(2 / 3) * OO.UNIT[dtype] * 1.1 + OO.F32 * (16 + 4 * dim + 4 * r["scores"])
    rows = torch.cat([torch.arange(*z) for z in short(c["q_off"])])
    for name in ("dq",) if causal else ("dq", "dk"):
        off = float((got[name][rows] - r[name][rows]).norm() / r[name][rows].norm())
        assert off < bound, (name, off / bound)


@dtypes
@pytest.mark.parametrize("heads", [4, 32])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_few_keys_beside_a_long_sequence(ctx, dtype, dim, heads):
    """The gradients of short sequences do not lose by what else is in the
    batch (32 heads: enough tiles for 128 rows each)."""
    lengths = [2, 3, 4] * 12 + [300, 65]
    few(ctx, dtype, lengths, lambda at: [(int(at[i]), int(at[i + 1])) for i in range(36)], heads, dim, False)


@dtypes
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_first_rows_of_causal_sequences(ctx, dtype, dim):
    """Rows 1 to 3 of long causal sequences see two to four keys."""
    lengths = [150, 70, 130] * 6
    few(ctx, dtype, lengths, lambda at: [(int(a) + 1, int(a) + 4) for a in at[:-1]], 8, dim, True)
