"""Attention at the sizes where its calls change kernels: 128-row tiles, the
cache split over workgroups, against the formulas in 64 bits."""
import math

import numpy as np
import pytest
import torch

import ops_oracle as OO
from mtpx import ops
from test_ops_gpu import IDS, DTYPES, attention_case, check_attention, close, rand

pytestmark = pytest.mark.gpu
dtypes = pytest.mark.parametrize("dtype", DTYPES, ids=IDS)

# 16-bit heads up to 64 wide take tiles of 128 rows, 32 a wave, where these
# are 512 or more and a sequence has more than 64 keys
BROAD = [130, 1, 257, 64, 90, 300, 0, 128, 129, 127, 65, 31, 200, 96, 17, 2, 160, 384, 33, 250, 1, 140, 66, 255, 100]


@dtypes
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("masked", [0.0, 0.3])
@pytest.mark.parametrize("heads,kv,dim", [(16, 4, 64), (16, 16, 32), (16, 2, 40)])
def test_tiles_of_128_rows(ctx, dtype, causal, masked, heads, kv, dim):
    assert sum(-(-n // 128) for n in BROAD) * heads >= 512
    check_attention(ctx, attention_case(dim, dtype, BROAD, BROAD, heads, kv, dim, masked=masked, empty_first=masked > 0), causal)


@dtypes
@pytest.mark.parametrize("causal", [False, True])
def test_tiles_of_128_rows_of_other_key_counts(ctx, dtype, causal):
    keys = [n * 7 % 190 for n in BROAD]
    check_attention(ctx, attention_case(5, dtype, BROAD, keys, 16, 8, 64, masked=0.1), causal)


@dtypes
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 32), (4, 1, 64), (20, 1, 40), (3, 3, 17), (2, 2, 128)])
@pytest.mark.parametrize("lengths", [[1500, 0, 1, 777, 1499], [4100], [33, 2100, 64, 1, 0, 2048, 1025]])
def test_caches_in_splits(ctx, dtype, heads, kv, dim, lengths):
    """More rows than one workgroup's waves take in four steps each; splits
    beyond a length are empty."""
    g = torch.Generator().manual_seed(dim + heads)
    n, cap = len(lengths), max(lengths) + 5
    q = rand(g, n, heads, 2, dim, dtype=dtype, scale=1.5)
    k, v = rand(g, n, cap, kv, 2, dim, dtype=dtype), rand(g, n, cap, kv, 2 * dim, dtype=dtype)
    lam = torch.rand(heads, generator=g)
    for i, m in enumerate(lengths):
        k[i, m:], v[i, m:] = math.nan, math.inf
    got = ops.diff_attention_cache(ctx, q.cuda(), k.cuda(), v.cuda(), lam.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda())
    u = OO.UNIT[dtype]
    for i, m in enumerate(lengths):
        r = OO.attention(q[i:i + 1].double(), k[i, :m].double(), v[i, :m].double(), lam.double(), dim ** -0.5, [0, 1], [0, m])
        f32 = OO.F32 * (16 + 4 * dim + m + 4 * r["scores"])
        tiny = 2.0 ** -25 * m * 8 if dtype == torch.float16 else 0.0
        close(got[i:i + 1], r["out"], r["|out|"], 1.25 * 2 * u + f32, tiny)


@dtypes
@pytest.mark.parametrize("dim", [32, 64])
def test_a_sequence_alone_and_in_a_large_batch(ctx, dtype, dim):
    """The forward result of a sequence is within rounding the same whichever
    tiles its batch takes."""
    c = attention_case(dim + 7, dtype, BROAD, BROAD, 16, 4, dim)
    dev = [c[n].cuda() for n in ("q", "k", "v", "lam")]
    whole = ops.diff_attention(ctx, *dev, ops.Sequences(ctx, c["q_off"]))
    for i in (0, 3, 5, 17):
        z = slice(int(c["q_off"][i]), int(c["q_off"][i + 1]))
        alone = ops.diff_attention(ctx, *(t[z] for t in dev[:3]), dev[3], ops.Sequences(ctx, np.array([0, z.stop - z.start])))
        assert float((alone.float() - whole[z].float()).abs().max()) <= 4 * OO.UNIT[dtype] * float(alone.abs().max())
