"""Elements of a head that the rotation copies: what one holds, infinities and NaN
among it, does not reach the next."""
import math

import pytest
import torch

from mtpx import ops
from test_ops_gpu import dtypes, rand

pytestmark = pytest.mark.gpu

ODD = (math.inf, -math.inf, math.nan, -0.0)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def same(a, b):
    """Bit for bit, NaN of any kind taken for another."""
    bits = {2: torch.int16, 4: torch.int32}[a.element_size()]
    return bool(((a.view(bits) == b.view(bits)) | (a.isnan() & b.isnan())).all())


@dtypes
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotated", [(32, 16), (40, 36), (64, 32), (7, 4), (16, 0), (200, 72)])
def test_appended_as_they_are(ctx, dtype, interleaved, dim, rotated):
    g = torch.Generator().manual_seed(dim)
    rows, kv = 9, 2
    k, v, q = (rand(g, *s, dtype=dtype).cuda() for s in ((rows, kv, 2, dim), (rows, kv, 2 * dim), (rows, 3, 2, dim)))
    for j, odd in enumerate(ODD):
        for t in (k, q):
            t[j, :, :, rotated + j % (dim - rotated)] = odd
            t[j + 4, 1, 0, dim - 1 - j % (dim - rotated)] = odd
    pos = torch.arange(rows)[:, None].cuda()
    freq, axis = torch.rand(rotated // 2, generator=g).cuda(), torch.zeros(rotated // 2, dtype=torch.int32).cuda()
    kp, vp = torch.zeros(2, 8, kv, 2, dim, dtype=dtype).cuda(), torch.zeros(2, 8, kv, 2 * dim, dtype=dtype).cuda()
    got = ops.append_paged(ctx, k, v, kp, vp, i32(1, 0)[None], i32(0, rows), i32(rows), pos, freq, axis, q=q, interleaved=interleaved)
    assert same(got[..., rotated:], q[..., rotated:])
    assert bool(torch.isfinite(got[..., :rotated]).all())
    kept = torch.cat([kp[1], kp[0, :1]])
    assert same(kept[..., rotated:], k[..., rotated:])
    assert bool(torch.isfinite(kept[..., :rotated]).all())


@dtypes
@pytest.mark.parametrize("interleaved", [False, True])
def test_weights_gradients_of_the_others(ctx, dtype, interleaved):
    """An infinite gradient of one copied element: that element's weight has it alone."""
    g = torch.Generator().manual_seed(1)
    rows, heads, dim, rotated = 5, 2, 48, 16
    q, dq, w = (rand(g, *s, dtype=dtype).cuda() for s in ((rows, heads, 2, dim), (rows, heads, 2, dim), (dim,)))
    pos, freq, axis = torch.rand(rows, 1, generator=g).cuda(), torch.rand(rotated // 2, generator=g).cuda(), torch.zeros(rotated // 2, dtype=torch.int32).cuda()
    back = lambda dy: ops.head_norm_rotary_backward(ctx, dy, None, q, None, w, None, pos, freq, axis, interleaved=interleaved)  # noqa: E731
    plain = back(dq)
    for e in (rotated, rotated + 1, 30, dim - 1):
        dy = dq.clone()
        dy[2, 1, 0, e] = math.inf
        got = back(dy)
        others = torch.arange(dim, device="cuda") != e
        assert not bool(torch.isfinite(got[2][e])) and torch.equal(got[2][others], plain[2][others])
        whole = torch.ones(rows, heads, 2, dtype=torch.bool, device="cuda")
        whole[2, 1, 0] = False
        assert torch.equal(got[0][whole], plain[0][whole])
