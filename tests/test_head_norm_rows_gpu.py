"""The backward pass of the norms of heads where a workgroup takes a row, and
another behind it; weights' gradients where there is nothing to add up."""
import pytest
import torch

from mtpx import ops
from test_head_norm_gpu import case, check

pytestmark = pytest.mark.gpu

# rows, heads, maps, dim, rotated, type, pairs side by side
WORKGROUP_ROWS = [
    (1100, 32, 2, 128, 128, torch.float32, False), (2047, 16, 2, 256, 200, torch.float32, True), (1500, 9, 2, 127, 126, torch.float32, False),
    (601, 64, 2, 128, 128, torch.bfloat16, False), (2048, 65, 2, 128, 96, torch.float16, True), (1025, 64, 2, 64, 64, torch.bfloat16, True)]


@pytest.mark.parametrize("rows,heads,maps,dim,rotated,dtype,interleaved", WORKGROUP_ROWS)
@pytest.mark.parametrize("real", [True, False])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_rows_one_after_the_other(ctx, rows, heads, maps, dim, rotated, dtype, interleaved, real, kind):
    """Sums of the positions' gradients and tables of cos and sin are kept for one row and used again for the next."""
    check(ctx, case(rows + dim, dtype, rows, heads, 3 if real else 0, maps, dim, rotated, kind, real), interleaved)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [0, 1, 37])
def test_a_weight_without_keys(ctx, dtype, rows):
    """Its gradient is written as zeros over whatever lay in its place: the binding's
    request with the results' addresses."""
    heads, dim = 2, 16
    q, w = torch.randn(rows, heads, 1, dim).to(dtype).cuda(), torch.ones(dim, dtype=dtype).cuda()
    pos, freq, axis = torch.rand(rows, 1).cuda(), torch.rand(8).cuda(), torch.zeros(8, dtype=torch.int32).cuda()
    dq, dwq, dwk = torch.empty_like(q), torch.full_like(w, float("nan")), torch.full_like(w, float("nan"))
    dpos, work = torch.full_like(pos, float("nan")), torch.full((1 << 18,), float("nan")).cuda()
    rows_of = lambda t: (t.data_ptr(), heads * dim, dim, dim)  # noqa: E731
    req = ops._pack_heads(ops._stream(ctx), ops.DTYPES[dtype], rows, heads, 0, 1, dim, 16, 0, 0, 1e-6, *rows_of(q), *(0,) * 12,
                          w.data_ptr(), w.data_ptr(), pos.data_ptr(), 0, 1, 1, 1, freq.data_ptr(), axis.data_ptr(), *rows_of(q), *(0,) * 4,
                          *rows_of(dq), *(0,) * 4, dwq.data_ptr(), dwk.data_ptr(), dpos.data_ptr(), work.data_ptr(), 4 * work.numel())
    ctx._check(ops._ops().mtpx_head_norm_rotary_backward(ctx.h, req), "gradients")
    assert torch.equal(dwk, torch.zeros_like(dwk))
    assert bool(torch.isfinite(dwq).all()) and bool(torch.isfinite(dq).all()) and bool(torch.isfinite(dpos).all())
    assert rows > 0 or torch.equal(dwq, torch.zeros_like(dwq))
