"""The operators among a program's other calls: errors that are not theirs,
handles that go away during a capture, broadcast inputs."""
import pytest
import torch

from mtpx import ops
from test_ops_gpu import rand

pytestmark = pytest.mark.gpu


def test_a_single_row_of_a_shared_gate(ctx):
    """One row's gate taken from a broadcast one has row stride 0 and is a gate
    per row all the same."""
    g = torch.Generator().manual_seed(4)
    x, gate = rand(g, 1, 24, dtype=torch.float32).cuda(), rand(g, 24, dtype=torch.float32).cuda()
    one = gate.expand(5, -1)[:1]
    assert one.stride(0) == 0
    got = ops.norm_block(ctx, x, x, one, save=True)
    want = ops.norm_block(ctx, x, x, one.clone(), save=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    grads = [ops.norm_block_backward(ctx, x, x, x, x, t, None, None, want[2]) for t in (one, one.clone())]
    assert grads[0][2].shape == (1, 24)
    assert all(a is None or torch.equal(a, b) for a, b in zip(*grads))
