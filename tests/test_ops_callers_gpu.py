"""The operators among a program's other calls: errors that are not theirs,
handles that go away during a capture, broadcast inputs."""
import ctypes as C
import gc

import pytest
import torch

from mtpx import capi, ops
from test_ops_gpu import rand

pytestmark = pytest.mark.gpu


def _hip():
    """The HIP runtime that torch and the library share."""
    for line in open("/proc/self/maps"):
        if "libamdhip64" in line:
            return C.CDLL(line.split()[-1])
    raise AssertionError("no HIP runtime is loaded")


def test_an_earlier_calls_error_is_not_this_calls(ctx):
    """An allocation that another part of the program asked for and did not
    get, without clearing the runtime's last error."""
    hip, p = _hip(), C.c_void_p()
    q = torch.ones(4, 2, 2, 8, device="cuda")
    v, lam, seqs = torch.ones(4, 2, 16, device="cuda"), torch.ones(2, device="cuda"), ops.Sequences(ctx, [0, 4])
    freq, axis = torch.ones(2, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    pos, x = torch.ones(4, 1, device="cuda"), torch.ones(4, 8, device="cuda")
    lengths = torch.tensor([2, 3], dtype=torch.int32, device="cuda")
    out, saved = ops.diff_attention(ctx, q, q, v, lam, seqs, save=True)
    _, _, stats = ops.norm_block(ctx, x, x, save=True)
    for call in (lambda: ops.rotary(ctx, q.flatten(1, 2), pos, freq, axis),
                 lambda: ops.diff_attention(ctx, q, q, v, lam, seqs),
                 lambda: ops.diff_attention_backward(ctx, v, q, q, v, lam, seqs, out, saved),
                 lambda: ops.diff_attention_cache(ctx, q[:2], q[None].expand(2, -1, -1, -1, -1), v[None].expand(2, -1, -1, -1), lam, lengths),
                 lambda: ops.norm_block(ctx, x, x),
                 lambda: ops.norm_block_backward(ctx, x, x, x, x, None, None, None, stats)):
        want = call()
        assert hip.hipMalloc(C.byref(p), C.c_size_t(1 << 60)) != 0
        try:
            got = call()
        finally:
            hip.hipGetLastError()
        for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
            assert a is None or torch.equal(a, b)


def test_sequences_may_go_away_during_a_capture(ctx):
    """The collector frees a handle whenever it likes, also while a graph is
    recorded; the graph and the next handle are whole."""
    g = torch.Generator().manual_seed(3)
    q, v, lam = rand(g, 90, 2, 2, 32, dtype=torch.bfloat16).cuda(), rand(g, 90, 2, 64, dtype=torch.bfloat16).cuda(), torch.rand(2).cuda()
    seqs, gone = ops.Sequences(ctx, [0, 30, 90]), ops.Sequences(ctx, [0, 90])
    want = ops.diff_attention(ctx, q, q, v, lam, seqs)
    other = ops.diff_attention(ctx, q, q, v, lam, gone)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.diff_attention(ctx, q, q, v, lam, seqs)
        del gone
        gc.collect()
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        again = ops.Sequences(ctx, [0, 90])
        assert torch.equal(ops.diff_attention(ctx, q, q, v, lam, again), other)
        again.close()


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


def test_a_loss_of_forces_is_refused(ctx):
    """Through all three autograd functions on the device, whose backward pass
    is another thread: the forces are there, a loss of them raises."""
    g = torch.Generator().manual_seed(5)
    w = rand(g, 24, 4 * 16, dtype=torch.float32).cuda().requires_grad_(True)
    x, pos = rand(g, 20, 24, dtype=torch.float32).cuda(), torch.rand(20, 3, generator=g).cuda().requires_grad_(True)
    freq, axis = torch.ones(4, device="cuda"), (torch.arange(4) % 3).int().cuda()
    seqs, lam = ops.Sequences(ctx, [0, 8, 20]), torch.rand(1, generator=g).cuda()

    def energy():
        qk = ops.RotaryFn.apply(ctx, (x @ w)[:, :32].unflatten(1, (4, 8)), pos, freq, axis)
        out = ops.DiffAttentionFn.apply(ctx, qk[:, None, :2], qk[:, None, 2:], (x @ w)[:, None, 32:48], lam, seqs)
        return ops.NormBlockFn.apply(ctx, None, out.flatten(1), None, None, None, {})[1].square().sum()

    want, = torch.autograd.grad(energy(), pos)
    e = energy()
    force, = torch.autograd.grad(e, pos, create_graph=True)
    assert torch.equal(force, want) and float(force.detach().abs().max()) > 0.0
    with pytest.raises(capi.MtpxError, match="second derivative"):
        (e + force.square().sum()).backward()
    with pytest.raises(capi.MtpxError, match="second derivative"):
        torch.autograd.grad(force.square().sum(), w)
    learned = freq.clone().requires_grad_(True)
    with pytest.raises(capi.MtpxError, match="freq"):
        ops.RotaryFn.apply(ctx, x[:, None, :8], pos, learned, axis).sum().backward()
