"""Backward passes that are recorded into a graph while another graph of the same
leaves lives: joined to the recording if that one was made on a stream of the
program's, refused if on the default one.  Passes that are not recorded are asked
nothing of it."""
from types import SimpleNamespace

import pytest
import torch

from mtpx import capi, ops
from test_ops_gpu import rand

CREATED = 0x7F0012345680  # a created stream's handle is an address


class _Node:
    def __init__(self, made):
        self.metadata, self.next_functions = {ops._STREAM: made}, ()
        self.variable = type("V", (), dict(is_cuda=True))


@pytest.mark.parametrize("made,refused", [(0, True), (1, True), (2, True), (CREATED, False), (CREATED + 64, False)])
def test_default_streams_are_refused(monkeypatch, made, refused):
    monkeypatch.setattr(ops, "_Leaf", _Node)
    monkeypatch.setattr(ops, "_stream", lambda ctx: CREATED)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    fn = SimpleNamespace(ctx=None, next_functions=((_Node(CREATED), 0), (None, 0), (_Node(made), 0)))
    if refused:
        with pytest.raises(capi.MtpxError, match="earlier graph"):
            ops._same_streams(fn)
    else:
        ops._same_streams(fn)


def test_a_pass_that_is_not_recorded_is_asked_nothing(monkeypatch):
    class Fn:
        @property
        def next_functions(self):
            raise AssertionError

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    ops._same_streams(Fn())


def test_streams_of_what_is_no_leaf():
    of = ops._calls().stream_of
    x = torch.ones(2, requires_grad=True)
    node = x.expand(2).grad_fn.next_functions[0][0]
    for other in (None, 7, "x", x, object(), torch.ones(1), node, (x * 2).grad_fn):  # (host tensors have no stream)
        assert of(other) is None
    for wrong in ((), (node, node)):
        with pytest.raises(TypeError):
            of(*wrong)


def _losses(ctx):
    """name: (leaves, loss of them), each function with leaves of its own."""
    g = torch.Generator().manual_seed(6)
    leaf = lambda *s: rand(g, *s, dtype=torch.float32).cuda().requires_grad_(True)  # noqa: E731
    rows, freq, axis = 40, torch.rand(8, generator=g).cuda(), torch.zeros(8, dtype=torch.int32).cuda()
    seqs = ops.Sequences(ctx, [0, 15, 40])
    heads = [leaf(rows, 4, 2, 16), leaf(rows, 2, 2, 16), leaf(16), leaf(16), leaf(rows, 1)]
    turned = [leaf(rows, 4, 16), leaf(rows, 1)]
    attended = [leaf(rows, 4, 2, 16), leaf(rows, 2, 2, 16), leaf(rows, 2, 32), leaf(4)]
    normed = [leaf(rows, 32), leaf(rows, 32), leaf(rows, 32), leaf(32), leaf(32)]
    square = lambda *t: sum(x.square().sum() for x in t)  # noqa: E731
    return dict(
        heads=(heads, lambda: square(*ops.HeadNormRotaryFn.apply(ctx, *heads, freq, axis, {}))),
        rotary=(turned, lambda: square(ops.RotaryFn.apply(ctx, *turned, freq, axis) + 1.0)),
        attention=(attended, lambda: square(ops.DiffAttentionFn.apply(ctx, *attended, seqs))),
        norm=(normed, lambda: square(*ops.NormBlockFn.apply(ctx, *normed, {}))))


def _set(leaves, g):
    with torch.no_grad():
        for t in leaves:
            t.copy_(torch.randn(t.shape, generator=g))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["heads", "rotary", "attention", "norm"])
def test_streams_of_leaves(ctx, name):
    """A leaf's end of a graph belongs to the stream that it was made on, whatever
    stream later passes use; a pass that is not recorded leaves no mark."""
    leaves, loss = _losses(ctx)[name]
    side = torch.cuda.Stream()
    for stream in (torch.cuda.default_stream(), side):
        with torch.cuda.stream(stream):
            ends = [t.expand_as(t).grad_fn.next_functions[0][0] for t in leaves]
        with torch.cuda.stream(side):
            loss().backward()
        assert not any(ops._STREAM in e.metadata for e in ends)
        assert [ops._made_on(SimpleNamespace(ctx=ctx), e) for e in ends] == [stream.cuda_stream] * len(leaves)
        torch.cuda.synchronize()
        del ends


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["heads", "rotary", "attention", "norm"])
def test_beside_a_graph_of_the_default_stream(ctx, name):
    leaves, loss = _losses(ctx)[name]
    alive = loss()
    torch.cuda.synchronize()
    with pytest.raises(capi.MtpxError, match="earlier graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(loss(), leaves)
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = torch.autograd.grad(loss(), leaves)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(loss(), leaves)))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["heads", "rotary", "attention", "norm"])
@pytest.mark.parametrize("gather", [False, True])
def test_beside_a_graph_of_a_side_stream(ctx, name, gather):
    """The leaves' ends live from a warm-up on a side stream, as a wrapper around a
    model keeps them: the pass is recorded and replayed with other values, eager
    passes between the replays.  gather: gradients gathered in the leaves."""
    leaves, loss = _losses(ctx)[name]
    side, g = torch.cuda.Stream(), torch.Generator().manual_seed(1)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = loss()
        torch.autograd.grad(alive, leaves, retain_graph=True)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        if gather:
            loss().backward()
            grads = [t.grad for t in leaves]
        else:
            grads = torch.autograd.grad(loss(), leaves)
    for _ in range(4):
        _set(leaves, g)
        want = torch.autograd.grad(loss(), leaves)
        torch.cuda.synchronize()
        for t in grads:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, want))
    del alive
