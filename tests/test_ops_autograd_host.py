"""The autograd functions of mtpx.ops over stand-ins for the library's calls:
what autograd does with them needs no GPU.  The stand-ins compute the real
formulas and return tensors without a graph, as the kernels do."""
import ctypes as C

import pytest
import torch

from mtpx import capi, ops

AXIS = torch.tensor([0, 1], dtype=torch.int32)


def _turned(x, positions, freq, sign=1.0):
    t = sign * positions[:, AXIS.long()] * freq
    c, s = t.cos()[:, None], t.sin()[:, None]
    a, b = x[..., :2], x[..., 2:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _mixed(q, k, v, lam):
    p = torch.softmax(torch.einsum("rhmd,khmd->hmrk", q, k), -1)
    return torch.einsum("hrk,khd->rhd", p[:, 0] - lam[:, None, None] * p[:, 1], v)


def _normed(x, y, gate, w1, w2):
    s = x + gate * w1 * y / (y * y).mean(1, keepdim=True).sqrt()
    return s, w2 * s / (s * s).mean(1, keepdim=True).sqrt()


def _gradients(f, inputs, grads):
    with torch.enable_grad():
        leaf = [t.detach().requires_grad_(True) for t in inputs]
        out = f(*leaf)
        out = out if isinstance(out, tuple) else (out,)
        pairs = [(o, g) for o, g in zip(out, grads) if g is not None]
        got = torch.autograd.grad([o for o, _ in pairs], leaf, [g.detach() for _, g in pairs],
                                  allow_unused=True)
    return tuple(t.detach() if t is not None else None for t in got)


@pytest.fixture
def calls(monkeypatch):
    """The plain functions without a library."""
    def rotary(ctx, x, positions, freq, axis, *, interleaved=False):
        return _turned(x, positions, freq).detach()

    def rotary_backward(ctx, dy, positions, freq, axis, *, interleaved=False, x=None):
        if x is None:
            return _turned(dy, positions, freq, -1.0).detach(), None
        return _gradients(lambda a, p: _turned(a, p, freq.detach()), (x, positions), (dy,))

    def diff_attention(ctx, q, k, v, lam, seqs, *, save, **kw):
        return _mixed(q, k, v, lam).detach(), (torch.zeros(1), torch.zeros(1))

    def diff_attention_backward(ctx, dout, q, k, v, lam, seqs, out, saved, **kw):
        return _gradients(_mixed, (q, k, v, lam), (dout,))

    def norm_block(ctx, x, y, gate, w1, w2, *, save, **kw):
        return (*(t.detach() for t in _normed(x, y, gate, w1, w2)), torch.zeros(1))

    def norm_block_backward(ctx, ds, dn, x, y, gate, w1, w2, stats, **kw):
        return _gradients(_normed, (x, y, gate, w1, w2), (ds, dn))

    for f in (rotary, rotary_backward, diff_attention, diff_attention_backward, norm_block, norm_block_backward):
        monkeypatch.setattr(ops, f.__name__, f)


def _rand(*shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(sum(shape))).double()


def _rotation(t):
    return ops.RotaryFn.apply(None, t[:, None].expand(-1, 3, 4), t[:, :2], _rand(2), AXIS)


def _attention(t):
    q = t[:, None, None].expand(-1, 2, 2, 4)
    return ops.DiffAttentionFn.apply(None, q, q * 0.5, t[:, None].expand(-1, 2, 4), t[0, :2], None)


def _norm(t):
    return ops.NormBlockFn.apply(None, t, t * t, t[0], t[1], t[2], {})[1]


@pytest.mark.parametrize("block", [_rotation, _attention, _norm])
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("named", [False, True])
def test_a_second_derivative_is_refused(calls, block, weighted, named):
    """An energy through the block, its forces, and a loss of both: the
    kernels' gradients carry no graph, so the forces' part would be lost.
    weighted: the gradient that reaches the block has a graph itself; named:
    the weight's gradient is asked for by name, not left on all leaves."""
    w = torch.nn.Parameter(torch.tensor(1.3).double())
    r = _rand(5, 4).requires_grad_(True)
    y = block(r * w)
    energy = (y * w if weighted else y).sum()
    force, = torch.autograd.grad(energy, r, create_graph=True)
    loss = energy + force.square().sum()
    with pytest.raises(capi.MtpxError, match="second derivative"):
        torch.autograd.grad(loss, [w]) if named else loss.backward()


@pytest.mark.parametrize("block", [_rotation, _attention, _norm])
def test_a_kept_graph_without_second_derivatives_is_not(calls, block):
    """create_graph for another part of the loss: the block's own gradients
    are used once and are those without create_graph."""
    r = _rand(5, 4).requires_grad_(True)
    want, = torch.autograd.grad(block(r).sum(), r)
    got, = torch.autograd.grad(block(r).sum(), r, create_graph=True)
    assert torch.equal(got, want)
    other, = torch.autograd.grad(r.pow(3).sum(), r, create_graph=True)
    second, = torch.autograd.grad(other.sum() + 0.0 * got.detach().sum(), r)
    assert torch.allclose(second, 6 * r)


def test_a_learned_frequency_is_refused(calls):
    """freq has no gradient; without one asked for it may be a parameter."""
    freq = torch.nn.Parameter(_rand(2))
    x, positions = _rand(5, 3, 4).requires_grad_(True), _rand(5, 2)
    y = ops.RotaryFn.apply(None, x, positions, freq, AXIS)
    with pytest.raises(capi.MtpxError, match="freq"):
        y.sum().backward()
    with torch.no_grad():
        ops.RotaryFn.apply(None, x, positions, freq, AXIS)


@pytest.mark.parametrize("name", ["residual_scale", "block_scale", "eps"])
def test_a_learned_scale_of_the_norms_is_refused(calls, name):
    t = _rand(5, 4).requires_grad_(True)
    learned = torch.nn.Parameter(torch.tensor(0.5))
    s, _ = ops.NormBlockFn.apply(None, t, t, t[0], t[1], t[2], {name: learned})
    with pytest.raises(capi.MtpxError, match=name):
        s.sum().backward()
    s, _ = ops.NormBlockFn.apply(None, t, t, t[0], t[1], t[2], {name: learned.detach()})
    s.sum().backward()


def test_a_learned_scale_of_the_scores_is_refused(calls):
    q, v = _rand(3, 2, 2, 4).requires_grad_(True), _rand(3, 2, 4)
    learned = torch.nn.Parameter(torch.tensor(0.5))
    out = ops.DiffAttentionFn.apply(None, q, q, v, _rand(2), None, False, learned)
    with pytest.raises(capi.MtpxError, match="scale"):
        out.sum().backward()


class _EmptiedByOthers(dict):
    """A dictionary that another thread empties after each call of this one."""

    def __contains__(self, key):
        found = dict.__contains__(self, key)
        self.clear()
        return found

    def get(self, key, default=None):
        value = dict.get(self, key, default)
        self.clear()
        return value

    def __setitem__(self, key, value):
        dict.__setitem__(self, key, value)
        self.clear()


@pytest.mark.parametrize("known", [False, True])
def test_workspace_sizes_while_another_thread_empties_them(known):
    """Autograd's backward pass is another thread on the same context."""
    class Ctx:
        h, workspaces = None, _EmptiedByOthers()

        @staticmethod
        def _check(rc, what):
            assert rc == 0

    def query(h, request, size):
        C.cast(size, C.POINTER(C.c_size_t))[0] = 4096
        return 0

    sizes = dict(dtype=0, rows=3, width=8)
    if known:
        dict.__setitem__(Ctx.workspaces, (ops.NormRequest, *sizes.values()), 4096)
    assert ops._bytes(Ctx, query, ops.NormRequest, **sizes) == 4096


def test_a_handle_outlives_the_module(monkeypatch):
    """At the end of a program the module's names may go before a handle that
    a global holds: it is still destroyed, and without an error."""
    destroyed = []

    class Library:
        @staticmethod
        def mtpx_sequences_create(h, n, q, k, out):
            C.cast(out, C.POINTER(C.c_void_p))[0] = 64
            return 0

        @staticmethod
        def mtpx_sequences_destroy(h):
            destroyed.append(h.value)

    class Ctx:
        h = None

        @staticmethod
        def _check(rc, what):
            assert rc == 0

    monkeypatch.setattr(ops, "_ops", lambda: Library)
    handle = ops.Sequences(Ctx, [0, 4])
    monkeypatch.setattr(ops, "_ops", None)
    handle.__del__()
    assert destroyed == [64]
    handle.close()
    assert destroyed == [64]
