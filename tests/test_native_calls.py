"""The serving calls as native steps: whatever is not plainly right is left to
the checks in Python, and what both take has one result."""
import numpy as np
import pytest
import torch

from mtpx import capi, ops
from test_ops_gpu import dtypes, rand

CALLS = (("head_norm_rotary", 13), ("head_norm_rotary_backward", 16), ("append_paged", 20), ("diff_attention_paged", 14))


@pytest.mark.parametrize("name,n", CALLS)
def test_left_to_the_checks(name, n):
    call = getattr(ops._calls(), name)
    for fill in (None, 0, -1, 1 << 80, 1.5, "x", object(), torch.zeros(0), torch.zeros(2, 2, 2, 2), torch.zeros(1, 1, 1, 1, 1, dtype=torch.int32)):
        assert call(*[fill] * n) is None
        assert call(1, 0, lambda device: 0, *[fill] * (n - 3)) is None  # the handle is not looked into
        assert call(1, torch.zeros(1).get_device(), None, *[fill] * (n - 3)) is None
    for wrong in (0, n - 1, n + 1):
        with pytest.raises(TypeError):
            call(*[None] * wrong)


def test_a_library_that_is_not_there():
    with pytest.raises(TypeError):
        ops._calls().setup(1, 2, 3)
    with pytest.raises(TypeError):
        ops._calls().setup("a", "b", "c", "d", "e", "f")
    with pytest.raises(ValueError):
        ops._calls().setup(0, 0, 0, 0, 0, 0)


class _NoneOfThem:
    """Leaves every call to the checks in Python."""

    def __getattr__(self, name):
        return lambda *a: None


def _both(monkeypatch, call):
    got = call()
    with monkeypatch.context() as m:
        m.setattr(ops, "_calls", _NoneOfThem)
        want = call()
    got, want = ([r] if not isinstance(r, tuple) else list(r) for r in (got, want))
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert (a is None) == (b is None)
        if a is not None:
            assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() and torch.equal(a, b)


def _wide(t):
    """The same values with other strides, the last dimension contiguous."""
    room = torch.full((*t.shape[:-1], t.shape[-1] + 8), float("nan"), dtype=t.dtype, device=t.device)
    room[..., :t.shape[-1]] = t
    return room[..., :t.shape[-1]]


@pytest.mark.gpu
@dtypes
@pytest.mark.parametrize("positions", [torch.float32, torch.float64, torch.int32, torch.int64])
def test_the_same_results(ctx, monkeypatch, dtype, positions):
    g = torch.Generator().manual_seed(7)
    rows, h, kv, d, page = 11, 4, 2, 16, 8
    q, k = rand(g, rows, h, 2, d, dtype=dtype).cuda(), rand(g, rows, kv, 2, d, dtype=dtype).cuda()
    v, w, u = (rand(g, *s, dtype=dtype).cuda() for s in ((rows, kv, 2 * d), (d,), (d,)))
    pos = (torch.rand(rows, 2, generator=g) * 40).to(positions).cuda()
    freq, axis = torch.rand(6, generator=g).cuda(), (torch.arange(6) % 2).int().cuda()
    for x, y in ((q, k), (q, None), (_wide(q), _wide(k)), (q[:, :, 0], k[:, :, 1]), (q[:0], k[:0]), (q[:1], k[:1])):
        p = pos[:len(x)]
        for kw in ({}, dict(kind="layer", eps=1e-3, interleaved=True), dict(eps=1)):
            for wq, wk in ((w, u), (None, u), (w, None)):
                _both(monkeypatch, lambda: ops.head_norm_rotary(ctx, x, y, wq, wk, p, freq, axis, **kw))
                for moved in (False, True)[:1 + positions.is_floating_point]:
                    _both(monkeypatch, lambda: ops.head_norm_rotary_backward(ctx, x * 0.5, None if y is None else _wide(y), x, y, wq, wk, p, freq, axis,
                                                                             dpositions=moved, **kw))
    _both(monkeypatch, lambda: ops.head_norm_rotary(ctx, q, k, w, u, pos.t().contiguous().t(), freq[:0], axis[:0]))

    def filled(kt, vt, **kw):
        kp, vp = torch.zeros(9, page, kv, 2, d, dtype=dtype).cuda(), torch.zeros(9, page, kv, 2 * d, dtype=dtype).cuda()
        done = ops.append_paged(ctx, kt, vt, kp, vp, table, off, n, pos, freq, axis, **kw)
        return done if done is None else done[:10], kp, vp  # (row 10 is of no sequence and not written)

    table, off, n = (torch.tensor(t, dtype=torch.int32).cuda() for t in ([[4, 1, 7, 0], [8, 2, 3, 0]], [0, 9, 10], [20, 17]))
    for kw in ({}, dict(q=q), dict(q=_wide(q), kind="rms", q_weight=w, k_weight=u), dict(q=q, kind="layer", k_weight=u, eps=1e-2, interleaved=True)):
        _both(monkeypatch, lambda: filled(k, v, **kw))
        _both(monkeypatch, lambda: filled(_wide(k), _wide(v), **kw))
    _both(monkeypatch, lambda: filled(k, v, q=q, out=torch.zeros_like(_wide(q))))
    _both(monkeypatch, lambda: filled(k, v, q=q, eps=np.float32(1e-3)))  # (not plainly right; taken all the same)

    kp, vp, lam = rand(g, 9, page, kv, 2, d, dtype=dtype).cuda(), rand(g, 9, page, kv, 2 * d, dtype=dtype).cuda(), torch.rand(h, generator=g).cuda()
    for x, kt, vt in ((q, kp, vp), (_wide(q), _wide(kp), _wide(vp))):
        for kw in ({}, dict(causal=False), dict(scale=0.5), dict(scale=1, max_rows=9), dict(max_rows=1 << 40), dict(max_rows=np.int64(9))):
            out = torch.zeros(rows, h, 2 * d, dtype=dtype).cuda()  # rows of no sequence are left as they are
            _both(monkeypatch, lambda: ops.diff_attention_paged(ctx, x, kt, vt, lam, table, off, n, out=out.clone(), **kw))
        _both(monkeypatch, lambda: ops.diff_attention_paged(ctx, x[:10], kt, vt, lam, table, off, n))
    room = _wide(torch.zeros(rows, h, 2 * d, dtype=dtype).cuda())
    _both(monkeypatch, lambda: ops.diff_attention_paged(ctx, q, kp, vp, lam, table, off, n, out=room.zero_()).clone())


@pytest.mark.gpu
def test_refused_either_way(ctx, monkeypatch):
    """The library's refusals and those of the checks, in the same words."""
    q, k, v = torch.zeros(3, 2, 2, 8).cuda(), torch.zeros(3, 1, 2, 8).cuda(), torch.zeros(3, 1, 16).cuda()
    kp, vp, lam = torch.zeros(2, 4, 1, 2, 8).cuda(), torch.zeros(2, 4, 1, 16).cuda(), torch.zeros(2).cuda()
    freq, axis, pos, w = torch.ones(4).cuda(), torch.zeros(4, dtype=torch.int32).cuda(), torch.zeros(3, 1).cuda(), torch.ones(8).cuda()
    table, off, n = (torch.tensor(t, dtype=torch.int32).cuda() for t in ([[0, 1]], [0, 3], [3]))
    head = lambda q=q, k=k, w=w, pos=pos, freq=freq, axis=axis, **kw: ops.head_norm_rotary(ctx, q, k, w, w, pos, freq, axis, **kw)  # noqa: E731
    put = lambda k=k, v=v, kp=kp, vp=vp, table=table, off=off, n=n, **kw: ops.append_paged(ctx, k, v, kp, vp, table, off, n, pos, freq, axis, **kw)  # noqa: E731
    attend = lambda q=q, kp=kp, vp=vp, lam=lam, table=table, off=off, n=n, **kw: ops.diff_attention_paged(ctx, q, kp, vp, lam, table, off, n, **kw)  # noqa: E731
    odd, far = torch.zeros(3, 2, 2, 7).cuda(), torch.zeros(3, 1, dtype=torch.int16).cuda()
    back = lambda dq=q, dk=k, q=q, k=k, w=w, pos=pos, **kw: ops.head_norm_rotary_backward(ctx, dq, dk, q, k, w, w, pos, freq, axis, **kw)  # noqa: E731
    for call in (lambda: back(dk=None), lambda: back(k=None), lambda: back(dq=q[:2]), lambda: back(dq=q.half()), lambda: back(dk=k[..., :4]),
                 lambda: back(pos=pos.int(), dpositions=True), lambda: back(eps=-1.0), lambda: back(kind="none"), lambda: back(w=w.half()),
                 lambda: head(eps=-1.0), lambda: head(eps=float("nan")), lambda: head(kind="none"), lambda: head(pos=far), lambda: head(q=q.double()),
                 lambda: head(q=q[:2]), lambda: head(q=odd, k=None), lambda: head(q=q[:, :0]), lambda: head(w=w.half()), lambda: head(w=torch.ones(8)),
                 lambda: head(axis=axis.long()), lambda: head(freq=torch.ones(5).cuda(), axis=torch.zeros(5, dtype=torch.int32).cuda()),
                 lambda: put(k=k[..., ::2], v=v), lambda: put(q=q, kind="other"), lambda: put(q=q, out=q[:2]), lambda: put(out=q), lambda: put(k_weight=w),
                 lambda: put(off=off[:1]), lambda: put(n=n.long()), lambda: put(kp=kp[:1]), lambda: put(q=q, out=q.half()),
                 lambda: attend(max_rows=0), lambda: attend(lam=lam[:1]), lambda: attend(table=table.long()), lambda: attend(out=q), lambda: attend(q=q.half()),
                 lambda: attend(scale=float("nan")), lambda: attend(off=off.cpu()), lambda: attend(q=odd), lambda: attend(q=torch.zeros(3, 2, 1, 8).cuda())):
        said = []
        for native in (True, False):
            with monkeypatch.context() as m:
                if not native:
                    m.setattr(ops, "_calls", _NoneOfThem)
                with pytest.raises(capi.MtpxError) as e:
                    call()
            said.append(str(e.value))
        assert said[0] == said[1]
    gone = capi.Context(0)
    gone.close()
    with pytest.raises(capi.MtpxError):
        ops.head_norm_rotary(gone, q, k, w, w, pos, freq, axis)
