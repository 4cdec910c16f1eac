"""The paged cache and the norms of heads among a program's other calls: errors
that are not theirs, gradients in place, captured steps, autograd through a block
and the serving of what it has learned."""
import ctypes as C
import threading

import numpy as np
import pytest
import torch

import ops_oracle as OO
import paged_oracle as PO
from mtpx import capi, ops
from test_ops_callers_gpu import _hip
from test_ops_gpu import dtypes, rand

pytestmark = pytest.mark.gpu


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def test_an_earlier_calls_error_is_not_this_calls(ctx):
    hip, p = _hip(), C.c_void_p()
    q, k = torch.ones(4, 2, 2, 8, device="cuda"), torch.ones(4, 1, 2, 8, device="cuda")
    v, lam, w = torch.ones(4, 1, 16, device="cuda"), torch.ones(2, device="cuda"), torch.ones(8, device="cuda")
    freq, axis, pos = torch.ones(2, device="cuda"), i32(0, 0), torch.ones(4, 1, device="cuda")
    kp, vp = torch.zeros(3, 4, 1, 2, 8, device="cuda"), torch.zeros(3, 4, 1, 16, device="cuda")
    table, off, n = i32(2, 0)[None], i32(0, 4), i32(6)
    for call in (lambda: ops.head_norm_rotary(ctx, q, k, w, None, pos, freq, axis),
                 lambda: ops.head_norm_rotary_backward(ctx, q, k, q, k, w, None, pos, freq, axis, dpositions=True),
                 lambda: ops.append_paged(ctx, k, v, kp, vp, table, off, n, pos, freq, axis, q=q),
                 lambda: ops.diff_attention_paged(ctx, q, kp, vp, lam, table, off, n)):
        want = call()
        assert hip.hipMalloc(C.byref(p), C.c_size_t(1 << 60)) != 0
        try:
            got = call()
        finally:
            hip.hipGetLastError()
        for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
            assert (a is None and b is None) or torch.equal(a, b)


@dtypes
def test_gradients_in_the_place_of_gradients(ctx, dtype):
    """The C entry lets dq be dq_out: the binding's request with the result's address changed."""
    g = torch.Generator().manual_seed(2)
    rows, heads, dim = 50, 3, 48
    q, dy, w = (rand(g, *s, dtype=dtype).cuda() for s in ((rows, heads, 2, dim), (rows, heads, 2, dim), (dim,)))
    pos, freq, axis = torch.rand(rows, 1, generator=g).cuda(), torch.rand(20, generator=g).cuda(), torch.zeros(20, dtype=torch.int32).cuda()
    want = ops.head_norm_rotary_backward(ctx, dy, None, q, None, w, None, pos, freq, axis)[0]
    rows_of = lambda t: (t.data_ptr(), heads * 2 * dim, 2 * dim, dim)  # noqa: E731
    work, dw = torch.empty(1 << 20, dtype=torch.uint8, device="cuda"), torch.empty_like(w)
    req = ops._pack_heads(ops._stream(ctx), ops.DTYPES[dtype], rows, heads, 0, 2, dim, 40, 0, 0, 1e-6, *rows_of(q), *(0,) * 12,
                          w.data_ptr(), 0, pos.data_ptr(), 0, 1, 1, 1, freq.data_ptr(), axis.data_ptr(), *rows_of(dy), *(0,) * 4,
                          *rows_of(dy), *(0,) * 4, dw.data_ptr(), 0, 0, work.data_ptr(), work.numel())
    ctx._check(ops._ops().mtpx_head_norm_rotary_backward(ctx.h, req), "in place")
    assert torch.equal(dy, want)


def test_a_training_step_in_a_graph(ctx):
    """Norms, rotation and attention, forward and backward, recorded once on plain
    functions and replayed with other inputs, eager work between the replays."""
    g = torch.Generator().manual_seed(4)
    rows, h, hk, d, dt = 90, 4, 2, 32, torch.bfloat16
    q, k, v, dout = (torch.zeros(rows, *s, dtype=dt).cuda() for s in ((h, 2, d), (hk, 2, d), (hk, 2 * d), (h, 2 * d)))
    w, lam, seqs = (1 + rand(g, d, dtype=dt, scale=0.1)).cuda(), torch.rand(h, generator=g).cuda(), ops.Sequences(ctx, [0, 30, 90])
    pos, freq, axis = torch.rand(rows, 3, generator=g).cuda(), (6.2832 * (1 + torch.arange(12) // 3)).float().cuda(), (torch.arange(12) % 3).int().cuda()

    def step():
        qt, kt = ops.head_norm_rotary(ctx, q, k, w, w, pos, freq, axis, kind="layer")
        out, saved = ops.diff_attention(ctx, qt, kt, v, lam, seqs, save=True)
        dq, dk, dv, dlam = ops.diff_attention_backward(ctx, dout, qt, kt, v, lam, seqs, out, saved)
        return (out, dv, dlam, *ops.head_norm_rotary_backward(ctx, dq, dk, q, k, w, w, pos, freq, axis, kind="layer", dpositions=True))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        for t in (q, k, v, dout):
            t.copy_(rand(g, *t.shape, dtype=dt))
        want = step()
        torch.cuda.synchronize()
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_a_recorded_backward_pass(ctx):
    """Through the autograd functions: recorded and replayed where no eager graph
    of the same leaves lives, refused where one does (autograd would hand the
    gradients over on that one's stream); the forward pass alone is recorded either way."""
    g = torch.Generator().manual_seed(6)
    leaf = [rand(g, *s, dtype=torch.float32).cuda().requires_grad_(True) for s in ((40, 4, 2, 16), (40, 2, 2, 16), (16,), (16,))]
    pos, freq, axis = torch.rand(40, 1, generator=g).cuda(), torch.rand(8, generator=g).cuda(), torch.zeros(8, dtype=torch.int32).cuda()
    v, lam, seqs = rand(g, 40, 2, 32, dtype=torch.float32).cuda(), torch.rand(4, generator=g).cuda(), ops.Sequences(ctx, [0, 15, 40])

    def loss():
        q, k = ops.HeadNormRotaryFn.apply(ctx, *leaf, pos, freq, axis, {})
        return ops.DiffAttentionFn.apply(ctx, q, k, v, lam, seqs).square().sum()

    want = torch.autograd.grad(loss(), leaf)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = torch.autograd.grad(loss(), leaf)
    for _ in range(3):
        for t in grads:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, want))
    alive = loss()
    torch.cuda.synchronize()
    with pytest.raises(capi.MtpxError, match="earlier graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(loss(), leaf)
    forward = torch.cuda.CUDAGraph()
    with torch.cuda.graph(forward):
        out = loss().detach()
    forward.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, alive.detach())
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(alive, leaf), want))


def test_two_graphs_share_what_they_may(ctx):
    """Two recorded steps over one cache from one memory pool, replayed in turn."""
    g = torch.Generator().manual_seed(8)
    c = PO.pool(g, [700, 90], 16, 2, 64, torch.bfloat16)
    kp, vp, table = (c[n].cuda() for n in ("k_pages", "v_pages", "table"))
    lam, off, lengths = torch.rand(8, generator=g).cuda(), i32(0, 1, 2), i32(700, 90)
    one, two = (rand(g, 2, 8, 2, 64, dtype=torch.bfloat16).cuda() for _ in range(2))
    want = [ops.diff_attention_paged(ctx, q, kp, vp, lam, table, off, lengths, max_rows=1) for q in (one, two)]
    torch.cuda.synchronize()
    graphs, outs, pool = [], [], torch.cuda.graph_pool_handle()
    for q in (one, two):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=pool):
            outs.append(ops.diff_attention_paged(ctx, q, kp, vp, lam, table, off, lengths, max_rows=1))
    for _ in range(3):
        for graph, out, w in zip(graphs, outs, want):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, w)


@dtypes
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 64), (6, 3, 24), (16, 2, 128)])
def test_a_block_is_served_as_it_was_trained(ctx, dtype, heads, kv, dim):
    """Sequences that come in chunks of different sizes through the cache give
    what the training path gives for them whole."""
    g = torch.Generator().manual_seed(dim)
    lengths, page, rot = [150, 61, 1, 333], 16, dim // 2 * 2
    ends = np.concatenate([[0], np.cumsum(lengths)])
    rows = int(ends[-1])
    q, k, v = (rand(g, rows, *s, dtype=dtype).cuda() for s in ((heads, 2, dim), (kv, 2, dim), (kv, 2 * dim)))
    wq, wk, lam = (1 + rand(g, dim, dtype=dtype, scale=0.2)).cuda(), (1 + rand(g, dim, dtype=dtype, scale=0.2)).cuda(), torch.rand(heads, generator=g).cuda()
    pos = torch.from_numpy(np.concatenate([np.arange(n) for n in lengths])).int()[:, None].cuda()
    freq, axis = (10000.0 ** (-torch.arange(rot // 2) / (rot // 2))).float().cuda(), torch.zeros(rot // 2, dtype=torch.int32).cuda()
    qt, kt = ops.head_norm_rotary(ctx, q, k, wq, wk, pos, freq, axis)
    whole = ops.diff_attention(ctx, qt, kt, v, lam, ops.Sequences(ctx, ends), causal=True)
    total = sum(-(-n // page) for n in lengths)
    kp, vp = torch.full((total, page, kv, 2, dim), float("nan"), dtype=dtype).cuda(), torch.full((total, page, kv, 2 * dim), float("nan"), dtype=dtype).cuda()
    table, at = torch.full((len(lengths), 30), -1, dtype=torch.int32), 0
    for i, n in enumerate(lengths):
        table[i, :-(-n // page)] = torch.arange(at, at + -(-n // page))
        at += -(-n // page)
    table, served, done = table.cuda(), torch.zeros_like(whole), [0] * len(lengths)
    rng = np.random.RandomState(1)
    while any(d < n for d, n in zip(done, lengths)):
        new = [int(min(n - d, rng.choice([0, 1, 1, 30, 100]))) for d, n in zip(done, lengths)]
        at = torch.cat([torch.arange(ends[i] + done[i], ends[i] + done[i] + m) for i, m in enumerate(new)]).cuda()
        done = [d + m for d, m in zip(done, new)]
        off = torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).cuda()
        rows_now = [t[at] for t in (q, k, v, pos)]
        turned = ops.append_paged(ctx, rows_now[1], rows_now[2], kp, vp, table, off, i32(*done), rows_now[3], freq, axis, q=rows_now[0],
                                  kind="rms", q_weight=wq, k_weight=wk)
        assert torch.equal(turned, qt[at])  # the same rows, normed and turned
        served[at] = ops.diff_attention_paged(ctx, turned, kp, vp, lam, table, off, i32(*done), max_rows=max(max(new), 1))
    r = OO.attention(qt.double().cpu(), kt.double().cpu(), v.double().cpu(), lam.double().cpu(), dim ** -0.5, ends, ends, True)
    f32 = OO.F32 * (16 + 4 * dim + 333 + 4 * r["scores"])
    tiny = 2.0 ** -25 * 333 * 8 if dtype == torch.float16 else 0.0
    # each of the two takes a rounding of P and one of its own
    over = (served - whole).double().abs().cpu() - 2 * (1.25 * 2 * OO.UNIT[dtype] + f32) * r["|out|"] - 2 * tiny
    assert float(over.max()) <= 0.0


def test_refused_on_the_device(ctx):
    q, pos = torch.zeros(2, 1, 8, device="cuda"), torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    freq, axis = torch.ones(4, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    with pytest.raises(capi.MtpxError, match="integer positions"):
        ops.head_norm_rotary_backward(ctx, q, None, q, None, None, None, pos, freq, axis, dpositions=True)
    with pytest.raises(capi.MtpxError, match="dim beyond 256"):
        ops.head_norm_rotary(ctx, torch.zeros(2, 1, 300, device="cuda"), None, None, None, pos, freq, axis)
    with pytest.raises(capi.MtpxError, match="rotated"):
        ops.head_norm_rotary(ctx, q[..., :6], None, None, None, pos, freq, axis)
    kp, vp = torch.zeros(3, 4, 1, 2, 132, device="cuda"), torch.zeros(3, 4, 1, 264, device="cuda")
    with pytest.raises(capi.MtpxError, match="dim beyond 128"):
        ops.diff_attention_paged(ctx, torch.zeros(2, 1, 2, 132, device="cuda"), kp, vp, torch.zeros(1, device="cuda"),
                                 i32(0)[None], i32(0, 2), i32(2))


def test_threads_of_their_own(ctx):
    """Two threads at once, each with its context and stream: a call leaves the interpreter while it queues its work."""
    g = torch.Generator().manual_seed(11)
    c = PO.pool(g, [300, 40, 77], 16, 2, 32, torch.bfloat16)
    q, k, v = (rand(g, *s, dtype=torch.bfloat16).cuda() for s in ((20, 4, 2, 32), (20, 2, 2, 32), (20, 2, 64)))
    w, lam, pos = rand(g, 32, dtype=torch.bfloat16).cuda(), torch.rand(4, generator=g).cuda(), torch.rand(20, 2, generator=g).cuda()
    freq, axis = torch.rand(16, generator=g).cuda(), (torch.arange(16) % 2).int().cuda()
    table, off, n = c["table"].cuda(), i32(0, 12, 13, 20), i32(300, 40, 77)

    def step(own):
        kp, vp = c["k_pages"].cuda(), c["v_pages"].cuda()
        qt = ops.append_paged(own, k, v, kp, vp, table, off, n, pos, freq, axis, q=q, kind="rms", q_weight=w)
        return (*ops.head_norm_rotary(own, q, k, w, w, pos, freq, axis), ops.diff_attention_paged(own, qt, kp, vp, lam, table, off, n))

    want = step(ctx)
    torch.cuda.synchronize()
    wrong, failed = [], []

    def work():
        try:
            own, stream = capi.Context(0), torch.cuda.Stream()
            for _ in range(40):
                with torch.cuda.stream(stream):
                    got = step(own)
                stream.synchronize()
                wrong.extend(1 for a, b in zip(got, want) if not torch.equal(a, b))
            own.close()
        except Exception as e:  # noqa: BLE001 -- a thread's failure is the test's
            failed.append(e)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed and not wrong


@dtypes
def test_a_cache_without_room(ctx, dtype):
    """Tables of no pages and pools of none: nothing is put anywhere, no row sees a key."""
    q, k, v = torch.ones(3, 2, 2, 16, dtype=dtype).cuda(), torch.ones(3, 1, 2, 16, dtype=dtype).cuda(), torch.ones(3, 1, 32, dtype=dtype).cuda()
    pos, freq, axis, lam = torch.ones(3, 1).cuda(), torch.ones(4).cuda(), torch.zeros(4, dtype=torch.int32).cuda(), torch.ones(2).cuda()
    off, n = i32(0, 1, 3), i32(5, 2)
    for pages, table in ((3, torch.zeros(2, 0, dtype=torch.int32).cuda()), (0, torch.zeros(2, 2, dtype=torch.int32).cuda())):
        kp, vp = torch.full((pages, 4, 1, 2, 16), 7.0, dtype=dtype).cuda(), torch.full((pages, 4, 1, 32), 7.0, dtype=dtype).cuda()
        ops.append_paged(ctx, k, v, kp, vp, table, off, n, pos, freq, axis)
        assert bool((kp == 7.0).all()) and bool((vp == 7.0).all())
        for causal in (True, False):
            out = ops.diff_attention_paged(ctx, q, kp, vp, lam, table, off, n, causal=causal)
            assert float(out.abs().max()) == 0.0
