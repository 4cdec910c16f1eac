"""The paged cache and the norms of heads, what needs no GPU: the binding's
structures against the header's, refusals before any device work, how the work
is split, the oracle's own gradients against differences, autograd over a
stand-in."""
import ctypes as C
import os
import random
import shutil
import subprocess

import pytest
import torch

import paged_oracle as PO
from mtpx import capi, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PAIRS = {"mtpx_head_norm_rotary_request": ops.HeadNormRequest, "mtpx_pages": ops.Pages,
         "mtpx_append_paged_request": ops.AppendRequest, "mtpx_diff_attention_paged_request": ops.PagedRequest}


@pytest.fixture(scope="module")
def calls(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc is not available")
    exe = str(tmp_path_factory.mktemp("calls") / "paged_calls")
    subprocess.run([hipcc, "-O1", "-std=c++17", "-w", "-I", os.path.join(ROOT, "include"),
                    "-I", os.path.join(ROOT, "imr-mlp_amd", "csrc"),
                    os.path.join(ROOT, "tests", "paged_calls.cpp"), "-o", exe], check=True)

    def run(*args):
        out = subprocess.run([exe, *map(str, args)], check=True, capture_output=True, text=True, timeout=60).stdout
        return [line.split() for line in out.splitlines()]

    return run


def test_structures_match_the_header(workdir):
    src, exe = os.path.join(workdir, "paged_layout.c"), os.path.join(workdir, "paged_layout")
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "mtpx.h"', "int main(void) {"]
    want = []
    for name, cls in PAIRS.items():
        lines.append('printf("%%zu\\n", sizeof(%s));' % name)
        want.append(C.sizeof(cls))
        for f, _ in cls._fields_:
            lines.append('printf("%%zu\\n", offsetof(%s, %s));' % (name, f.rstrip("_")))
            want.append(getattr(cls, f).offset)
    open(src, "w").write("\n".join(lines + ["return 0; }"]))
    subprocess.run([os.environ.get("CC", "gcc"), "-I", os.path.dirname(capi.HEADER), src, "-o", exe], check=True)
    got = [int(v) for v in subprocess.run([exe], check=True, capture_output=True).stdout.split()]
    assert got == want


def test_packed_requests_are_the_structures():
    """A request packed as a flat list of numbers, field by field."""
    for pack, cls in ((ops._pack_heads, ops.HeadNormRequest), (ops._pack_append, ops.AppendRequest), (ops._pack_paged, ops.PagedRequest)):
        def flat(c):
            return [t for _, f in c._fields_ for t in (flat(f) if issubclass(f, C.Structure) else [f])]

        def read(s):
            for n, f in s._fields_:
                v = getattr(s, n)
                yield from read(v) if isinstance(v, C.Structure) else [v or 0]

        values = [float(i + 1) if f is C.c_float else i + 1 for i, f in enumerate(flat(cls))]
        assert list(read(cls.from_buffer_copy(pack(*values)))) == values


def test_null_arguments_are_refused():
    L, n = ops._ops(), C.c_size_t()
    for name, cls in (("head_norm_rotary", ops.HeadNormRequest), ("head_norm_rotary_backward", ops.HeadNormRequest),
                      ("append_paged", ops.AppendRequest), ("diff_attention_paged", ops.PagedRequest)):
        assert getattr(L, "mtpx_" + name)(None, None) == -1
        assert getattr(L, "mtpx_" + name)(None, C.byref(cls())) == -1
    for name, cls in (("head_norm_rotary", ops.HeadNormRequest), ("diff_attention_paged", ops.PagedRequest)):
        assert getattr(L, "mtpx_%s_workspace" % name)(None, C.byref(cls()), C.byref(n)) == -1


def test_the_callers_device_stays_current(calls):
    for name, code, queued, after in calls("device"):
        assert (code, queued, after) == ("0", "0", "1"), name


def test_refusals_queue_nothing(calls):
    invalid, capacity = (str(capi.ERRORS_BY_NAME[n]) for n in ("MTPX_E_INVALID", "MTPX_E_CAPACITY"))
    big = {"head_many_rows", "head_wide", "append_many_sequences", "append_room", "append_pages", "attend_dim",
           "attend_rows", "attend_launch", "attend_room"}
    seen = calls("refuse")
    assert len(seen) == 52
    for name, code, queued in seen:
        assert code == (capacity if name in big else invalid) and queued == "-1", name


def test_a_keys_page_by_multiplication(calls):
    """The kernels' quotient by page_rows, for keys up to 2^30, at every multiple's edges that a sample meets."""
    rng = random.Random(1)
    for n, magic, shift in ((int(v) for v in line) for line in calls("pages")):
        keys = [0, 1, n - 1, n, 2 ** 30 - 1, 2 ** 30] + [k for _ in range(8) for m in (rng.randrange(1, 2 ** 30 // n + 1) * n,)
                                                      for k in (m - 1, m, m + 1)]
        assert magic < 2 ** 32
        for k in keys:
            assert ((2 * k * magic) >> 32) >> shift == k // n, (n, k)


def test_a_tile_costs_what_it_takes(calls):
    """Workgroups share keys by costs: a tile whose cost were below its steps would lose the last of them."""
    looked, wrong = (int(v) for v in calls("costs", 200000)[0])
    assert looked > 1000000 and wrong == 0


@pytest.mark.parametrize("seed", range(60))
def test_plans_cover_the_work(calls, seed):
    """Every sequence's columns lie in a narrow tile or in wide ones, a tile's
    number names one place, and the workspace holds all partial results."""
    rng = random.Random(seed)
    n, kv = rng.choice([1, 3, 64, 500, 5000]), rng.choice([1, 2, 8])
    group, dim, dtype = rng.choice([1, 3, 4, 17, 33, 64]), rng.choice([16, 64, 128]), rng.choice([0, 1])
    new = [rng.choice([0, 1, 1, 2, 40, 700]) if rng.random() < 0.5 and n < 5000 else 1 for _ in range(n)]
    first = 2
    rows = sum(new) + 5
    most = rng.choice([0, max(1, max(new))])
    page, width = rng.choice([16, 100]), rng.choice([3, 300])
    out = calls("plan", rows, n, most, group * kv, kv, dim, dtype, page, width)[0]
    code, limit, narrow, narrow_each, wide, wide_each, tiles, level, quarters, size = (int(v) for v in out)
    if rows * group * kv > (2 ** 32 - 1) // 512:
        return
    assert code == 0
    # columns of the tiles, as the kernels have them
    columns = {(0, 16): 64, (0, 64): 64, (0, 128): 32, (1, 16): 128, (1, 64): 128, (1, 128): 64}[dtype, dim]
    at, off = first, [first]
    for m in new:
        at += m
        off.append(at)
    place = {}
    for i, m in enumerate(new):
        if m == 0:
            continue
        if m * group <= limit:
            assert narrow > 0 and m * group <= 32 and (not narrow_each or narrow == n * kv)
            continue
        assert wide > 0
        start = off[i] * group // columns + i
        for t in range(-(-m * group // columns)):
            assert (level and t * n + i < tiles) or start + t < tiles
            assert start + t not in place
            place[start + t] = i
    # the number of a tile leads back to its sequence
    starts = [off[i] * group // columns + i for i in range(n)]
    for t, i in place.items():
        assert max(j for j in range(n) if starts[j] <= t) == i
    if wide and wide_each:
        assert wide == (tiles + quarters) * kv
    assert not level or wide_each
    wide_part = 2 * 4 * (4 + 2 * (32 if dim <= 32 else 64 if dim <= 64 else 128))
    want = 0 if narrow_each or narrow < 2 else narrow * 2 * 32 * wide_part
    want += 0 if wide_each or wide < 2 else wide * 2 * columns * wide_part
    assert size == want


class _Ctx:
    device, h, workspaces = 0, None, {}


def test_host_tensors_are_refused():
    x, pos, freq, axis = torch.zeros(2, 1, 4), torch.zeros(2, 3), torch.ones(2), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(capi.MtpxError):
        ops.head_norm_rotary(_Ctx, x, None, None, None, pos, freq, axis)
    k, v, kp, vp = torch.zeros(2, 1, 2, 4), torch.zeros(2, 1, 8), torch.zeros(3, 4, 1, 2, 4), torch.zeros(3, 4, 1, 8)
    table, off, n = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(capi.MtpxError):
        ops.append_paged(_Ctx, k, v, kp, vp, table, off, n, pos, freq, axis)
    with pytest.raises(capi.MtpxError):
        ops.diff_attention_paged(_Ctx, k, kp, vp, torch.zeros(1), table, off, n)


class _Library:
    """Counts calls; every call succeeds."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(h, req, *rest):
            self.calls.append(name)
            return 0

        return call


class _OnHost(_Ctx):
    def _check(self, rc, what=""):
        assert rc == 0


@pytest.fixture
def on_host(monkeypatch):
    """The binding's own checks, with host tensors taken for the device's."""
    lib = _Library()
    monkeypatch.setattr(ops, "_ops", lambda: lib)
    monkeypatch.setattr(ops, "_stream", lambda ctx: 0)
    monkeypatch.setattr(ops, "_workspace", lambda ctx, size: torch.empty(max(size, 1), dtype=torch.uint8))
    ctx = _OnHost()
    ctx.device, ctx.workspaces = torch.zeros(1).get_device(), {}
    ctx.lib = lib
    return ctx


def _heads(**change):
    c = dict(q=torch.zeros(4, 2, 2, 8), k=torch.zeros(4, 1, 2, 8), wq=torch.ones(8), wk=torch.ones(8), pos=torch.zeros(4, 3),
             freq=torch.ones(4), axis=torch.zeros(4, dtype=torch.int32), kw={})
    c.update(change)
    return [c[n] for n in ("q", "k", "wq", "wk", "pos", "freq", "axis")], c["kw"]


@pytest.mark.parametrize("change", [
    dict(k=torch.zeros(4, 1, 8)), dict(k=torch.zeros(3, 1, 2, 8)), dict(k=torch.zeros(4, 1, 2, 6)), dict(k=torch.zeros(4, 0, 2, 8)),
    dict(k=torch.zeros(4, 1, 2, 8, dtype=torch.bfloat16)), dict(q=torch.zeros(4, 2, 3, 8), k=None), dict(wq=torch.ones(7)),
    dict(wk=torch.ones(8, dtype=torch.float64)), dict(pos=torch.zeros(5, 3)), dict(pos=torch.zeros(4, 3, dtype=torch.int16)),
    dict(freq=torch.ones(4, dtype=torch.float64)), dict(axis=torch.zeros(3, dtype=torch.int32)),
    dict(q=torch.zeros(4, 2, 8, 2).transpose(2, 3)), dict(q=torch.zeros(4, 2, 2, 8, dtype=torch.int32)), dict(kw=dict(kind="none"))])
def test_refused_heads(on_host, change):
    given, kw = _heads(**change)
    with pytest.raises(capi.MtpxError):
        ops.head_norm_rotary(on_host, *given, **kw)
    with pytest.raises(capi.MtpxError):
        ops.head_norm_rotary_backward(on_host, given[0], given[1], *given, **kw)
    assert "mtpx_head_norm_rotary" not in on_host.lib.calls and "mtpx_head_norm_rotary_backward" not in on_host.lib.calls


def _cache(**change):
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    c = dict(k=torch.zeros(6, 1, 2, 8), v=torch.zeros(6, 1, 16), kp=torch.zeros(5, 4, 1, 2, 8), vp=torch.zeros(5, 4, 1, 16), table=i(2, 3),
             off=i(3), n=i(2), pos=torch.zeros(6, 1), freq=torch.ones(4), axis=i(4), q=torch.zeros(6, 2, 2, 8), lam=torch.zeros(2), kw={})
    c.update(change)
    return c


def _append(ctx, c):
    return ops.append_paged(ctx, *(c[n] for n in ("k", "v", "kp", "vp", "table", "off", "n", "pos", "freq", "axis")), q=c["q"], **c["kw"])


def _attend(ctx, c):
    return ops.diff_attention_paged(ctx, *(c[n] for n in ("q", "kp", "vp", "lam", "table", "off", "n")), **c["kw"])


@pytest.mark.parametrize("change", [
    dict(kp=torch.zeros(5, 4, 1, 16)), dict(vp=torch.zeros(5, 3, 1, 16)), dict(vp=torch.zeros(4, 4, 1, 16)), dict(kp=torch.zeros(5, 4, 1, 2, 8).half()),
    dict(table=torch.zeros(3, 3, dtype=torch.int32)), dict(table=torch.zeros(2, 3, dtype=torch.int64)),
    dict(table=torch.zeros(3, 2, dtype=torch.int32).T), dict(off=torch.zeros(2, dtype=torch.int32)), dict(n=torch.zeros(2, dtype=torch.int64)),
    dict(n=torch.zeros(2, 1, dtype=torch.int32))])
def test_refused_caches(on_host, change):
    for call in (_append, _attend):
        with pytest.raises(capi.MtpxError):
            call(on_host, _cache(**change))
    assert not any(n in ("mtpx_append_paged", "mtpx_diff_attention_paged") for n in on_host.lib.calls)


@pytest.mark.parametrize("change", [
    dict(v=torch.zeros(6, 1, 15)), dict(v=torch.zeros(5, 1, 16)), dict(k=torch.zeros(6, 2, 2, 8)), dict(q=torch.zeros(5, 2, 2, 8)),
    dict(q=torch.zeros(6, 2, 2, 8, dtype=torch.half)), dict(kw=dict(kind="all")), dict(kw=dict(k_weight=torch.ones(8))),
    dict(kw=dict(kind="rms", k_weight=torch.ones(9))), dict(q=None, kw=dict(out=torch.zeros(6, 2, 2, 8))),
    dict(kw=dict(out=torch.zeros(6, 2, 2, 7)))])
def test_refused_appends(on_host, change):
    with pytest.raises(capi.MtpxError):
        _append(on_host, _cache(**change))
    assert "mtpx_append_paged" not in on_host.lib.calls


@pytest.mark.parametrize("change", [
    dict(lam=torch.zeros(3)), dict(lam=torch.zeros(2).double()), dict(q=torch.zeros(6, 2, 8)), dict(q=torch.zeros(6, 2, 2, 7)),
    dict(kw=dict(max_rows=0)), dict(kw=dict(out=torch.zeros(6, 2, 15)))])
def test_refused_attention(on_host, change):
    with pytest.raises(capi.MtpxError):
        _attend(on_host, _cache(**change))
    assert "mtpx_diff_attention_paged" not in on_host.lib.calls


def test_what_is_not_refused(on_host):
    assert _attend(on_host, _cache()).shape == (6, 2, 16) and _append(on_host, _cache()).shape == (6, 2, 2, 8)
    assert _append(on_host, _cache(q=None)) is None
    given, kw = _heads()
    assert [t.shape for t in ops.head_norm_rotary(on_host, *given, **kw)] == [given[0].shape, given[1].shape]
    assert on_host.lib.calls.count("mtpx_append_paged") == 2


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_oracle_gradients_against_differences(kind, interleaved):
    g = torch.Generator().manual_seed(5)
    x, dy = torch.randn(5, 3, 2, 10, generator=g).double(), torch.randn(5, 3, 2, 10, generator=g).double()
    w, pos, freq, axis = torch.rand(10, generator=g).double(), torch.rand(5, 3, generator=g).double(), torch.rand(4, generator=g).double(), torch.arange(4) % 3

    def loss(x, w, pos):
        return float((PO.forward(x, w, pos[:, axis] * freq, kind, 0.01, interleaved)[0] * dy).sum())

    grads = PO.backward(x, w, dy, pos[:, axis] * freq, freq, axis, 3, kind, 0.01, interleaved)
    at = [x, w, pos]
    for i in range(3):
        d = torch.randn(at[i].shape, generator=g).double()
        h = 1e-5
        up, down = ([t + s * d if j == i else t for j, t in enumerate(at)] for s in (h, -h))
        # central differences: h^2 third derivatives (about 1e-8 here), cancellation 1e-16 / h
        assert abs((loss(*up) - loss(*down)) / (2 * h) - float((grads[i][0] * d).sum())) < 1e-6
        assert bool((grads[i][0].abs() <= grads[i][1] * (1 + 1e-12) + 1e-12).all())


class _OnStream(torch.autograd.Function):
    @staticmethod
    def forward(fn, x, note):
        fn.ctx = None
        ops._mark_leaves(fn)
        note.append(fn.next_functions[0][0].metadata)
        return x * 2

    @staticmethod
    def backward(fn, g):
        ops._same_streams(fn)
        return g * 2, None


class _Node:
    def __init__(self, is_cuda=True, **metadata):
        self.metadata, self.next_functions = dict(metadata), ()
        self.variable = type("V", (), dict(is_cuda=is_cuda))


def test_leaves_are_marked_by_the_first_graph(monkeypatch):
    """The mark lives as long as the leaf's end of a graph; recording beside another stream's raises."""
    x, note = torch.ones(2, requires_grad=True), []
    _OnStream.apply(x, note).sum().backward()
    assert ops._STREAM not in note[0]  # a host tensor has no stream
    monkeypatch.setattr(ops, "_Leaf", _Node)
    monkeypatch.setattr(ops, "_stream", lambda ctx: stream)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    fn = type("F", (), dict(ctx=None, next_functions=((_Node(), 0), (None, 0), (_Node(is_cuda=False), 0))))
    stream, capturing = 7, False
    ops._mark_leaves(fn)
    stream = 9
    ops._mark_leaves(fn)
    assert [n.metadata for n, _ in fn.next_functions if n is not None] == [{ops._STREAM: 7}, {}]
    ops._same_streams(fn)
    capturing = True
    with pytest.raises(capi.MtpxError, match="earlier graph"):
        ops._same_streams(fn)
    stream = 7
    ops._same_streams(fn)
