"""A cache in pages: rows appended (mtpx.ops.append_paged) and attention over
it (mtpx.ops.diff_attention_paged) against their formulas in 64 bits, with the
bounds of the other operators: one rounding of what a kernel rounds, 2^-24
times the length of a 32-bit sum, times the size of what is added up.  float16
numbers below 2^-14 lie 2^-24 apart: a rounding there is off by up to 2^-25."""
import math

import numpy as np
import pytest
import torch

import ops_oracle as OO
import paged_oracle as PO
from mtpx import ops
from test_ops_gpu import close, dtypes, rand

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32)


def offsets(new, first=0):
    return i32(np.concatenate([[0], np.cumsum(new)]) + first)


# ---- append ---------------------------------------------------------------------


def check_append(ctx, dtype, new, lengths, page, heads, kv, dim, rotated, kind, interleaved, before=0, behind=0,
                 seed=0, spoil=None, align=0):
    """New rows of each sequence, its rows with them, rows of no sequence before
    and behind; spoil(table) changes the tables."""
    g = torch.Generator().manual_seed(seed + dim)
    rows = before + sum(new) + behind
    c = PO.pool(g, np.maximum(lengths, 0), page, kv, dim, dtype, fill=3.0)
    if spoil is not None:
        spoil(c["table"], len(c["k_pages"]))
    pairs = rotated // 2
    q, k, v = rand(g, rows, heads, 2, dim, dtype=dtype), rand(g, rows, kv, 2, dim, dtype=dtype), rand(g, rows, kv, 2 * dim, dtype=dtype)
    wq, wk = (None, None) if kind == "none" else (1 + rand(g, dim, dtype=dtype), 1 + rand(g, dim, dtype=dtype))
    pos = torch.randint(0, 5000, (rows, 2), generator=g)
    freq, axis = (100.0 ** (-torch.arange(pairs) / max(pairs, 1))).float(), (torch.arange(pairs) % 2).int()
    off = offsets(new, before)
    on = lambda t: None if t is None else t.cuda()  # noqa: E731
    # what lies in the pages goes at any alignment
    room = torch.empty(c["k_pages"].numel() + align, dtype=dtype).cuda()[align:]
    k_pages = room.view(c["k_pages"].shape).copy_(c["k_pages"])
    v_pages = on(c["v_pages"])
    out = torch.full((rows, heads, 2, dim), 5.0, dtype=dtype).cuda()
    got = ops.append_paged(ctx, on(k), on(v), k_pages, v_pages, on(c["table"]), on(off), on(i32(lengths)), on(pos), on(freq),
                           on(axis), q=on(q), kind=kind, q_weight=on(wq), k_weight=on(wk), eps=1e-3, interleaved=interleaved, out=out)
    assert got is out
    theta = pos.double()[:, axis.long()] * freq.double()
    u, f32, tiny = OO.UNIT[dtype], OO.F32 * (32 + 2 * dim), 2.0 ** -25 if dtype == torch.float16 else 0.0
    yq, sq = PO.forward(q, wq, theta, kind, 1e-3, interleaved)
    yk, sk = PO.forward(k, wk, theta, kind, 1e-3, interleaved)
    held = slice(before, before + sum(new))
    if sum(new):
        assert float(((out.double().cpu() - yq).abs() - u * yq.abs() - f32 * sq - tiny)[held].max()) <= 0.0
    rest = torch.ones(rows, dtype=torch.bool)
    rest[held] = False
    assert torch.equal(out.cpu()[rest], torch.full_like(out.cpu()[rest], 5.0))
    # the pools: every row that went in, and all others as they were
    want_k, want_v, bound = c["k_pages"].double(), c["v_pages"].clone(), torch.zeros(c["k_pages"].shape).double()
    for i, (m, n) in enumerate(zip(new, lengths)):
        for j in range(m):
            t, r = n - m + j, int(off[i]) + j
            if t < 0 or t >= c["table"].shape[1] * page:
                continue
            p = int(c["table"][i, t // page])
            if 0 <= p < len(want_k):
                want_k[p, t % page], want_v[p, t % page] = yk[r], v[r]
                bound[p, t % page] = u * yk[r].abs() + f32 * sk[r] + tiny
    assert torch.equal(v_pages.cpu(), want_v)
    assert float(((k_pages.double().cpu() - want_k).abs() - bound).max()) <= 0.0


@dtypes
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("kind", ["none", "rms", "layer"])
@pytest.mark.parametrize("new,lengths,page,heads,kv,dim,rotated", [
    ([1], [1], 1, 1, 1, 2, 2), ([1, 1, 1], [7, 16, 33], 16, 8, 2, 64, 64), ([5, 0, 40], [5, 3, 90], 16, 4, 4, 40, 36),
    ([70], [170], 3, 2, 1, 128, 96), ([3, 2], [100, 101], 100, 3, 3, 7, 6), ([2, 9], [9, 9], 8, 1, 1, 256, 128)])
def test_append(ctx, dtype, interleaved, kind, new, lengths, page, heads, kv, dim, rotated):
    check_append(ctx, dtype, new, lengths, page, heads, kv, dim, rotated, kind, interleaved, before=2, behind=5)
    check_append(ctx, dtype, new, lengths, page, heads, kv, dim, rotated, kind, interleaved, align=1)


def test_append_drops_what_has_no_place(ctx):
    """Rows before a sequence's start and beyond its room, negative lengths,
    pages that are none: dropped, everything else whole."""
    def spoil(table, pages):
        table[0, 1], table[2, 0], table[3, 0] = -1, pages, 2 ** 31 - 1

    check_append(ctx, torch.bfloat16, [4, 6, 3, 5], [20, 2, 9, 5], 8, 2, 2, 16, 16, "rms", False, spoil=spoil)
    check_append(ctx, torch.float32, [4, 40, 3], [-2, 400, 3], 8, 2, 1, 16, 8, "none", True, spoil=lambda t, n: t[1, -4:].fill_(-1))


def test_append_among_many_sequences(ctx):
    """The search for a row's sequence over several rounds, empty ones among them."""
    g = np.random.RandomState(3)
    for n in (63, 64, 65, 300, 5000):
        new = g.randint(0, 4, n)
        lengths = new + g.randint(0, 5, n)
        check_append(ctx, torch.bfloat16, new.tolist(), lengths.tolist(), 4, 1, 1, 8, 8, "none", False, behind=3, seed=n)


def test_append_in_place_and_in_one_pool(ctx):
    """Queries in their own place; keys and values side by side in one tensor, and heads outside slots."""
    g = torch.Generator().manual_seed(2)
    k, v, q = rand(g, 9, 2, 2, 32, dtype=torch.bfloat16).cuda(), rand(g, 9, 2, 64, dtype=torch.bfloat16).cuda(), rand(g, 9, 4, 2, 32, dtype=torch.bfloat16).cuda()
    table, off, length = i32([[3, 0], [2, 5]]).cuda(), i32([0, 4, 9]).cuda(), i32([6, 9]).cuda()
    pos, freq, axis = torch.arange(9)[:, None].cuda(), torch.rand(16, generator=g).cuda(), torch.zeros(16, dtype=torch.int32).cuda()
    plain = torch.zeros(6, 8, 2, 2, 32, dtype=torch.bfloat16).cuda(), torch.zeros(6, 8, 2, 64, dtype=torch.bfloat16).cuda()
    want = ops.append_paged(ctx, k, v, *plain, table, off, length, pos, freq, axis, q=q, kind="rms")
    both = torch.zeros(6, 2, 2, 8, 64, dtype=torch.bfloat16).cuda()  # pages, keys or values, heads, slots
    kp, vp = both[:, 0].unflatten(3, (2, 32)).permute(0, 2, 1, 3, 4), both[:, 1].permute(0, 2, 1, 3)
    place = q.clone()
    got = ops.append_paged(ctx, k, v, kp, vp, table, off, length, pos, freq, axis, q=place, kind="rms", out=place)
    assert got is place and torch.equal(got, want)
    assert torch.equal(kp, plain[0]) and torch.equal(vp, plain[1])
    assert ops.append_paged(ctx, k, v, kp, vp, table, off, length, pos, freq, axis, kind="rms") is None
    assert torch.equal(kp, plain[0])
    # nothing of a norm: the rotation alone is mtpx.ops.rotary's, bit for bit
    ops.append_paged(ctx, k, v, *plain, table, off, length, pos, freq, axis)
    assert torch.equal(plain[0][2, 4:8], ops.rotary(ctx, k.flatten(1, 2), pos, freq, axis).view(k.shape)[4:8])


# ---- attention --------------------------------------------------------------------


def check_paged(ctx, dtype, new, lengths, page, heads, kv, dim, causal=True, before=0, behind=0, max_rows=None, seed=0,
                scale=None, hidden=0.0, align=0):
    """hidden: the share of pages that the tables do not name."""
    g = torch.Generator().manual_seed(seed + dim + heads)
    rows = before + sum(new) + behind
    c = PO.pool(g, lengths, page, kv, dim, dtype)
    q, lam = rand(g, rows, heads, 2, dim, dtype=dtype, scale=1.5), torch.rand(heads, generator=g) - 0.2
    mask = None
    if hidden:
        mask, at = torch.ones(len(c["k"]), dtype=torch.bool), 0
        for i, n in enumerate(lengths):
            for p in range(-(-n // page)):
                if torch.rand((), generator=g) < hidden:
                    c["table"][i, p] = [-1, len(c["k_pages"]), 2 ** 31 - 1, -2 ** 31][p % 4]
                    mask[at + p * page:at + min(n, (p + 1) * page)] = False
            at += n
    store = torch.empty(q.numel() + align, dtype=dtype).cuda()[align:]
    qd = store.view(q.shape).copy_(q)
    out = torch.full((rows, heads, 2 * dim), 7.0, dtype=dtype).cuda()
    args = (qd, c["k_pages"].cuda(), c["v_pages"].cuda(), lam.cuda(), c["table"].cuda(), offsets(new, before).cuda(), i32(lengths).cuda())
    kw = dict(causal=causal, scale=scale)
    got = ops.diff_attention_paged(ctx, *args, max_rows=max_rows, out=out, **kw)
    assert got is out
    held = slice(before, before + sum(new))
    k_off = np.concatenate([[0], np.cumsum(lengths)])
    r = OO.attention(q[held].double(), c["k"].double(), c["v"].double(), lam.double(), dim ** -0.5 if scale is None else scale,
                     np.concatenate([[0], np.cumsum(new)]), k_off, causal, mask)
    longest = max(lengths, default=0)
    f32 = OO.F32 * (16 + 4 * dim + longest + 4 * r["scores"])
    tiny = 2.0 ** -25 * longest * 8 if dtype == torch.float16 else 0.0
    close(out[held], r["out"], r["|out|"], 1.25 * 2 * OO.UNIT[dtype] + f32, tiny)
    rest = torch.ones(rows, dtype=torch.bool)
    rest[held] = False
    assert torch.equal(out.cpu()[rest], torch.full_like(out.cpu()[rest], 7.0))
    again = ops.diff_attention_paged(ctx, *args, max_rows=max_rows, **kw)
    assert torch.equal(again[held], out[held])


BATCHES = [([1], [1], 16), ([1, 1, 1], [5, 64, 0], 16), ([1, 1, 1, 1], [700, 31, 32, 2100], 64), ([3, 1, 0, 2], [3, 40, 5, 130], 1),
           ([70], [70], 16), ([40, 1, 150], [300, 1, 150], 24), ([5, 9], [1, 4], 8), ([33, 64, 17], [1500, 1100, 17], 100),
           ([200], [1300], 3)]


@dtypes
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new,lengths,page", BATCHES)
@pytest.mark.parametrize("heads,kv,dim", [(2, 2, 32), (8, 2, 64), (6, 1, 128)])
def test_paged(ctx, dtype, causal, new, lengths, page, heads, kv, dim):
    check_paged(ctx, dtype, new, lengths, page, heads, kv, dim, causal, before=1, behind=2)
    check_paged(ctx, dtype, new, lengths, page, heads, kv, dim, causal, max_rows=max(new))


@dtypes
@pytest.mark.parametrize("dim", [1, 5, 8, 16, 24, 40, 72, 100, 127])
def test_paged_odd_dims(ctx, dtype, dim):
    check_paged(ctx, dtype, [37, 1, 90], [400, 77, 90], 16 if dim % 2 else 6, 3, 3, dim, scale=0.3)
    check_paged(ctx, dtype, [1, 2], [600, 77], 5, 4, 2, dim, max_rows=2, align=1)


@dtypes
@pytest.mark.parametrize("heads,kv,dim", [(8, 1, 16), (17, 1, 32), (33, 1, 64), (40, 1, 128), (36, 3, 64)])
def test_paged_shared_heads(ctx, dtype, heads, kv, dim):
    """Groups of heads that fill one block of columns, several, and part of one."""
    check_paged(ctx, dtype, [1, 1, 1], [90, 1, 1300], 32, heads, kv, dim, max_rows=1)
    check_paged(ctx, dtype, [3, 1, 20], [90, 1, 1300], 32, heads, kv, dim)


@dtypes
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("page", [2, 16, 128])
def test_paged_hidden_pages(ctx, dtype, causal, page):
    """Entries that name no page hide their keys; rows without any key give 0."""
    check_paged(ctx, dtype, [1, 60, 2, 1], [300, 1200, 2, 3000], page, 4, 2, 64, causal, hidden=0.4)
    check_paged(ctx, dtype, [1, 60], [300, 200], page, 2, 2, 24, causal, hidden=1.0)


@dtypes
def test_paged_broad_tiles(ctx, dtype):
    """Enough columns for tiles of 128, sequences that end inside one and begin in another."""
    new = [700, 1, 129, 3, 800, 0, 64, 395]
    check_paged(ctx, dtype, new, [n + 40 * i for i, n in enumerate(new)], 64, 32, 16, 32)


@dtypes
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new", [[520] * 8, [1500, 90, 700, 1, 5, 1900]])
def test_paged_a_tile_a_workgroup(ctx, dtype, causal, new):
    """So many tiles that each is a workgroup's: of sequences alike, and of others."""
    check_paged(ctx, dtype, new, [n + i for i, n in enumerate(new)], 48, 72, 72, 16, causal, behind=3, max_rows=max(new))


@dtypes
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("page", [2, 4, 8, 24, 100])
def test_paged_pages_of_runs(ctx, dtype, dim, page):
    """Pages that end inside a wave's rows of a tile, at the end of one of its loads or within one."""
    check_paged(ctx, dtype, [1, 70, 1], [500, 333, 77], page, 4, 2, dim, hidden=0.1)


@dtypes
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_paged_long_among_short(ctx, dtype, dim):
    """Shares of both widths beside each other, of fewer workgroups each; a tile a workgroup and parts of tiles."""
    check_paged(ctx, dtype, [1] * 12 + [90], [700 + 200 * i for i in range(12)] + [3000], 16, 4, 2, dim, max_rows=90)
    check_paged(ctx, dtype, [1] * 9 + [70, 40], [100 * i for i in range(1, 12)], 32, 2, 1, dim, max_rows=70)


@dtypes
def test_paged_large_scores(ctx, dtype):
    check_paged(ctx, dtype, [1, 60], [2000, 300], 16, 4, 2, 32, scale=12.0)


def test_paged_many_sequences(ctx):
    g = np.random.RandomState(5)
    new = g.randint(0, 3, 500)
    check_paged(ctx, torch.bfloat16, new.tolist(), (new + g.randint(0, 40, 500)).tolist(), 8, 2, 1, 32)
    new[::50] = 40
    check_paged(ctx, torch.bfloat16, new.tolist(), (new + g.randint(0, 40, 500)).tolist(), 8, 2, 1, 32)


def test_paged_thousands_of_sequences(ctx):
    """More than workgroups share: a tile of each is one workgroup's."""
    g = np.random.RandomState(6)
    new = g.randint(0, 2, 4200)
    new[7], new[4000] = 50, 9
    check_paged(ctx, torch.bfloat16, new.tolist(), (new + g.randint(0, 30, 4200)).tolist(), 8, 2, 1, 32)


@dtypes
def test_paged_layouts(ctx, dtype):
    """Keys and values in pools of different strides, one behind the other in one
    tensor, at any alignment, heads outside slots: the result of contiguous ones."""
    g = torch.Generator().manual_seed(12)
    lengths, new, page, kv, d = [500, 3, 90], [40, 1, 1], 32, 2, 64
    c = PO.pool(g, lengths, page, kv, d, dtype, fill=0.0)
    q, lam = rand(g, 42, 6, 2, d, dtype=dtype).cuda(), torch.rand(6, generator=g).cuda()
    k, v = c["k_pages"].cuda(), c["v_pages"].cuda()
    rest = (lam, c["table"].cuda(), offsets(new).cuda(), i32(lengths).cuda())
    want = ops.diff_attention_paged(ctx, q, k, v, *rest)
    n = len(k)
    apart = torch.zeros(n, page + 3, kv, 2 * d + 16, dtype=dtype).cuda()
    apart[:, :page, :, :2 * d] = v
    both = torch.stack([k.flatten(3), v], 1)  # pages, keys or values, slots, heads, elements
    heads_out = torch.stack([k.flatten(3).transpose(1, 2), v.transpose(1, 2)])
    odd = torch.zeros(k.numel() + 1, dtype=dtype).cuda()[1:].view(k.shape).copy_(k)
    for kp, vp in ((k, apart[:, :page, :, :2 * d]), (both[:, 0].unflatten(3, (2, d)), both[:, 1]),
                   (heads_out[0].transpose(1, 2).unflatten(3, (2, d)), heads_out[1].transpose(1, 2)), (odd, v)):
        assert torch.equal(ops.diff_attention_paged(ctx, q, kp, vp, *rest), want)
    wide = torch.zeros(3, c["table"].shape[1] + 5, dtype=torch.int32).cuda()
    wide[:, 2:2 + c["table"].shape[1]] = rest[1]
    part = wide[:, 2:2 + c["table"].shape[1]]
    assert part.stride(0) != part.shape[1]
    assert torch.equal(ops.diff_attention_paged(ctx, q, k, v, lam, part, *rest[2:]), want)


def test_lengths_beyond_the_room_and_below_zero(ctx):
    """A length counts what its table has room for, its rows' places those it says; below zero it is 0."""
    g = torch.Generator().manual_seed(1)
    c = PO.pool(g, [64, 64, 64], 16, 2, 32, torch.float32, width=4)
    q, lam = rand(g, 9, 2, 2, 32, dtype=torch.float32), torch.rand(2, generator=g)
    off = i32([0, 3, 6, 9]).cuda()
    args = (q.cuda(), c["k_pages"].cuda(), c["v_pages"].cuda(), lam.cuda(), c["table"].cuda(), off)
    for causal in (True, False):
        got = ops.diff_attention_paged(ctx, *args, i32([1000, 66, -5]).cuda(), causal=causal)
        want = ops.diff_attention_paged(ctx, *args, i32([64, 64, 0]).cuda(), causal=False)
        if causal:  # rows 63, 64 and 65 of the second sequence: all see its 64 keys
            assert torch.equal(got[:6], want[:6])
        else:
            assert torch.equal(got, want)
        assert float(got[6:].abs().max()) == 0.0


@pytest.mark.parametrize("n,rows", [(5, 1), (5, 90), (70, 7), (70, 90), (300, 90)])
def test_offsets_that_do_not_ascend(ctx, n, rows):
    """The same rows again and again, more of them than there are: no row is written, and the call ends."""
    g = torch.Generator().manual_seed(2)
    c = PO.pool(g, [128], 16, 2, 32, torch.bfloat16)
    table, lengths = c["table"].repeat(n, 1).cuda(), i32([128] * n).cuda()
    q, lam = rand(g, rows, 4, 2, 32, dtype=torch.bfloat16).cuda(), torch.rand(4, generator=g).cuda()
    out = torch.full((rows, 4, 64), 7.0, dtype=torch.bfloat16).cuda()
    for off in (i32([0, rows] * n)[:n + 1], i32([rows, 0] + [rows] * n)[:n + 1]):
        ops.diff_attention_paged(ctx, q, c["k_pages"].cuda(), c["v_pages"].cuda(), lam, table, off.cuda(), lengths, out=out)
        assert bool((out == 7.0).all())


def test_common_prefix_and_the_contiguous_cache(ctx):
    """Pages that several tables name; a row per sequence is diff_attention_cache's, up to the order of sums."""
    g = torch.Generator().manual_seed(7)
    c = PO.pool(g, [512], 32, 2, 64, torch.float32)
    table = c["table"][:, :16].repeat(3, 1).cuda()
    q, lam = rand(g, 3, 4, 2, 64, dtype=torch.float32).cuda(), torch.rand(4, generator=g).cuda()
    lengths = i32([512, 100, 33]).cuda()
    got = ops.diff_attention_paged(ctx, q, c["k_pages"].cuda(), c["v_pages"].cuda(), lam, table, i32([0, 1, 2, 3]).cuda(), lengths, max_rows=1)
    k, v = c["k"][None].expand(3, -1, -1, -1, -1).cuda(), c["v"][None].expand(3, -1, -1, -1).cuda()
    want = ops.diff_attention_cache(ctx, q, k, v, lam, lengths)
    assert float((got - want).abs().max()) < 512 * OO.F32 * float(c["v"].abs().max()) * 2


def test_offsets_beyond_32_bits(ctx):
    """Pages 2^31 + 2^20 elements apart in one allocation."""
    g = torch.Generator().manual_seed(1)
    apart, page, d = 2 ** 31 + 2 ** 20, 16, 32
    store = torch.zeros(apart + 40 * page * 2 * d, dtype=torch.bfloat16, device="cuda")
    far = store.as_strided((2, page, 1, 2, d), (apart, 2 * d, 2 * d, d, 1))
    rows, new = rand(g, 20, 1, 2, d, dtype=torch.bfloat16).cuda(), i32([0, 20]).cuda()
    q, lam, table, lengths = rand(g, 20, 4, 2, d, dtype=torch.bfloat16).cuda(), torch.rand(4, generator=g).cuda(), i32([[1, 0]]).cuda(), i32([20]).cuda()
    pos, none, axis = torch.zeros(20, 1).cuda(), torch.zeros(0).cuda(), torch.zeros(0, dtype=torch.int32).cuda()
    near = torch.zeros(2, page, 1, 2, d, dtype=torch.bfloat16, device="cuda")
    for t in (far, near):
        ops.append_paged(ctx, rows, rows.flatten(2), t, t.flatten(3), table, new, lengths, pos, none, axis)
    assert torch.equal(far, near) and torch.equal(near[1], rows[:16])
    for causal in (True, False):
        got, want = (ops.diff_attention_paged(ctx, q, t, t.flatten(3), lam, table, new, lengths, causal=causal) for t in (far, near))
        assert torch.equal(got, want)


def test_serving_a_graph(ctx):
    """A step as a program runs it, recorded once: rows normed, turned and
    appended, then attended to, with offsets, lengths and tables that change
    between replays; each replay against the eager step and against attention
    over the whole sequences."""
    g = torch.Generator().manual_seed(9)
    dt, heads, kv, d, page, seqs, rows = torch.bfloat16, 8, 2, 64, 16, 3, 40
    k_pages, v_pages = torch.zeros(30, page, kv, 2, d, dtype=dt).cuda(), torch.zeros(30, page, kv, 2 * d, dtype=dt).cuda()
    table = i32(np.random.RandomState(0).permutation(30).reshape(3, 10)).cuda()
    q, k, v = (torch.zeros(rows, *s, dtype=dt).cuda() for s in ((heads, 2, d), (kv, 2, d), (kv, 2 * d)))
    off, lengths, pos = torch.zeros(4, dtype=torch.int32).cuda(), torch.zeros(3, dtype=torch.int32).cuda(), torch.zeros(rows, 1).cuda()
    w, lam = (1 + rand(g, d, dtype=dt, scale=0.1)).cuda(), torch.rand(heads, generator=g).cuda()
    freq, axis = (100.0 ** (-torch.arange(32) / 32)).float().cuda(), torch.zeros(32, dtype=torch.int32).cuda()

    def step(kp, vp):
        turned = ops.append_paged(ctx, k, v, kp, vp, table, off, lengths, pos, freq, axis, q=q, kind="rms", q_weight=w, k_weight=w)
        return ops.diff_attention_paged(ctx, turned, kp, vp, lam, table, off, lengths)

    kept = [[] for _ in range(seqs)]
    first = True
    for new in ([30, 0, 10], [1, 1, 1], [1, 20, 1], [0, 1, 7], [1, 1, 1]):
        n = sum(new)
        off.copy_(offsets(new))
        lengths += i32(new).cuda()
        for t in (q, k, v):
            t[:n] = rand(g, n, *t.shape[1:], dtype=dt).cuda()
        pos[:n, 0] = torch.cat([torch.arange(int(lengths[i]) - m, int(lengths[i])) for i, m in enumerate(new)]).cuda().float()
        copies = k_pages.clone(), v_pages.clone()
        eager = step(*copies)
        torch.cuda.synchronize()
        if first:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step(k_pages, v_pages)
            first = False
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:n], eager[:n])
        assert torch.equal(k_pages, copies[0]) and torch.equal(v_pages, copies[1])
        at = 0
        for i, m in enumerate(new):
            kept[i].append((q[at:at + m].clone(), k[at:at + m].clone(), v[at:at + m].clone(), pos[at:at + m].clone()))
            at += m
        # the same rows as whole sequences, through the training path
        whole = [[torch.cat(t) for t in zip(*s)] for s in kept]
        ends = np.concatenate([[0], np.cumsum([len(s[0]) for s in whole])])
        qa, ka, va, pa = (torch.cat(t) for t in zip(*whole))
        qa, ka = ops.head_norm_rotary(ctx, qa, ka, w, w, pa, freq, axis)
        full = ops.diff_attention(ctx, qa, ka, va, lam, ops.Sequences(ctx, ends), causal=True)
        for i, m in enumerate(new):
            a, b = out[int(off[i]):int(off[i]) + m].double(), full[ends[i + 1] - m:ends[i + 1]].double()
            # two results in bfloat16, each with a rounding of P and its own: of values up to 4 or so
            assert m == 0 or float((a - b).abs().max()) <= 4 * OO.UNIT[dt] * float(va.abs().max()) * 2


def test_on_another_stream(ctx):
    g = torch.Generator().manual_seed(3)
    c = PO.pool(g, [90, 200], 16, 2, 32, torch.bfloat16)
    q, lam = rand(g, 12, 4, 2, 32, dtype=torch.bfloat16).cuda(), torch.rand(4, generator=g).cuda()
    args = (q, c["k_pages"].cuda(), c["v_pages"].cuda(), lam, c["table"].cuda(), i32([0, 2, 12]).cuda(), i32([90, 200]).cuda())
    want = ops.diff_attention_paged(ctx, *args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.diff_attention_paged(ctx, *args)
    side.synchronize()
    assert torch.equal(got, want)
