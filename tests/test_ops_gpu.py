"""Operators on device tensors (mtpx.ops) against their formulas in 64 bits.

Bounds are set element by element from what an element adds up: `u` is the
largest relative error of one rounding to the type (2^-8, 2^-11, 2^-24).  A
16-bit result takes one rounding of every factor that the kernels round (P,
dS, the saved results) and one of its own; sums in 32 bits add 2^-24 times
their length, and exp of a score s is off by 2^-24 |s| and a few units."""
import math

import numpy as np
import pytest
import torch

import ops_oracle as OO
from mtpx import capi, ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]
dtypes = pytest.mark.parametrize("dtype", DTYPES, ids=IDS)


def rand(g, *shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def close(got, want, size, factor, floor=0.0):
    """|got - want| <= factor * size + floor, element by element."""
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    assert bool(torch.isfinite(got).all())
    over = (got - want).abs() - factor * size - floor
    assert float(over.max() if over.numel() else -1.0) <= 0.0, float(((got - want).abs() / (factor * size + floor)).max())


# ---- rotary ---------------------------------------------------------------------


@dtypes
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,dim,rotated,kind", [
    (1, 1, 2, 2, torch.int64), (3, 32, 64, 64, torch.int32), (17, 5, 40, 36, torch.float32),
    (5, 2, 7, 6, torch.float64), (130, 3, 128, 96, torch.int64), (2, 1, 1024, 1024, torch.float32),
    (9, 70, 16, 0, torch.int32), (4, 1, 200, 200, torch.float64)])
def test_rotary(ctx, dtype, interleaved, rows, heads, dim, rotated, kind):
    g = torch.Generator().manual_seed(rows * dim)
    x, dy = rand(g, rows, heads, dim, dtype=dtype), rand(g, rows, heads, dim, dtype=dtype)
    real = kind.is_floating_point
    pos = torch.rand((rows, 4), generator=g).to(kind) if real else torch.randint(-9000, 90000, (rows, 4), generator=g).to(kind)
    freq = (6.2831853 * (1 + torch.arange(rotated // 2) // 3)).float() if real else (10000.0 ** (-torch.arange(rotated // 2) / max(1, rotated // 2))).float()
    axis = (torch.arange(rotated // 2) % 4).int()
    theta = pos.double()[:, axis.long()] * freq.double()
    dev = [t.cuda() for t in (x, pos, freq, axis)]
    y = ops.rotary(ctx, *dev, interleaved=interleaved)
    u = OO.UNIT[dtype]
    want, size = OO.turned(x.double(), theta, interleaved)
    # one rounding; cos and sin of a 32-bit fraction of a turn: 2 pi 2^-25 and two units each
    close(y, want, want.abs(), u, 16 * OO.F32 * float(size.max()))
    assert torch.equal(y[..., rotated:].cpu(), x[..., rotated:])
    back = ops.rotary_backward(ctx, dy.cuda(), *dev[1:], interleaved=interleaved, x=dev[0] if real else None)
    dx, dx_size = OO.turned(dy.double(), -theta, interleaved)
    close(back[0], dx, dx.abs(), u, 16 * OO.F32 * float(dx_size.max()))
    if real:
        r = rotated
        i = torch.arange(r // 2)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
        t = (dx[..., b] * x.double()[..., a] - dx[..., a] * x.double()[..., b]).sum(1) * freq.double()
        s = (dx_size[..., b] * x.double()[..., a].abs() + dx_size[..., a] * x.double()[..., b].abs()).sum(1) * freq.double()
        want, size = torch.zeros(rows, 4).double(), torch.zeros(rows, 4).double()
        want.index_add_(1, axis.long(), t)
        size.index_add_(1, axis.long(), s)
        assert back[1].dtype == kind
        close(back[1], want, size, (16 + heads + rotated) * OO.F32)
    inplace = dev[0].clone()
    assert ops.rotary(ctx, inplace, *dev[1:], interleaved=interleaved, out=inplace) is inplace
    assert torch.equal(inplace, y)


@dtypes
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_rotary_strided_rows(ctx, dtype, offset):
    """Queries and keys side by side in one projection, at any alignment."""
    g = torch.Generator().manual_seed(11)
    whole = rand(g, 6, 4 * 48 + 7, dtype=dtype).cuda()
    x = whole[:, offset:offset + 4 * 48].unflatten(1, (4, 48))
    pos = torch.randint(0, 500, (3, 6), generator=g, dtype=torch.int32).cuda().T  # axes apart
    freq, axis = torch.rand(24, generator=g).cuda(), (torch.arange(24) % 3).int().cuda()
    for inter in (False, True):
        got = ops.rotary(ctx, x, pos, freq, axis, interleaved=inter)
        assert torch.equal(got, ops.rotary(ctx, x.contiguous(), pos.contiguous(), freq, axis, interleaved=inter))


def test_rotary_keeps_the_phase_of_large_positions(ctx):
    pos = torch.tensor([[2 ** 40 + 12345], [-(2 ** 37) - 77]])
    freq = torch.tensor([1.0, 0.37], dtype=torch.float32)
    x = torch.tensor([[[1.0, 1.0, 0.0, 0.0]]] * 2)
    y = ops.rotary(ctx, x.cuda(), pos.cuda(), freq.cuda(), torch.zeros(2, dtype=torch.int32).cuda())
    want, _ = OO.turned(x.double(), pos.double() * freq.double(), False)
    # turns of 2^38: their fraction in 64 bits is good to 2^-14
    assert float((y.double().cpu() - want).abs().max()) < 2 * math.pi * 2 ** -13


# ---- attention --------------------------------------------------------------------


def attention_case(seed, dtype, q_len, k_len, heads, kv, dim, masked=0.0, empty_first=False):
    g = torch.Generator().manual_seed(seed)
    q_off, k_off = np.concatenate([[0], np.cumsum(q_len)]), np.concatenate([[0], np.cumsum(k_len)])
    c = dict(q=rand(g, q_off[-1], heads, 2, dim, dtype=dtype, scale=1.5),
             k=rand(g, k_off[-1], kv, 2, dim, dtype=dtype), v=rand(g, k_off[-1], kv, 2 * dim, dtype=dtype),
             lam=torch.rand(heads, generator=g) - 0.2, q_off=q_off, k_off=k_off, mask=None,
             dout=rand(g, q_off[-1], heads, 2 * dim, dtype=dtype))
    if masked:
        c["mask"] = torch.rand(int(k_off[-1]), generator=g) >= masked
        if empty_first:
            c["mask"][:k_off[1]] = False
        # what masked keys hold does not matter
        for t in ("k", "v"):
            c[t][~c["mask"]] = torch.tensor([math.nan, math.inf])[torch.randint(0, 2, (1,), generator=g)].to(dtype)
    return c


def check_attention(ctx, c, causal, scale=None):
    dtype, dim = c["q"].dtype, c["q"].shape[-1]
    dev = {n: c[n].cuda() for n in ("q", "k", "v", "lam", "dout")}
    mask = None if c["mask"] is None else c["mask"].cuda()
    seqs = ops.Sequences(ctx, c["q_off"], c["k_off"])
    kw = dict(causal=causal, key_mask=mask, scale=scale)
    args = [dev[n] for n in ("q", "k", "v", "lam")]
    out, saved = ops.diff_attention(ctx, *args, seqs, save=True, **kw)
    grads = ops.diff_attention_backward(ctx, dev["dout"], *args, seqs, out, saved, **kw)
    assert torch.equal(out, ops.diff_attention(ctx, *args, seqs, **kw))
    again = ops.diff_attention_backward(ctx, dev["dout"], *args, seqs, out, saved, **kw)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    r = OO.attention(*(c[n].double() for n in ("q", "k", "v", "lam")), dim ** -0.5 if scale is None else scale,
                     c["q_off"], c["k_off"], causal, c["mask"], c["dout"].double())
    u, longest = OO.UNIT[dtype], int(max(np.diff(c["k_off"]).max(initial=1), np.diff(c["q_off"]).max(initial=1)))
    f32 = OO.F32 * (16 + 4 * dim + longest + 4 * r["scores"])
    # probabilities below the smallest normal number of the type lose more: relative to a row's largest (1)
    tiny = 2.0 ** -25 * longest * 8 if dtype == torch.float16 else 0.0
    close(out, r["out"], r["|out|"], 1.25 * 2 * u + f32, tiny)
    lse = r["lse"]
    assert torch.equal(saved[1].cpu() == -math.inf, lse == -math.inf)
    live = lse > -math.inf
    # scores in 32 bits, and the hardware logarithm of a sum
    assert float((saved[1].double().cpu() - lse)[live].abs().max() if live.any() else 0.0) <= f32 + 1e-5
    group = c["q"].shape[1] // c["k"].shape[1]
    for got, name, n in zip(grads, ("dq", "dk", "dv"), (1, group, group)):
        close(got, r[name], r["|%s|" % name], 1.25 * 3 * u + n * f32, 4 * tiny * float(c["dout"].abs().max()) * n)
    # D is formed from 32-bit values; a rounding of P or out does not reach it
    close(grads[3], r["dlam"], r["|dlam|"], 4 * f32)


RAGGED = [([1], [1]), ([5, 0, 17, 1], [5, 0, 17, 1]), ([64, 65, 63], [64, 65, 63]), ([128, 130], [128, 130]),
          ([3, 40, 0, 9], [70, 1, 6, 0]), ([200], [33])]


@dtypes
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("q_len,k_len", RAGGED)
@pytest.mark.parametrize("heads,kv,dim", [(2, 2, 32), (4, 1, 64), (2, 1, 128)])
def test_attention(ctx, dtype, causal, q_len, k_len, heads, kv, dim):
    check_attention(ctx, attention_case(dim + len(q_len), dtype, q_len, k_len, heads, kv, dim), causal)


@dtypes
@pytest.mark.parametrize("dim", [1, 5, 8, 16, 24, 40, 72, 100, 127])
def test_attention_odd_dims(ctx, dtype, dim):
    check_attention(ctx, attention_case(dim, dtype, [37, 90], [37, 90], 3, 3, dim), dim % 2 == 1, scale=0.3)


@dtypes
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [20, 64, 128])
def test_attention_masks(ctx, dtype, causal, dim):
    """Masked keys hold NaN or infinity; the first sequence has no key at all."""
    c = attention_case(dim, dtype, [20, 150, 70], [20, 150, 70], 4, 2, dim, masked=0.3, empty_first=True)
    check_attention(ctx, c, causal)


@dtypes
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 32), (2, 2, 64), (2, 1, 128)])
def test_attention_single_keys(ctx, dtype, heads, kv, dim):
    """Sequences of one key: its probability is 1, so the scores have no
    gradient, exactly; values and lambda have theirs."""
    c = attention_case(dim, dtype, [1, 3, 1, 0, 2] * 9, [1, 1, 1, 1, 1] * 9, heads, kv, dim)
    for causal in (False, True):
        check_attention(ctx, c, causal)
        dev = [c[n].cuda() for n in ("q", "k", "v", "lam")]
        seqs = ops.Sequences(ctx, c["q_off"], c["k_off"])
        out, saved = ops.diff_attention(ctx, *dev, seqs, causal=causal, save=True)
        dq, dk, dv, _ = ops.diff_attention_backward(ctx, c["dout"].cuda(), *dev, seqs, out, saved, causal=causal)
        assert float(dq.abs().max()) == 0.0 and float(dk.abs().max()) == 0.0 and float(dv.abs().max()) > 0.0


@dtypes
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("q_len,k_len,heads,kv,dim", [([700], [90], 4, 1, 32), ([530, 0, 70], [530, 3, 70], 2, 2, 64),
                                                      ([257, 400], [300, 1], 6, 2, 128), ([600], [600], 3, 1, 5),
                                                      ([900], [40], 1, 1, 50)])
def test_attention_shared_key_pass(ctx, dtype, causal, q_len, k_len, heads, kv, dim):
    """Few keys and many rows: several workgroups share a tile of keys, some
    of which have no row that sees it."""
    check_attention(ctx, attention_case(dim, dtype, q_len, k_len, heads, kv, dim, masked=0.2), causal)


@dtypes
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_attention_few_keys(ctx, dtype, dim):
    """Sequences of two to four rows, where dS is a small difference: two
    roundings (of dS and of the result), each at most u and u / sqrt(3) in the
    mean over many elements, and nothing of the roundings of the saved results."""
    n = [2, 3, 4] * 30
    c = attention_case(dim + 1, dtype, n, n, 4, 4, dim)
    dev = [c[t].cuda() for t in ("q", "k", "v", "lam")]
    seqs = ops.Sequences(ctx, c["q_off"], c["k_off"])
    out, saved = ops.diff_attention(ctx, *dev, seqs, save=True)
    grads = ops.diff_attention_backward(ctx, c["dout"].cuda(), *dev, seqs, out, saved)
    r = OO.attention(*(c[t].double() for t in ("q", "k", "v", "lam")), dim ** -0.5, c["q_off"], c["k_off"], dout=c["dout"].double())
    for got, name in zip(grads, ("dq", "dk")):
        off = float((got.double().cpu() - r[name]).norm() / r[name].norm())
        assert off < math.sqrt(2 / 3) * OO.UNIT[dtype] * 1.1 + OO.F32 * (16 + 4 * dim + 4 * r["scores"])


@dtypes
def test_attention_large_scores(ctx, dtype):
    """Scores of several hundred: one key takes a row, exponentials of the others vanish."""
    c = attention_case(3, dtype, [100], [100], 2, 2, 32)
    c["q"] = c["q"] * 30
    check_attention(ctx, c, False)


def test_attention_gradient_against_differences(ctx):
    """The loss sum(out dout) along a direction in all inputs, from 64-bit
    differences of the formula, against the 32-bit kernels' gradients."""
    c = attention_case(8, torch.float32, [30, 7], [12, 50], 4, 2, 24)
    g = torch.Generator().manual_seed(9)
    names = ("q", "k", "v", "lam")
    d = {n: torch.randn(c[n].shape, generator=g).double() for n in names}
    h = 1e-5

    def loss(s):
        t = [c[n].double() + s * d[n] for n in names]
        return float((OO.attention(*t, 0.2, c["q_off"], c["k_off"])["out"] * c["dout"].double()).sum())

    seqs = ops.Sequences(ctx, c["q_off"], c["k_off"])
    leaf = [c[n].cuda().requires_grad_(True) for n in names]
    out = ops.DiffAttentionFn.apply(ctx, *leaf, seqs, False, 0.2, None)
    out.backward(c["dout"].cuda())
    got = sum(float((t.grad.double().cpu() * d[n]).sum()) for t, n in zip(leaf, names))
    size = sum(float((t.grad.double().cpu() * d[n]).abs().sum()) for t, n in zip(leaf, names))
    assert abs(got - (loss(h) - loss(-h)) / (2 * h)) < 1e-5 * size


@dtypes
@pytest.mark.parametrize("offset", [0, 1])
def test_attention_strides(ctx, dtype, offset):
    """Heads first, maps last, one projection for all three, and rows that
    start anywhere: the same bytes as from contiguous tensors."""
    g = torch.Generator().manual_seed(21)
    rows, h, d = 75, 3, 40
    whole = rand(g, rows, h * 6 * d + 5, dtype=dtype).cuda()[:, offset:offset + h * 6 * d]
    q = whole[:, :2 * h * d].unflatten(1, (2, h, d)).transpose(1, 2)  # maps outside heads
    k = whole[:, 2 * h * d:4 * h * d].unflatten(1, (h, 2, d))
    v = whole[:, 4 * h * d:].unflatten(1, (h, 2 * d))
    lam = torch.rand(h, generator=g).cuda()
    dout = rand(g, h, rows, 2 * d, dtype=dtype).cuda().transpose(0, 1)  # heads outside rows
    seqs = ops.Sequences(ctx, [0, 30, 75])
    got, want = [], []
    for to, t in ((got, (q, k, v)), (want, [x.contiguous() for x in (q, k, v)])):
        out, saved = ops.diff_attention(ctx, *t, lam, seqs, save=True)
        to += [out, *saved]
        do = dout if to is got else dout.contiguous()
        to += ops.diff_attention_backward(ctx, do, *t, lam, seqs, out, saved)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@dtypes
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 16), (8, 8, 32), (8, 1, 64), (34, 2, 128), (6, 2, 33)])
@pytest.mark.parametrize("lengths", [[1], [0, 31, 32, 33], [700, 2, 1000, 129]])
def test_cache(ctx, dtype, heads, kv, dim, lengths):
    """Cache rows beyond a length hold NaN; one length is beyond the capacity."""
    g = torch.Generator().manual_seed(dim + heads)
    n, cap = len(lengths), max(lengths) + 3
    q = rand(g, n, heads, 2, dim, dtype=dtype, scale=1.5)
    k, v = rand(g, n, cap, kv, 2, dim, dtype=dtype), rand(g, n, cap, kv, 2 * dim, dtype=dtype)
    lam = torch.rand(heads, generator=g)
    given, ends = torch.tensor(lengths, dtype=torch.int32), list(lengths)
    for i, m in enumerate(lengths):
        k[i, m:], v[i, m:] = math.nan, math.nan
    if n > 1:
        given[-1], ends[-1] = cap + 9, cap
        k[-1, lengths[-1]:], v[-1, lengths[-1]:] = 0.25, -0.5
    got = ops.diff_attention_cache(ctx, q.cuda(), k.cuda(), v.cuda(), lam.cuda(), given.cuda())
    u = OO.UNIT[dtype]
    for i, m in enumerate(ends):
        r = OO.attention(q[i:i + 1].double(), k[i, :m].double(), v[i, :m].double(), lam.double(), dim ** -0.5, [0, 1], [0, m])
        f32 = OO.F32 * (16 + 4 * dim + m + 4 * r["scores"])
        tiny = 2.0 ** -25 * m * 8 if dtype == torch.float16 else 0.0
        close(got[i:i + 1], r["out"], r["|out|"], 1.25 * 2 * u + f32, tiny)


def test_cache_offsets_beyond_32_bits(ctx):
    """Two caches 2^31 + 2^20 elements apart in one allocation."""
    g = torch.Generator().manual_seed(1)
    apart, cap, d = 2 ** 31 + 2 ** 20, 300, 32
    store = torch.empty(apart + cap * 2 * d, dtype=torch.bfloat16, device="cuda")
    k = store.as_strided((2, cap, 1, 2, d), (apart, 2 * d, 2 * d, d, 1))
    k.copy_(rand(g, 2, cap, 1, 2, d, dtype=torch.bfloat16))
    v = k.as_strided((2, cap, 1, 2 * d), (apart, 2 * d, 2 * d, 1))
    q, lam = rand(g, 2, 4, 2, d, dtype=torch.bfloat16).cuda(), torch.rand(4, generator=g).cuda()
    lengths = torch.tensor([cap, cap - 7], dtype=torch.int32).cuda()
    got = ops.diff_attention_cache(ctx, q, k, v, lam, lengths)
    near = ops.diff_attention_cache(ctx, q, k.contiguous(), v.contiguous(), lam, lengths)
    assert torch.equal(got, near)
    # the same rows as one ragged batch whose rows are far apart
    seqs = ops.Sequences(ctx, [0, 2], [0, 2])
    far = store.as_strided((2, 1, 2, d), (apart, 2 * d, d, 1))
    out = ops.diff_attention(ctx, q, far, far.flatten(2), lam, seqs)
    assert torch.equal(out, ops.diff_attention(ctx, q, far.contiguous(), far.flatten(2).contiguous(), lam, seqs))


# ---- norms ---------------------------------------------------------------------------


@dtypes
@pytest.mark.parametrize("kind,act", [("rms", "none"), ("layer", "sigmoid"), ("rms", "tanh")])
@pytest.mark.parametrize("rows,width,gated", [(1, 1, 2), (3, 7, 1), (70, 64, 2), (33, 512, 1), (9, 1000, 2),
                                              (5, 1025, 1), (4, 4096, 0), (2, 5001, 2), (1, 16384, 1)])
def test_norm_block(ctx, dtype, kind, act, rows, width, gated):
    """gated: 0 no gate and no residual, 1 a gate for all rows, 2 one per row."""
    g = torch.Generator().manual_seed(width)
    x = rand(g, rows, width, dtype=dtype, scale=2.0) if gated else None
    y = rand(g, rows, width, dtype=dtype) + 0.25
    gate = [None, rand(g, width, dtype=dtype), rand(g, rows, width, dtype=dtype)][gated]
    w1 = 1 + rand(g, width, dtype=dtype, scale=0.1) if width != 4096 else None
    w2 = 1 + rand(g, width, dtype=dtype, scale=0.1)
    ds, dn = rand(g, rows, width, dtype=dtype), rand(g, rows, width, dtype=dtype)
    kw = dict(kind=kind, gate_act=act, residual_scale=0.8, block_scale=-0.6, eps=1e-2)
    # eps of 1e-2: a row of one element (or the layer norm of it, zero) stays well conditioned
    cpu = [x, y, gate, w1, w2]
    dev = [None if t is None else t.cuda() for t in cpu]
    s, n, stats = ops.norm_block(ctx, *dev, save=True, **kw)
    got = ops.norm_block_backward(ctx, ds.cuda(), dn.cuda(), *dev, stats, **kw)
    leaf = [None if t is None else t.double().requires_grad_(True) for t in cpu]
    s64, n64 = OO.norm_block(*leaf, kind, act, 0.8, -0.6, 1e-2)
    u, f32 = OO.UNIT[dtype], OO.F32 * (64 + math.sqrt(width))
    big = 1 + float(max(t.detach().abs().max() for t in (s64, n64)))
    close(s, s64.detach(), s64.detach().abs(), u, f32 * big)
    close(n, n64.detach(), n64.detach().abs(), u, 16 * f32 * big)
    (s64 * ds.double()).sum().add((n64 * dn.double()).sum()).backward()
    # a row's gradient is at most 1 / sqrt(eps) times what comes in, through each norm
    for a, b in zip(got, leaf):
        if b is None:
            assert a is None
            continue
        total = float(b.grad.abs().max()) + 10 * float(dn.abs().max() + ds.abs().max()) * big
        close(a, b.grad, b.grad.abs(), u, f32 * total * (math.sqrt(rows) if a.dim() == 1 else 1) * 16)
    only_s, none = ops.norm_block(ctx, *dev, next_norm=False, **kw)
    assert none is None and torch.equal(only_s, s)


@dtypes
@pytest.mark.parametrize("kind,act", [("rms", "sigmoid"), ("layer", "tanh")])
@pytest.mark.parametrize("rows,width,gated", [(1100, 1024 + 8, 1), (3, 1536, 2), (3, 1537, 1), (600, 2353, 2),
                                              (300, 4104, 1), (2, 6144, 0), (270, 6145, 2), (2, 8193, 1)])
def test_norm_block_thread_counts(ctx, dtype, kind, act, rows, width, gated):
    """Rows held by numbers of threads that are not powers of two, and the
    widths beside them; several rows a workgroup."""
    test_norm_block(ctx, dtype, kind, act, rows, width, gated)


def test_norm_block_autograd_without_a_gradient_of_n(ctx):
    g = torch.Generator().manual_seed(2)
    x, y, gate, w1, w2 = (rand(g, *shape, dtype=torch.float32).cuda().requires_grad_(True)
                          for shape in ((6, 24), (6, 24), (24,), (24,), (24,)))
    opts = dict(kind="layer", gate_act="tanh", eps=1e-3)
    s, n = ops.NormBlockFn.apply(ctx, x, y, gate, w1, w2, opts)
    s.sum().backward()
    leaf = [t.detach().double().requires_grad_(True) for t in (x, y, gate, w1)]
    s64, _ = OO.norm_block(*leaf, None, "layer", "tanh", 1.0, 1.0, 1e-3)
    s64.sum().backward()
    for a, b in zip((x, y, gate, w1), leaf):
        assert float((a.grad.double() - b.grad).abs().max()) < 64 * OO.F32 * 24 * float(b.grad.abs().max() + 1)
    assert float(w2.grad.abs().max()) == 0.0


@dtypes
def test_norm_block_strided_rows(ctx, dtype):
    g = torch.Generator().manual_seed(4)
    whole = rand(g, 20, 333, dtype=dtype).cuda()
    for a, w in ((0, 96), (1, 97), (5, 64)):
        x, y, gate = whole[:, a:a + w], whole[:, 100 + a:100 + a + w], whole[:, 200 + a:200 + a + w]
        w1 = whole[0, 40:40 + w]
        one = ops.norm_block(ctx, x, y, gate, w1, None, kind="layer")
        two = ops.norm_block(ctx, x.contiguous(), y.contiguous(), gate.contiguous(), w1.clone(), None, kind="layer")
        for p, q in zip(one, two):
            assert float((p.float() - q.float()).abs().max()) <= 4 * OO.UNIT[dtype] * float(q.abs().max())


# ---- no rows, streams, graphs, refusals --------------------------------------------------


def test_no_rows(ctx):
    dev = torch.device("cuda")
    e = torch.empty
    freq, axis = torch.ones(2, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    assert ops.rotary(ctx, e(0, 2, 4, device=dev), e(0, 1, device=dev), freq, axis).shape == (0, 2, 4)
    q, v, lam = e(0, 2, 2, 8, device=dev), e(0, 2, 16, device=dev), torch.ones(2, device=dev)
    for off in ([0], [0, 0, 0]):
        seqs = ops.Sequences(ctx, off)
        out, saved = ops.diff_attention(ctx, q, q, v, lam, seqs, save=True)
        grads = ops.diff_attention_backward(ctx, out, q, q, v, lam, seqs, out, saved)
        assert float(grads[3].abs().max()) == 0.0
    # keys without rows: their gradients are zero
    seqs, k, kv = ops.Sequences(ctx, [0, 0], [0, 3]), torch.ones(3, 2, 2, 8, device=dev), torch.ones(3, 2, 16, device=dev)
    out, saved = ops.diff_attention(ctx, q, k, kv, lam, seqs, save=True)
    _, dk, dv, _ = ops.diff_attention_backward(ctx, out, q, k, kv, lam, seqs, out, saved)
    assert float(dk.abs().max()) == 0.0 and float(dv.abs().max()) == 0.0
    none = ops.diff_attention_cache(ctx, torch.ones(2, 2, 2, 8, device=dev), e(2, 0, 2, 2, 8, device=dev),
                                    e(2, 0, 2, 16, device=dev), lam, torch.zeros(2, dtype=torch.int32, device=dev))
    assert float(none.abs().max()) == 0.0
    w = torch.ones(8, device=dev)
    s, n, stats = ops.norm_block(ctx, e(0, 8, device=dev), e(0, 8, device=dev), w, w, w, save=True)
    grads = ops.norm_block_backward(ctx, s, n, s, n, w, w, w, stats)
    assert all(float(t.abs().max()) == 0.0 for t in grads[2:])


def _block(ctx, seqs, t):
    """Rotation, attention and residual glue of one block, as a program joins them."""
    qk = ops.rotary(ctx, t["qk"], t["pos"], t["freq"], t["axis"])
    q, k = qk[:, :8].unflatten(1, (4, 2)), qk[:, 8:].unflatten(1, (2, 2))
    out = ops.diff_attention(ctx, q, k, t["v"], t["lam"], seqs)
    cache = ops.diff_attention_cache(ctx, q[:2], k[None].expand(2, -1, -1, -1, -1), t["v"][None].expand(2, -1, -1, -1),
                                     t["lam"], t["lengths"])
    s, n = ops.norm_block(ctx, t["x"], out.flatten(1), t["gate"], t["w"], t["w"])
    return s, n, cache


def _block_inputs(seed):
    g = torch.Generator().manual_seed(seed)
    t = dict(qk=rand(g, 50, 12, 32, dtype=torch.bfloat16), v=rand(g, 50, 2, 64, dtype=torch.bfloat16),
             x=rand(g, 50, 256, dtype=torch.bfloat16), gate=rand(g, 256, dtype=torch.bfloat16),
             w=rand(g, 256, dtype=torch.bfloat16), lam=torch.rand(4, generator=g), pos=torch.rand(50, 3, generator=g),
             freq=torch.rand(16, generator=g), axis=(torch.arange(16) % 3).int(),
             lengths=torch.tensor([50, 17], dtype=torch.int32))
    return {k: v.cuda() for k, v in t.items()}


def test_on_another_stream_and_in_a_graph(ctx):
    seqs = ops.Sequences(ctx, [0, 20, 50])
    inputs = [_block_inputs(s) for s in (1, 2, 3)]
    want = [[r.clone() for r in _block(ctx, seqs, t)] for t in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _block(ctx, seqs, inputs[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    held = {k: v.clone() for k, v in inputs[0].items()}
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _block(ctx, seqs, held)
    for i in (1, 2, 0, 1):
        for k, v in inputs[i].items():
            held[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
        eager = _block(ctx, seqs, inputs[(i + 1) % 3])
        assert all(torch.equal(a, b) for a, b in zip(eager, want[(i + 1) % 3]))


def refused(code, f, *a, **k):
    with pytest.raises(capi.MtpxError) as e:
        f(*a, **k)
    assert e.value.code == capi.ERRORS_BY_NAME[code], e.value


def test_refusals(ctx):
    dev, bad = torch.device("cuda"), "MTPX_E_INVALID"
    z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device=dev)  # noqa: E731
    f, ax, i32 = z(2), z(2, dtype=torch.int32), torch.int32
    refused(bad, ops.rotary, ctx, z(3, 1, 3), z(3, 1), f, ax)                    # 4 rotated of 3
    refused(bad, ops.rotary, ctx, z(3, 1, 4, dtype=torch.float64), z(3, 1), f, ax)
    refused(bad, ops.rotary, ctx, z(3, 1, 4), z(2, 1), f, ax)
    refused(bad, ops.rotary, ctx, z(3, 1, 4), z(3, 9), f, ax)                    # nine axes
    refused(bad, ops.rotary, ctx, z(3, 1, 8)[..., ::2], z(3, 1), f, ax)          # last dimension strided
    refused(bad, ops.rotary_backward, ctx, z(3, 1, 4), z(3, 1, dtype=i32), f, ax, x=z(3, 1, 4))
    refused("MTPX_E_CAPACITY", ops.rotary, ctx, z(1, 1, 1026), z(1, 1), f, ax)
    for off in ([1, 2], [0, 5, 3], []):
        refused(bad, ops.Sequences, ctx, off)
    refused(bad, ops.Sequences, ctx, [0, 4], [0, 2, 4])
    refused("MTPX_E_CAPACITY", ops.Sequences, ctx, [0, 2 ** 31])
    seqs = ops.Sequences(ctx, [0, 4])
    q, v, lam = z(4, 2, 2, 8), z(4, 2, 16), z(2)
    refused(bad, ops.diff_attention, ctx, q, q, v, lam, ops.Sequences(ctx, [0, 5]))
    refused(bad, ops.diff_attention, ctx, q, q, v, z(3), seqs)
    refused(bad, ops.diff_attention, ctx, q, q, z(4, 2, 15), lam, seqs)
    refused(bad, ops.diff_attention, ctx, q, q, v.half(), lam, seqs)
    refused(bad, ops.diff_attention, ctx, z(4, 3, 2, 8), q, v, z(3), seqs)       # 3 heads over 2
    refused(bad, ops.diff_attention, ctx, q, q, v, lam, seqs, scale=0.0)
    refused(bad, ops.diff_attention, ctx, q, q, v, lam, seqs, scale=math.nan)
    refused(bad, ops.diff_attention, ctx, q, q, v, lam, seqs, key_mask=z(4))
    refused("MTPX_E_CAPACITY", ops.diff_attention, ctx, z(4, 2, 2, 129), z(4, 2, 2, 129), z(4, 2, 258), lam, seqs)
    closed = ops.Sequences(ctx, [0, 4])
    closed.close()
    refused(bad, ops.diff_attention, ctx, q, q, v, lam, closed)
    refused(bad, ops.diff_attention_cache, ctx, z(1, 2, 2, 8), z(1, 5, 2, 2, 8), z(1, 5, 2, 16), lam, z(1))
    refused(bad, ops.norm_block, ctx, z(2, 8), z(3, 8))
    refused(bad, ops.norm_block, ctx, None, z(3, 8), kind="group")
    refused(bad, ops.norm_block, ctx, None, z(3, 8), eps=-1.0)
    refused(bad, ops.norm_block, ctx, None, z(3, 8), None, z(9))
    refused("MTPX_E_CAPACITY", ops.norm_block, ctx, None, z(1, 16385))
    # through the C entry: a workspace that is too small, an unknown type, an unaligned tensor
    L = ops._ops()
    out, saved = ops.diff_attention(ctx, q, q, v, lam, seqs, save=True)
    req = ops._attention(ctx, q, q, v, lam, seqs, False, None, None)
    wide = lambda t: ops.Rows(t.data_ptr(), t.stride(0), t.stride(1), 8)  # noqa: E731
    maps = lambda t: ops.Rows(t.data_ptr(), *t.stride()[:3])  # noqa: E731
    req.out, req.dout = wide(out), wide(out)
    req.out1, req.lse, req.dlambda = saved[0].data_ptr(), saved[1].data_ptr(), lam.data_ptr()
    req.dq, req.dk, req.dv = maps(q), maps(q), wide(v)
    req.workspace, req.workspace_bytes = out.data_ptr(), 8
    assert L.mtpx_diff_attention_backward(ctx.h, req) == -1
    req.workspace = None
    assert L.mtpx_diff_attention_backward(ctx.h, req) == -1
    req.dtype = 3
    assert L.mtpx_diff_attention(ctx.h, req) == -1
    req.dtype, req.q.data = 0, q.data_ptr() + 2
    assert L.mtpx_diff_attention(ctx.h, req) == -1
    req.q.data, req.q.row = q.data_ptr(), -1
    assert L.mtpx_diff_attention(ctx.h, req) == -1
