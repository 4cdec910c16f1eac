"""The norms around a block in 64 bits, written out, with the size of what each
element adds up: the error of 32-bit arithmetic is at most ROUNDINGS 2^-24
times that size, and a result takes one rounding to its type on top.

ROUNDINGS.  A sum over a row adds, for each term, at most 16 numbers of a
thread, 6 steps within a wave and 16 waves: 38 roundings relative to the sum of
absolute terms.  The longest way from an input to a result passes four such
sums (the two statistics, the two means of the backward pass), 152, and fewer
than 40 products, divisions, roots and differences.  A weight's gradient adds
the rows of a group, of a workgroup and the workgroups' parts on top
(COLUMN)."""
import torch

F32 = 2.0 ** -24
ROUNDINGS = 192
COLUMN = 160  # rows a group (under 16), groups (16), parts of a run (96), runs (16)

NAMES = ("s", "n", "dx", "dy", "dgate", "dw1", "dw2")


def _act(kind, g):
    """Activation, its slope, and the slope's size: 1 - a and 1 - a^2 cancel."""
    if kind == "sigmoid":
        a = torch.sigmoid(g)
        return a, a * (1 - a), a
    if kind == "tanh":
        a = torch.tanh(g)
        return a, 1 - a * a, torch.ones_like(a)
    return g, torch.ones_like(g), torch.ones_like(g)


def norm_block(x, y, gate, w1, w2, ds, dn, kind, act, alpha, beta, eps, mutate=""):
    """({name: value}, {name: size}) in float64; None inputs as in the call.
    mutate names a mistake to make: mean1 or mean2 (the mean of that norm's
    backward pass left out), slope (1% off), half (dn w2 rounded to bfloat16)."""
    layer = kind == "layer"
    x, y, gate, w1, w2, ds, dn = (None if t is None else t.double() for t in (x, y, gate, w1, w2, ds, dn))
    one = torch.ones(y.shape[1]).double()
    a, slope, slope_size = (one, one, one) if gate is None else _act(act, gate)
    p1, p2 = one if w1 is None else w1, one if w2 is None else w2

    def mean(t):
        return t.mean(1, keepdim=True)

    def normed(t, size):
        mu = mean(t) if layer else torch.zeros(len(t), 1).double()
        r = 1 / torch.sqrt(mean((t - mu) ** 2) + eps)
        v = (t - mu) * r
        return v, r, (size + (mean(size) if layer else 0.0)) * r + v.abs()

    u, r1, u_size = normed(y, y.abs())
    z, z_size = u * p1, u_size * p1.abs()
    s, s_size = beta * a * z, abs(beta) * a.abs() * z_size
    if x is not None:
        s, s_size = s + alpha * x, s_size + abs(alpha) * x.abs()
    v, r2, v_size = normed(s, s_size)
    val, size = dict(s=s, n=v * p2), dict(s=s_size, n=v_size * p2.abs())

    dv = dn * p2
    if mutate == "half":
        dv = dv.bfloat16().double()
    m1, m1_size = mean(dv * v), mean(dv.abs() * v_size)
    back = dv - v * m1 - (mean(dv) if layer and mutate != "mean2" else 0.0)
    t = ds + r2 * back
    t_size = ds.abs() + r2 * (dv.abs() + (mean(dv.abs()) if layer else 0.0) + v.abs() * m1_size + m1.abs() * v_size)
    val["dw2"], size["dw2"] = (dn * v).sum(0), (dn.abs() * v_size).sum(0)
    if x is not None:
        val["dx"], size["dx"] = alpha * t, abs(alpha) * t_size
    if gate is not None:
        off = 1.01 if mutate == "slope" else 1.0
        val["dgate"] = beta * slope * off * z * t
        size["dgate"] = abs(beta) * (slope_size * (z * t).abs() + slope.abs() * (z_size * t.abs() + z.abs() * t_size))
        if gate.dim() == 1:
            val["dgate"], size["dgate"] = val["dgate"].sum(0), size["dgate"].sum(0)
    dz, dz_size = beta * a * t, abs(beta) * a.abs() * t_size
    val["dw1"], size["dw1"] = (dz * u).sum(0), (dz_size * u.abs() + dz.abs() * u_size).sum(0)
    du, du_size = dz * p1, dz_size * p1.abs()
    q1, q1_size = mean(du * u), mean(du_size * u.abs() + du.abs() * u_size)
    val["dy"] = r1 * (du - u * q1 - (mean(du) if layer and mutate != "mean1" else 0.0))
    size["dy"] = r1 * (du_size + (mean(du_size) if layer else 0.0) + u.abs() * q1_size + q1.abs() * u_size)
    if w1 is None:
        del val["dw1"]
    if w2 is None:
        del val["dw2"]
    return val, size


def passed(got, want, size, name, unit):
    """The largest error in units of its bound (1 is the limit)."""
    many = ROUNDINGS + (COLUMN if got.dim() == 1 else 0)
    # (subnormal results round to multiples of 2^-24 in float16)
    bound = unit * want.abs() + many * F32 * size + 2.0 ** -25 * (unit == 2.0 ** -11)
    return float(((got.double() - want).abs() / bound.clamp_min(1e-300)).max()) if got.numel() else 0.0
