"""The operators of an encoder's layer from their formulas in 64 bits, with how
far a result may be before its last rounding (train_reference.assert_near adds
that).

Bounds.  A float32 sum of which no term takes part in more than h additions is
off by at most h U32 times the sum of the magnitudes.  Group norm's kernels add at
most 64 terms in a lane, `positions` in a thread of the largest groups, 128 rows
out of LDS a lane, a few levels of lanes and waves, and up to 1,100 runs: h = 1400 +
positions covers all of them."""
import numpy as np
import torch

import train_reference as ref
from train_reference import FUN, U32


def threshold(p):
    return min(65535, int(np.floor(p * 65536 + 0.5)))


def random_halves(count, seed, offset):
    """The 16 bits of elements 0 .. count - 1: Philox 4x32 with seven rounds."""
    mask = np.uint64(0xFFFFFFFF)
    i = np.arange(-(-count // 8), dtype=np.uint64)
    c = [i & mask, i >> np.uint64(32), np.full_like(i, offset & 0xFFFFFFFF), np.full_like(i, offset >> 32)]
    k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(7):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & mask,
             (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & mask]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    words = np.stack(c, 1)
    return np.stack([words & np.uint64(0xFFFF), words >> np.uint64(16)], 2).reshape(-1)[:count]


def factor(shape, p, seed, offset):
    """What each element is multiplied by."""
    t = threshold(p)
    keep = random_halves(int(np.prod(shape)), seed, offset) >= t
    return torch.from_numpy(keep.reshape(shape)).double() * (65536.0 / (65536 - t))


def _over(v, positions_channels):
    """Means over positions and the group's channels of (n, positions, g, d)."""
    return v.sum((1, 3), keepdim=True) / positions_channels


def group_norm(x, groups, w, b, eps, act, by=None, dy=None):
    """A dict of (value, bound): y, mean, rstd and, with dy, dx, dw, db; `by` is
    dropout's factor."""
    shape = x.shape
    n, c = shape[0], shape[-1]
    d = c // groups
    v = x.double().reshape(n, -1, groups, d)
    s = v.shape[1]
    count = s * d
    h = 1400 + s
    one = torch.ones(groups, d, dtype=torch.float64)
    w4 = one if w is None else w.double().view(groups, d)
    b4 = 0 * one if b is None else b.double().view(groups, d)
    by = torch.ones_like(v) if by is None else by.reshape(v.shape)
    mean = _over(v, count)
    far = v - mean
    var = _over(far * far, count)
    rstd = 1 / torch.sqrt(var + eps)
    off_mean = h * U32 * _over(v.abs(), count)
    # squares about the mean, or of differences from some element of the group
    spread = var + far.abs().amax((1, 3), keepdim=True) ** 2
    off_var = 2 * (h + 4) * U32 * spread + off_mean ** 2
    rel = 0.5 * off_var / (var + eps) + 4 * U32
    xh = far * rstd
    off_xh = rstd * (off_mean + U32 * far.abs()) + xh.abs() * rel
    z = xh * w4 + b4
    off_z = w4.abs() * off_xh + 2 * U32 * ((xh * w4).abs() + b4.abs())
    y, slope = ref.act(z, act)
    smooth = act not in ("none", "relu")
    off_y = 1.2 * off_z + (FUN * z.abs() if smooth else 0)
    out = dict(y=((y * by).reshape(shape), ((off_y + U32 * y.abs()) * by).reshape(shape)),
               mean=(mean.view(n, groups), off_mean.view(n, groups)),
               rstd=(rstd.view(n, groups), (rstd * rel).view(n, groups)))
    if dy is None:
        return out
    g = dy.double().reshape(v.shape) * by
    dz = g * slope
    if act == "relu":  # a slope of 0 or 1 where z's sign may be either
        off_dz = torch.where(z.abs() <= off_z, g.abs(), 0 * g)
    else:
        off_dz = g.abs() * ((off_z + FUN * (1 + z * z)) if smooth else 0 * z)
    off_dz = off_dz + 2 * U32 * dz.abs()
    t, off_t = dz * w4, w4.abs() * off_dz + U32 * (dz * w4).abs()
    tx, off_tx = t * xh, off_t * xh.abs() + t.abs() * off_xh
    m1, m2 = _over(t, count), _over(tx, count)
    off_1 = _over(off_t, count) + h * U32 * _over(t.abs(), count)
    off_2 = _over(off_tx, count) + h * U32 * _over(tx.abs(), count)
    dx = rstd * (t - m1 - xh * m2)
    off = rstd * (off_t + off_1 + xh.abs() * off_2 + m2.abs() * off_xh
                  + 4 * U32 * (t.abs() + m1.abs() + (xh * m2).abs())) + rel * dx.abs()
    out["dx"] = (dx.reshape(shape), off.reshape(shape))
    rows = h + n
    out["db"] = (dz.sum((0, 1)).view(c), (off_dz.sum((0, 1)) + rows * U32 * dz.abs().sum((0, 1))).view(c))
    dwx, off_w = dz * xh, off_dz * xh.abs() + dz.abs() * off_xh
    out["dw"] = (dwx.sum((0, 1)).view(c), (off_w.sum((0, 1)) + rows * U32 * dwx.abs().sum((0, 1))).view(c))
    return out


# ---- 8-bit floating point ----

def _power(e):
    return torch.ldexp(torch.ones(e.shape, dtype=torch.float64), e.to(torch.int32))


def e4m3(q):
    """q rounded to three bits of fraction, from 2^-6 down to multiples of 2^-9, half
    to even; what is not finite is NaN."""
    q = torch.where(q.isfinite(), q, torch.full_like(q, float("nan")))
    _, e = torch.frexp(torch.nan_to_num(q))
    step = _power((e - 1).clamp(min=-6) - 3)
    return torch.round(q / step) * step


def scale_exponents(top):
    """The least e with top <= 448 * 2^e, 0 for nothing, -127 at least."""
    f, e = torch.frexp(top / 448)
    return torch.where(top > 0, torch.where(f == 0.5, e - 1, e).clamp(min=-127), torch.zeros_like(e))


def fp8_blocks(v, rows=1):
    """(values, codes' values, exponents of every block): v (float64) in 8 bits, a
    scale for `rows` x 128."""
    n, k = v.shape
    room = torch.zeros(-(-n // rows) * rows, -(-k // 128) * 128, dtype=torch.float64)
    room[:n, :k] = v
    b = room.view(-1, rows, room.shape[1] // 128, 128)
    finite = torch.where(b.isfinite(), b.abs(), torch.zeros_like(b))
    e = scale_exponents(finite.amax((1, 3)))
    up = _power(e)[:, None, :, None]
    q = e4m3(b / up)
    return (q * up).reshape(room.shape)[:n, :k], q.reshape(room.shape)[:n], e


def fp8_near(v, off):
    """What 8 bits hold of rows v whose elements are known to `off`: (values, bound)."""
    val, _, _ = fp8_blocks(v)
    n, k = v.shape
    pad = -(-k // 128) * 128

    def top(t):
        room = torch.zeros(n, pad, dtype=torch.float64)
        room[:, :k] = t
        return scale_exponents(room.view(n, -1, 128).amax(2)).repeat_interleave(128, 1)[:, :k]

    e = top(v.abs())
    up = _power(e)
    bound = (e4m3((v + off) / up) - e4m3((v - off) / up)).abs() * up
    # a largest magnitude at the border of two scales: either may be taken
    either = (top(v.abs() + off) != e) | (top((v.abs() - off).clamp(min=0)) != e)
    return val, torch.where(either, bound + v.abs() / 4 + up * 2.0 ** -7, bound)


def cut_off(a, b, dtype):
    """What the 8-bit matrix instruction leaves out of a b^T (rows with k
    contiguous).  It adds eight adjacent products after cutting each, towards zero, to
    a multiple of 2^-13 of the largest one's power of two: less than that for each of
    seven, and the largest is at most the product of the largest factors.  (Measured
    with one product of 2^16 beside another of m 2^j, m = 1, 1.25, 1.5, 1.75, either
    sign: 2^3 is the smallest step of what is added, and a place further than eight
    away keeps all of f32's.)  f32 calls use other instructions."""
    if dtype == torch.float32:
        return 0.0

    def tops(v):
        room = torch.zeros(v.shape[0], -(-v.shape[1] // 8) * 8, dtype=torch.float64)
        room[:, :v.shape[1]] = v.abs().nan_to_num()
        return room.view(v.shape[0], -1, 8).amax(2)

    return 7 * 2.0 ** -13 * (tops(a) @ tops(b).t())


def linear_fp8(x, w, bias, act, residual):
    """((y, bound), (z, bound)), from what 8 bits hold of x and w."""
    xq, wq = fp8_blocks(x.double())[0], fp8_blocks(w.double(), 128)[0]
    (y, off_y), (z, off_z) = ref.linear(xq, wq, bias, act, residual)
    cut = cut_off(xq, wq, x.dtype)
    return (y, off_y + 1.2 * cut), (z, off_z + cut)  # |slope| <= 1.13


def linear_fp8_grad(dy, x, w, z, act):
    """((dx, bound), (dw, bound), (db, bound))."""
    dtype = x.dtype
    dy, x, w = dy.double(), x.double(), fp8_blocks(w.double(), 128)[0]
    n, m = dy.shape
    if act == "none":
        dz, off = dy, torch.zeros_like(dy)
    else:
        dz = dy * ref.act(z.double(), act)[1]
        off = 2 * U32 * dz.abs() if act == "relu" else FUN * dy.abs() * (1 + z.double() ** 2)
    q, made = fp8_near(dz, off)
    dx = q @ w
    off_x = made @ w.abs() + ref.dot_bound(m) * (q.abs() @ w.abs()) + cut_off(q, w.t(), dtype)
    q, made = fp8_near(dz.t().contiguous(), off.t().contiguous())
    xt = fp8_blocks(x.t().contiguous())[0]
    dw = q @ xt.t()
    off_w = made @ xt.abs().t() + ref.dot_bound(n) * (q.abs() @ xt.abs().t()) + cut_off(q, xt, dtype)
    db = dz.sum(0)
    return (dx, off_x), (dw, off_w), (db, off.sum(0) + ref.dot_bound(n) * dz.abs().sum(0))
