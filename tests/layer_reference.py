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
