"""Group norm and its gradient in 64 bits, with bounds that follow the kernels' sums.

A float32 sum of which no term takes part in more than h additions is off by at most
h U32 times the sum of the magnitudes.  What a term takes part in:

rows (one position): 16 terms of a lane, 6 levels of lanes, 8 waves: h = 30.
slabs: P positions of a thread (12 at most of a slab that is kept; 6 of a run, up to 12
  where runs are fewer than workgroups), 16 rows of LDS a slice, then a group's channels
  and slices, 32 of one thread or one in 64 of a lane, and 6 levels of lanes: h = 12 + 16
  + max(32, d / 64) + 6.  Groups split into runs: 24 of those a lane and 6 levels more
  (1024 runs at most, of which a group takes 64 lanes, or of more groups as many as 256
  threads have for each; `runs` below checks that a shape is within it).
The parameters' sums: as far as a thread's or slice's, then samples one after another
  (10 at most of the shapes here), 64 slices, and the parts of 32 lanes and their join.
  Rows: those samples and the parts alone.

The squares of a split group's threads are of differences from the thread's first
element of a channel: their sum is at most 2 + 2 P times that about the mean, whichever
elements those are, and only the thread's own P + 5 roundings go by it."""
import torch

import train_reference as ref
from train_reference import FUN, U32

POSITIONS = 12


def split(shape, groups, dtype):
    """Whether a sample's groups may be split into runs: whether a thread would hold
    more than two of its positions (a slab of groups is half a line of memory at
    least and 512 threads hold it)."""
    if len(shape) == 2:
        return False
    d = shape[-1] // groups
    wide = max(1, -(-64 // (4 if dtype == torch.float32 else 2) // d)) * d
    s = 1
    for k in shape[1:-1]:
        s *= k
    return s > 2 * (512 // max(1, -(-wide // 8)))


def inputs(seed, shape, groups, dtype, mean=0.5, std=1.0):
    """x, w, b and a dy whose means with 1 and xh over a group are of order one."""
    g = torch.Generator().manual_seed(seed)

    def normal(*k):
        return torch.randn(*k, generator=g, dtype=torch.float64)

    c = shape[-1]
    x = normal(*shape)
    dy = 0.5 * normal(*shape) + 0.8 + 0.7 * x
    return ((x * std + mean).to(dtype), (1 + 0.3 * normal(c)).to(dtype), (0.3 * normal(c)).to(dtype), dy.to(dtype))


def group_norm(x, groups, w, b, eps, act, by, dy, is_split, change=None):
    """A dict of (value, bound): y, mean, rstd, dx, dw, db; `by` is dropout's factor.
    `change` leaves something out of the values, for the test of the bounds."""
    shape = x.shape
    n, c = shape[0], shape[-1]
    d = c // groups
    v = x.double().reshape(n, -1, groups, d)
    s = v.shape[1]
    count = s * d
    rows = s == 1
    h = 30 if rows else POSITIONS + 16 + max(32, -(-d // 64)) + 6 + (30 if is_split else 0)
    h_param = (10 if rows else POSITIONS + 16 + 10 + 64 + 33) + n // 32 + 1 + 32
    one = torch.ones(groups, d, dtype=torch.float64)
    w4, b4 = (w.double().view(groups, d), b.double().view(groups, d)) if w is not None else (one, 0 * one)
    by = torch.ones_like(v) if by is None else by.reshape(v.shape)

    def over(t):
        return t.sum((1, 3), keepdim=True) / count

    mean = over(v)
    far = v - mean
    var = over(far * far)
    size = over(v.abs())
    if is_split:
        off_mean = (h + (POSITIONS + 3) * (1 + POSITIONS)) * U32 * size + 2 * U32 * mean.abs()
        off_var = ((POSITIONS + 5) * (2 + 2 * POSITIONS) + h + 8) * U32 * var
        # the channels' and the runs' means are rounded before their squares are taken
        spread = 3 * U32 * (far.abs() + mean.abs()).amax((1, 3), keepdim=True) + off_mean
        off_var = off_var + 2 * spread * var.sqrt() + spread ** 2
    else:
        off_mean = (h + 2) * U32 * size + 2 * U32 * mean.abs()
        off_var = (h + 6) * U32 * var + off_mean ** 2
    rel = 0.5 * off_var / (var + eps) + 4 * U32
    rstd = 1 / torch.sqrt(var + eps)
    if change == "rstd":
        rstd = rstd * 1.01
    xh = far * rstd
    off_xh = rstd * (off_mean + U32 * far.abs()) + xh.abs() * (rel + U32)
    z = xh * w4 + b4
    off_z = w4.abs() * off_xh + 2 * U32 * ((xh * w4).abs() + b4.abs())
    y, slope = ref.act(z, act)
    smooth = act not in ("none", "relu")
    off_y = 1.2 * off_z + (FUN * z.abs() if smooth else 0)
    out = dict(y=((y * by).reshape(shape), ((off_y + 3 * U32 * y.abs()) * by).reshape(shape)),
               mean=(mean.view(n, groups), off_mean.view(n, groups)),
               rstd=(rstd.view(n, groups), (rstd * rel).view(n, groups)))
    g = dy.double().reshape(v.shape) * by
    dz = g * slope
    if act == "relu":  # a slope of 0 or 1 where z's sign may be either
        off_dz = torch.where(z.abs() <= off_z, g.abs(), 0 * g)
    else:
        off_dz = g.abs() * ((off_z + FUN * (1 + z * z)) if smooth else 0 * z)
    off_dz = off_dz + 4 * U32 * dz.abs()
    t, off_t = dz * w4, w4.abs() * off_dz + U32 * (dz * w4).abs()
    off_tx = off_t * xh.abs() + t.abs() * off_xh
    m1, m2 = over(t), over(t * xh)
    off_1 = over(off_t) + (h + 3) * U32 * over(t.abs())
    off_2 = over(off_tx) + (h + 3) * U32 * over((t * xh).abs())
    dx = rstd * (t - (0 if change == "m1" else m1) - (0 if change == "m2" else xh * m2))
    off = rstd * (off_t + off_1 + xh.abs() * off_2 + m2.abs() * off_xh
                  + 4 * U32 * (t.abs() + m1.abs() + (xh * m2).abs())) + rel * dx.abs()
    out["dx"] = (dx.reshape(shape), off.reshape(shape))
    for name, value, off in (("db", dz, off_dz), ("dw", dz * xh, off_dz * xh.abs() + dz.abs() * off_xh)):
        out[name] = (value.sum((0, 1)).view(c),
                     (off.sum((0, 1)) + h_param * U32 * value.abs().sum((0, 1))).view(c))
    return out


# rows, slabs and runs; few and many channels of a group; groups that end inside eight
# channels; a last slab of fewer groups; the largest groups
SHAPES = [((70, 96), 4), ((2, 1024), 128), ((7, 2000), 1), ((1000, 64), 8), ((2, 8192), 1), ((333, 42), 7),
          ((5, 6, 96), 4), ((5, 49, 250), 10), ((2, 2, 512), 128), ((2, 256, 72), 9), ((3, 1000, 100), 5),
          ((1, 700, 200), 4), ((40, 9, 128), 16),
          ((2, 5000, 40), 8), ((1, 70001, 8), 2), ((2, 300, 2000), 1), ((1, 20, 16384), 2), ((2, 64, 64, 100), 20),
          ((3, 2500, 330), 33), ((2, 9000, 24), 3)]
