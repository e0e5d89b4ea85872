"""The training operators from their formulas in 64 bits (8-bit optimizer
states: in the 32-bit steps that define them), with how far a result may be.

Bounds.  `U32` = 2^-24 is half a unit in the last place of float32, `UNIT[t]`
that of an operand type.  A sum of k products kept in float32 is off by at most
2 (k + 8) U32 times the sum of their magnitudes (the factor 2: the matrix cores
may truncate); a result rounded to t by UNIT[t] times itself, and by half a
subnormal step (TINY).  exp, the logistic function and erf are good to 2^-20."""
import math

import numpy as np
import torch

U32 = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 1e-38, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-38}
FUN = 2.0 ** -20


def dot_bound(k):
    return 2.0 * (k + 8) * U32


def act(z, name):
    """The activation and its slope, float64."""
    if name == "relu":
        on = (z > 0).double()
        return z * on, on
    if name == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    return z, torch.ones_like(z)


def linear(x, w, bias, name, residual):
    """(y, z) and their bounds before the last rounding."""
    x, w = x.double(), w.double()
    z = x @ w.t()
    off = dot_bound(x.shape[1]) * (x.abs() @ w.abs().t())
    if bias is not None:
        z = z + bias.double()
        off = off + U32 * z.abs()
    y, _ = act(z, name)
    off_y = 1.2 * off + (0 if name in ("none", "relu") else FUN * z.abs())  # |slope| <= 1.13
    if residual is not None:
        y = y + residual.double()
        off_y = off_y + U32 * y.abs()
    return (y, off_y), (z, off)


def linear_grad(dy, x, w, z, name, dtype):
    """((dx, bound), (dw, bound), (db, bound))."""
    dy, x, w = dy.double(), x.double(), w.double()
    dz = dy
    off = torch.zeros_like(dz)
    if name != "none":
        slope = act(z.double(), name)[1]
        dz = dy * slope
        if name != "relu":
            off = FUN * dy.abs() * (1 + z.double().abs() ** 2)
    n, m = dz.shape
    made = off + UNIT[dtype] * dz.abs() + (0 if name == "none" else TINY[dtype])
    if name == "none":
        made = off
    dx = dz @ w
    off_x = made @ w.abs() + dot_bound(m) * (dz.abs() @ w.abs())
    dw = dz.t() @ x
    off_w = made.t() @ x.abs() + dot_bound(n) * (dz.abs().t() @ x.abs())
    db = dz.sum(0)
    off_b = off.sum(0) + dot_bound(n) * dz.abs().sum(0)
    return (dx, off_x), (dw, off_w), (db, off_b)


def xent(h, w, bias, target, ignore, grad, dtype):
    """A dict of (value, bound): loss, lse, dh, dw, db."""
    h, w = h.double(), w.double()
    z = h @ w.t()
    k = h.shape[1]
    off = dot_bound(k) * (h.abs() @ w.abs().t())
    if bias is not None:
        z = z + bias.double()
        off = off + U32 * torch.where(z.isinf(), torch.zeros_like(z), z.abs())
    v = z.shape[1]
    lse = torch.logsumexp(z, dim=1)
    worst = off.amax(1)
    # positive terms: a relative error of each and of their sum is one of the sum
    off_lse = worst + 4 * FUN + dot_bound(min(v, 4096)) + 2 * U32 * lse.abs()
    kept = target != ignore
    at = torch.where(kept, target, 0)
    zt = z.gather(1, at[:, None])[:, 0]
    loss = torch.where(kept, lse - zt, torch.zeros_like(lse))
    off_loss = torch.where(kept, off_lse + worst + 2 * U32 * (lse.abs() + zt.abs()), torch.zeros_like(lse))
    p = torch.exp(z - lse[:, None])
    hot = torch.zeros_like(p)
    hot.scatter_(1, at[:, None], 1.0)
    g = torch.where(kept, grad.double(), torch.zeros_like(lse))
    far = torch.where(p > 0, (z - lse[:, None]).abs(), torch.zeros_like(p))
    off_p = p * (worst[:, None] + off_lse[:, None] + far * 2 * U32 + FUN) + 1e-37
    dz = (p - hot) * g[:, None]
    made = off_p * g.abs()[:, None] + UNIT[dtype] * dz.abs()
    if dtype == torch.float16:
        made = made + 2.0 ** -38 * g.abs().max()  # half a subnormal step, scaled back
    out = dict(loss=(loss, off_loss), lse=(lse, off_lse))
    out["dh"] = (dz @ w, made @ w.abs() + dot_bound(v) * (dz.abs() @ w.abs()))
    out["dw"] = (dz.t() @ h, made.t() @ h.abs() + dot_bound(len(h)) * (dz.abs().t() @ h.abs()))
    out["db"] = (dz.sum(0), made.sum(0) + dot_bound(len(h)) * dz.abs().sum(0))
    return out


def assert_near(got, want, what):
    """`got` (any type, any device) within its bound and its type's rounding."""
    value, bound = want
    dtype = got.dtype
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    # a result past the type's range is an infinity of its sign
    over = value.abs() - bound > torch.finfo(dtype).max * (1 + UNIT[dtype])
    value = torch.where(over, value.sign() * float("inf"), value)
    off = torch.where(over & (got == value), torch.zeros_like(value), (got - value).abs())
    room = bound + UNIT[dtype] * value.abs() * (1 + UNIT[dtype]) + TINY[dtype]
    bad = ~(off <= room)
    assert not bad.any(), "%s: %d of %d out of bounds, worst %.3g of %.3g at %s" % (
        what, int(bad.sum()), bad.numel(), float(off[bad].max()), float(room[bad].max()), bad.nonzero()[0].tolist())


# ---- the optimizer ----

def adamw(p, g, m, v, step, lr, betas, eps, decay, scale=1.0):
    """New (p, m, v) in 64 bits."""
    p, g, m, v = (np.asarray(t, dtype=np.float64) for t in (p, g, m, v))
    b1, b2 = betas
    g = g * scale
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    mh, vh = m / (1 - b1 ** step), v / (1 - b2 ** step)
    return p * (1 - lr * decay) - lr * mh / (np.sqrt(vh) + eps), m, v


def mix32(x):
    x = np.asarray(x, dtype=np.uint64)
    x = ((x ^ (x >> np.uint64(16))) * np.uint64(0x6A09E667)) & np.uint64(0xFFFFFFFF)
    x = ((x ^ (x >> np.uint64(15))) * np.uint64(0xBB67AE85)) & np.uint64(0xFFFFFFFF)
    return x ^ (x >> np.uint64(16))


def code_values(code, mant):
    """A magnitude's code: four bits of exponent (15 is 2^0), `mant` of fraction."""
    code = np.asarray(code, dtype=np.int64)
    e, f = code >> mant, code & ((1 << mant) - 1)
    return np.where(e > 0, np.ldexp(1.0 + f / (1 << mant), e - 15), f * 2.0 ** (-14 - mant)).astype(np.float32)


def codes_of(y, r16, mant):
    """Codes of magnitudes, rounded up where the remainder of a step, in 65536
    parts of it rounded down, and r16 reach a whole step."""
    y = np.asarray(y, dtype=np.float64)
    e = np.floor(np.log2(np.maximum(y, 2.0 ** -40)))
    e = np.where(np.ldexp(1.0, e.astype(int)) > y, e - 1, e)
    e = np.maximum(e, -14)
    quantum = np.ldexp(1.0, (e - mant).astype(int))
    steps = y / quantum  # exact: a power of two
    r = np.asarray(r16, dtype=np.float64)
    normal = y >= 2.0 ** -14
    # below 2^-14 the sum of the steps and the random part is one float32 sum
    small = np.floor(np.float32(steps) + np.float32(r * 2.0 ** -16)).astype(np.int64)
    big = np.floor(steps + r * 2.0 ** -16).astype(np.int64) + ((e + 14).astype(np.int64) << mant)
    return np.minimum(np.where(normal, big, small), (16 << mant) - 1)


def adamw8(p, g, codes_m, codes_r, scale_m, scale_r, ordinal, step, lr, betas, eps, decay, seed, scale=1.0, first=0):
    """New (p, codes_m, codes_r, scale_m, scale_r) of one tensor, or of its
    elements from `first` (a multiple of 256) on, by the float32 steps of the
    definition, each rounded by itself."""
    f = np.float32
    n, block = len(p), 256
    sm, sr = (np.repeat(s, block)[:n] for s in (scale_m, scale_r))
    b1, b2 = betas
    m = code_values(codes_m & 127, 3)
    m = np.where(codes_m > 127, -m, m) * sm
    r = code_values(codes_r, 4) * sr
    g = g.astype(f) * f(scale)
    v = r * r
    m = m * f(b1) + g * f(1 - b1)
    v = v * f(b2) + (g * f(1 - b2)) * g
    r = np.sqrt(v)
    root, step_size = f(1 / math.sqrt(1 - b2 ** step)), f(lr / (1 - b1 ** step))
    p = p * f(1 - lr * decay) - (m / (r * root + f(eps))) * step_size
    pad = -(-n // block) * block - n
    new_sm = np.pad(np.abs(m), (0, pad)).reshape(-1, block).max(1) / f(1.875)
    new_sr = np.pad(r, (0, pad)).reshape(-1, block).max(1) / f(1.9375)
    key = mix32((seed + ordinal * 0x9E3779B1) & 0xFFFFFFFF)
    index = np.arange(first, first + n, dtype=np.uint64)
    low, high = index & np.uint64(0xFFFFFFFF), index >> np.uint64(32)
    u = mix32(((low ^ key) + high * np.uint64(0x9E3779B1)) & np.uint64(0xFFFFFFFF))
    sm, sr = (np.repeat(s, block)[:n] for s in (new_sm, new_sr))
    with np.errstate(divide="ignore", invalid="ignore"):
        ym = np.where(sm > 0, np.abs(m) / sm, f(0))
        yr = np.where(sr > 0, r / sr, f(0))
    cm = codes_of(ym, u & np.uint64(0xFFFF), 3) + np.where(m < 0, 128, 0)
    cr = codes_of(yr, u >> np.uint64(16), 4)
    cr = np.where((r > 0) & (cr == 0), 1, cr)
    return p, cm.astype(np.uint8), cr.astype(np.uint8), new_sm, new_sr
