"""Dropout, group norm and 8-bit products of more than 2^31 elements."""
import numpy as np
import pytest
import torch

import layer_reference as layer
import norm_bounds
import train_reference as ref
from mlrs_amd import prims

pytestmark = pytest.mark.gpu

BF16, P = torch.bfloat16, 0.3


def factor_at(start, count, seed, offset):
    """Dropout's factor of elements start .. start + count - 1."""
    first = start // 8
    mask = np.uint64(0xFFFFFFFF)
    i = np.arange(first, (start + count + 7) // 8, dtype=np.uint64)
    c = [i & mask, i >> np.uint64(32), np.full_like(i, offset), np.zeros_like(i)]
    k = [seed, 0]
    for _ in range(7):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & mask,
             (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & mask]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    words = np.stack(c, 1)
    halves = np.stack([words & np.uint64(0xFFFF), words >> np.uint64(16)], 2).reshape(-1)[start - 8 * first:][:count]
    t = layer.threshold(P)
    return torch.from_numpy(halves >= t).double() * (65536.0 / (65536 - t))


def test_dropout():
    n = (1 << 31) + 4099
    y = prims.dropout(torch.ones(n, dtype=BF16, device="cuda"), P, 3, 7)
    for start in (0, (1 << 31) - 5000, n - 9001):
        want = factor_at(start, 9001, 3, 7)
        ref.assert_near(y[start:start + 9001], (want, 2 * ref.U32 * want), "from %d" % start)


# rows, and slabs of a few positions
@pytest.mark.parametrize("n,positions,c,groups", [((1 << 20) + 5, 1, 2056, 2), ((1 << 21) + 3, 4, 264, 8)])
def test_norm_of_many_samples(n, positions, c, groups):
    """The last samples, whose dy alone is not zero, so that they make the parameters'
    gradients."""
    last = 40
    tail, w, b, dy = norm_bounds.inputs(1, (last, positions, c) if positions > 1 else (last, c), groups, BF16)
    x = torch.empty((n,) + tail.shape[1:], dtype=BF16, device="cuda").normal_()
    x[-last:] = tail.cuda()
    wd, bd = w.cuda(), b.cuda()
    kw = dict(weight=wd, bias=bd, activation="silu", p=P, seed=3, offset=7)
    y, mean, rstd = prims.group_norm(x, groups, keep_stats=True, **kw)
    assert x.numel() > 1 << 31 and y.isfinite().all()
    by = factor_at(x.numel() - tail.numel(), tail.numel(), 3, 7).view(tail.shape)
    want = norm_bounds.group_norm(tail, groups, w, b, 1e-5, "silu", by, dy, False)
    for name, t in (("y", y), ("mean", mean), ("rstd", rstd)):
        ref.assert_near(t[-last:], want[name], name)
    del y
    dyd = torch.zeros_like(x)
    dyd[-last:] = dy.cuda()
    dx, dw, db = prims.group_norm_grad(dyd, x, mean, rstd, **kw)
    ref.assert_near(dx[-last:], want["dx"], "dx")
    ref.assert_near(dw, want["dw"], "dw")
    ref.assert_near(db, want["db"], "db")


def test_norm_of_large_groups():
    """Runs of positions that are all alike, so that the statistics are those of one,
    with a mask that differs.  A thread adds 1,533 of them: with the rest of the sums
    1,700 additions, 1.0e-4 of the magnitudes, in the gradient's two means, and in the
    parameters' sums; the statistics are sums of differences, which are zero."""
    n, s, c, groups = 3, 1 << 20, 1000, 10
    row, w, b, dy = norm_bounds.inputs(2, (n, c), groups, BF16)
    x = row.cuda()[:, None].expand(n, s, c).contiguous()
    kw = dict(weight=w.cuda(), bias=b.cuda(), activation="silu")
    y, mean, rstd = prims.group_norm(x, groups, keep_stats=True, p=P, seed=3, offset=7, **kw)
    want = norm_bounds.group_norm(row, groups, w, b, 1e-5, "silu", None, dy, True)
    ref.assert_near(mean, want["mean"], "mean")
    ref.assert_near(rstd, want["rstd"], "rstd")
    for sample, at in ((0, 0), (1, s - 30), (2, 0), (2, 147483), (2, s - 30)):
        by = factor_at((sample * s + at) * c, 30 * c, 3, 7).view(30, c)
        value, off = (t[sample].expand(30, c) * by for t in want["y"])
        ref.assert_near(y[sample, at:at + 30], (value, off + 3 * ref.U32 * value.abs()), "y")
    del y
    dyd = dy.cuda()[:, None].expand(n, s, c).contiguous()
    dx, dw, db = prims.group_norm_grad(dyd, x, mean, rstd, **kw)
    more = 1700 * ref.U32
    for i in range(n):
        assert all(torch.equal(part, dx[i, :1].expand_as(part)) for part in dx[i].split(1 << 16))
    value, off = want["dx"]
    xh = ((row.double().view(n, groups, -1) - want["mean"][0][:, :, None]) * want["rstd"][0][:, :, None]).view(n, c)
    size = (dy.double().abs() * 1.2 * w.double().abs() * (1 + xh.abs())).view(n, groups, -1).mean(2)
    size = (want["rstd"][0] * size)[:, :, None].expand(n, groups, c // groups).reshape(n, c)
    ref.assert_near(dx[:, 0], (value, off + more * size * (1 + xh.abs())), "dx")
    for name, t, by in (("dw", dw, xh.abs()), ("db", db, torch.ones_like(xh))):
        value, off = (s * k for k in want[name])
        ref.assert_near(t, (value, off + more * s * (1.2 * dy.double().abs() * by).sum(0)), name)


def ternary(seed, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-1, 2, shape, dtype=torch.int8, device="cuda", generator=g).to(BF16)


def product(a, b):
    """a b^T of small whole numbers, exact in float32, a few rows at a time."""
    return torch.cat([(part.float() @ b.float().t()).to(BF16) for part in a.split(1 << 18)])


def test_fp8_products():
    """Values -1, 0 and 1: 8 bits hold them, and all sums are whole numbers below 2^24."""
    n, k, m = (1 << 21) + 9, 1032, 40
    big, w = ternary(1, n, k), ternary(2, m, k)
    assert big.numel() > 1 << 31
    assert torch.equal(prims.linear_fp8(big, prims.fp8_weight(w)), product(big, w))
    # big as dy of a layer of 40 inputs
    x, w8 = ternary(3, n, m), prims.fp8_weight(w.t().contiguous(), backward=True)
    dx, dw, db = prims.linear_fp8_grad(big, x, w8)
    assert torch.equal(dx, product(big, w))
    want = sum(p.float().t() @ q.float() for p, q in zip(big.split(1 << 18), x.split(1 << 18)))
    assert torch.equal(dw, want.to(BF16))
    assert torch.equal(db, sum(p.float().sum(0) for p in big.split(1 << 18)).to(BF16))
