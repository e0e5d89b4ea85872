"""The training operators on the GPU against their formulas in 64 bits."""
import numpy as np
import pytest
import torch

import train_reference as ref
from mlrs_amd import _lib, prims

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
IGNORE = -100


def rand(seed, *shape, dtype=F32, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * std).to(dtype)


def dev(t, offset=0):
    """On the GPU; with `offset` elements before it, so that it is aligned to
    its element size alone."""
    if t is None:
        return None
    if not offset:
        return t.cuda()
    flat = torch.empty(t.numel() + offset, dtype=t.dtype, device="cuda")
    view = flat[offset:].view(t.shape)
    view.copy_(t)
    return view


def check_linear(n, k, m, dtype, act, bias=True, residual=True, keep=True, offset=0, seed=0):
    x, w = rand(seed, n, k, dtype=dtype), rand(seed + 1, m, k, dtype=dtype, std=k ** -0.5)
    b = rand(seed + 2, m, dtype=dtype, std=0.3) if bias else None
    res = rand(seed + 3, n, m, dtype=dtype) if residual else None
    got = prims.linear(dev(x, offset), dev(w, offset), bias=dev(b, offset), activation=act,
                       residual=dev(res, offset), keep_preact=keep)
    y, z = got if keep else (got, None)
    want_y, want_z = ref.linear(x, w, b, act, res)
    what = "linear n=%d k=%d m=%d %s %s" % (n, k, m, dtype, act)
    ref.assert_near(y, want_y, what + " y")
    if keep:
        ref.assert_near(z, want_z, what + " z")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_linear_activations(dtype, act):
    check_linear(70, 96, 80, dtype, act)
    check_linear(5, 96, 80, dtype, act)


# one row and few rows; one column, one output; sizes around the widths of a
# fragment, a wave, a tile and a staged width; none a multiple of the next
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,m", [
    (1, 1, 1), (1, 64, 16), (1, 1000, 33), (3, 17, 5), (15, 63, 31), (16, 64, 32), (17, 65, 33), (32, 128, 48),
    (33, 129, 47), (63, 40, 100), (64, 512, 64), (65, 1, 65), (66, 64, 64), (127, 100, 129), (128, 256, 128),
    (129, 31, 257), (257, 257, 130), (300, 72, 520), (1000, 33, 7),
])
def test_linear_sizes(dtype, n, k, m):
    check_linear(n, k, m, dtype, "gelu", seed=n + k + m)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias,residual,keep", [(False, False, False), (True, False, True), (False, True, False)])
@pytest.mark.parametrize("n", [9, 130])
def test_linear_options(dtype, bias, residual, keep, n):
    check_linear(n, 72, 136, dtype, "silu", bias, residual, keep)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,m", [(7, 64, 40), (100, 64, 64), (131, 65, 67)])
@pytest.mark.parametrize("offset", [1, 3])
def test_linear_unaligned(dtype, n, k, m, offset):
    check_linear(n, k, m, dtype, "relu", offset=offset)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_every_tile(dtype):
    """Sizes that the rule gives the largest tile, the middle one, and parts of
    a long contraction."""
    check_linear(2100, 72, 2100, dtype, "gelu_tanh", seed=3)
    check_linear(1100, 40, 1030, dtype, "none", seed=4)
    check_linear(130, 8200, 130, dtype, "silu", seed=5)


def test_linear_no_rows_and_in_place():
    w = dev(rand(1, 24, 16))
    assert prims.linear(torch.empty(0, 16, device="cuda"), w).shape == (0, 24)
    x, res = rand(2, 90, 16), rand(3, 90, 24)
    r = dev(res)
    y = prims.linear(dev(x), w, residual=r, out=r)
    assert y.data_ptr() == r.data_ptr()
    ref.assert_near(y, ref.linear(x, w.cpu(), None, "none", res)[0], "residual's buffer")


def test_linear_out_is_no_operand():
    x, w, r = (dev(rand(i, 64, 64)) for i in range(3))
    both = torch.empty(65, 64, device="cuda")
    for kw in (dict(out=x), dict(out=w), dict(out=both[1:], residual=both[:-1])):
        with pytest.raises(_lib.InvalidParam, match="overlaps"):
            prims.linear(x, w, **kw)
    ref.assert_near(prims.linear(x, w, residual=r), ref.linear(x.cpu(), w.cpu(), None, "none", r.cpu())[0], "after")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [4, 100])
def test_linear_infinities_stay_in_their_rows(dtype, n):
    x, w = rand(5, n, 40, dtype=dtype), rand(6, 50, 40, dtype=dtype, std=0.1)
    clean = prims.linear(dev(x), dev(w))
    x[1, 3] = float("inf")
    x[2, 7] = float("nan")
    got = prims.linear(dev(x), dev(w))
    keep = [i for i in range(n) if i not in (1, 2)]
    assert torch.equal(got[keep], clean[keep])
    assert got[2].isnan().all()
    want = torch.where(w[:, 3].float() > 0, float("inf"), float("-inf"))
    assert torch.equal(got[1].float().cpu(), want)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_tail_of_k_reads_no_neighbours(dtype):
    """Rows that end inside a staged width: the next row's elements, NaN here,
    must not reach the sum."""
    n, k, m = 70, 24, 70
    x, w = rand(7, n, k, dtype=dtype), rand(8, m, k, dtype=dtype)
    x[1::2] = float("nan")
    w[1::2] = float("nan")
    got = prims.linear(dev(x), dev(w))[::2, ::2]
    assert not got.isnan().any()
    ref.assert_near(got, ref.linear(x[::2], w[::2], None, "none", None)[0], "rows between NaN rows")


def test_layer_of_more_elements_than_32_bits_count():
    """70,000 x 65,536 outputs: the last rows and columns are where they belong."""
    n, k, m = 70000, 32, 65536
    x, w = rand(1, n, k, dtype=BF16), rand(2, m, k, dtype=BF16, std=0.2)
    xd, wd = dev(x), dev(w)
    y = prims.linear(xd, wd, activation="relu")
    for r in (slice(0, 3), slice(32767, 32770), slice(65534, 65538), slice(n - 3, n)):
        ref.assert_near(y[r], ref.linear(x[r], w, None, "relu", None)[0], "rows %s" % r)
    dx, dw, db = prims.linear_grad(y, xd, wd)
    ones = torch.ones(n, dtype=torch.float64, device="cuda")
    for r in (slice(0, 2), slice(65535, 65537), slice(n - 2, n)):
        want = ref.linear_grad(y[r].cpu(), x[r], w, None, "none", BF16)
        ref.assert_near(dx[r], want[0], "dx rows %s" % r)
    for c in (slice(0, 64), slice(m - 64, m)):
        part = y[:, c].double()
        size = part.t().abs() @ xd.double().abs()
        room = (ref.dot_bound(n) + ref.UNIT[BF16]) * size
        assert bool(((dw[c].double() - part.t() @ xd.double()).abs() <= room).all())
        assert bool(((db[c].double() - ones @ part).abs() <= (ref.dot_bound(n) + ref.UNIT[BF16]) * (ones @ part.abs())).all())


def check_grad(n, k, m, dtype, act, offset=0, seed=0, bias=True):
    x, w = rand(seed, n, k, dtype=dtype), rand(seed + 1, m, k, dtype=dtype, std=k ** -0.5)
    dy = rand(seed + 2, n, m, dtype=dtype, std=0.1)
    z = rand(seed + 3, n, m, dtype=dtype) if act != "none" else None
    dx, dw, db = prims.linear_grad(dev(dy, offset), dev(x, offset), dev(w, offset), preact=dev(z, offset),
                                   activation=act, bias=bias)
    want = ref.linear_grad(dy, x, w, z, act, dtype)
    what = "linear_grad n=%d k=%d m=%d %s %s " % (n, k, m, dtype, act)
    ref.assert_near(dx, want[0], what + "dx")
    ref.assert_near(dw, want[1], what + "dw")
    if bias:
        ref.assert_near(db, want[2], what + "db")
    else:
        assert db is None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_linear_grad_activations(dtype, act):
    check_grad(70, 96, 80, dtype, act)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,m", [
    (1, 1, 1), (1, 64, 64), (2, 33, 17), (31, 8, 9), (63, 65, 64), (64, 64, 64), (65, 63, 66), (128, 40, 200),
    (129, 257, 31), (300, 72, 520), (513, 130, 66),
])
def test_linear_grad_sizes(dtype, n, k, m):
    check_grad(n, k, m, dtype, "silu", seed=n + k + m)
    check_grad(n, k, m, dtype, "none", seed=n + k + m, bias=False)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_grad_unaligned_and_every_tile(dtype):
    check_grad(70, 64, 72, dtype, "gelu", offset=1)
    check_grad(70, 64, 72, dtype, "none", offset=3)
    check_grad(2100, 2100, 40, dtype, "relu", seed=1)
    check_grad(40, 2100, 2100, dtype, "relu", seed=2)
    check_grad(8300, 72, 66, dtype, "gelu_tanh", seed=3)
    check_grad(66, 72, 8300, dtype, "none", seed=4)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_grad_no_rows(dtype):
    x, w = torch.empty(0, 24, device="cuda", dtype=dtype), dev(rand(1, 40, 24, dtype=dtype))
    dy = torch.empty(0, 40, device="cuda", dtype=dtype)
    for act, z in (("none", None), ("relu", dy)):
        dx, dw, db = prims.linear_grad(dy, x, w, preact=z, activation=act)
        assert dx.shape == (0, 24) and not dw.any() and not db.any()
        assert dw.shape == (40, 24) and db.shape == (40,)


def test_linear_grad_parts_asked_for():
    n, k, m = 50, 16, 24
    x, w, dy = (dev(rand(i, *s)) for i, s in enumerate([(n, k), (m, k), (n, m)]))
    all3 = prims.linear_grad(dy, x, w)
    for need in range(8):
        got = prims.linear_grad(dy, x, w, bias=bool(need & 1), need_dx=bool(need & 2), need_dw=bool(need & 4))
        for part, asked, whole in zip(got, (need & 2, need & 4, need & 1), all3):
            assert torch.equal(part, whole) if asked else part is None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_activations_of_the_largest_numbers(dtype, act):
    """Far from zero an activation is z or 0 and its slope 1 or 0, up to the
    largest finite number, whose square and cube f32 cannot hold."""
    most = torch.finfo(dtype).max
    far = torch.tensor([t for t in (300.0, 6e4, 1e10, 1e13, 2e19, 1e20, 1e38, most) if t <= most], dtype=dtype)
    z = torch.cat([far, -far])
    one = torch.ones(1, 1, dtype=dtype)
    y, kept = prims.linear(dev(z[:, None]), dev(one), activation=act, keep_preact=True)
    assert torch.equal(kept.cpu()[:, 0], z)
    on = torch.cat([torch.ones_like(far), torch.zeros_like(far) if act != "none" else torch.ones_like(far)])
    assert torch.equal(y.cpu()[:, 0], z * on)
    dx, dw, db = prims.linear_grad(torch.ones_like(y), torch.ones_like(y), dev(one), preact=kept, activation=act)
    assert torch.equal(dx.cpu()[:, 0], on) and float(dw) == float(db) == float(on.sum())


def test_linear_grad_against_differences():
    """Along random directions, the loss sum(c * y) in 64 bits changes by what
    the kernel's float32 gradient says."""
    n, k, m, e = 40, 24, 32, 1e-5
    x, w, b, c = rand(1, n, k), rand(2, m, k, std=0.2), rand(3, m), rand(4, n, m)
    for act in ("gelu", "gelu_tanh", "silu"):
        _, z = prims.linear(dev(x), dev(w), bias=dev(b), activation=act, keep_preact=True)
        grads = prims.linear_grad(dev(c), dev(x), dev(w), preact=z, activation=act)
        for i, (t, g) in enumerate(zip((x, w, b), grads)):
            u = rand(9 + i, *t.shape).double()

            def value(s):
                a = [q.double() + (s * u if j == i else 0) for j, q in enumerate((x, w, b))]
                return float((c.double() * ref.act(a[0] @ a[1].t() + a[2], act)[0]).sum())

            slope = (value(e) - value(-e)) / (2 * e)
            got = float((g.cpu().double() * u).sum())
            # differences: e^2 of the third derivative and 2^-52 / e of the value;
            # the gradient: 2^-20 of each of its terms
            room = 1e-6 * float((g.cpu().double() * u).abs().sum()) + 1e-5
            assert abs(got - slope) <= room, (act, i, got, slope)


def targets(seed, n, v, ignored=0.2):
    g = torch.Generator().manual_seed(seed)
    t = torch.randint(0, v, (n,), generator=g)
    t[torch.rand(n, generator=g) < ignored] = IGNORE
    return t


def check_xent(n, v, k, dtype, bias=True, offset=0, seed=0, spread=1.5, masked=(), grad=None):
    h, w = rand(seed, n, k, dtype=dtype), rand(seed + 1, v, k, dtype=dtype, std=spread * k ** -0.5)
    b = rand(seed + 2, v, dtype=dtype, std=0.5) if bias else None
    t = targets(seed + 3, n, v)
    for c in masked:
        b[c] = float("-inf")
        t[t == c] = IGNORE
    g = rand(seed + 4, n).abs() / n if grad is None else grad
    args = [dev(h, offset), dev(w, offset), dev(t)]
    loss, lse = prims.softmax_xent(*args, bias=dev(b, offset), ignore_index=IGNORE)
    dh, dw, db = prims.softmax_xent_grad(*args, lse, dev(g), bias=dev(b, offset), ignore_index=IGNORE)
    want = ref.xent(h, w, b, t, IGNORE, g, dtype)
    what = "softmax_xent n=%d v=%d k=%d %s " % (n, v, k, dtype)
    for name, got in (("loss", loss), ("lse", lse), ("dh", dh), ("dw", dw), ("db", db)):
        if name == "db" and not bias:
            assert got is None
        else:
            ref.assert_near(got, want[name], what + name)
    gone = (t == IGNORE).cuda()
    assert not loss[gone].any() and not dh[gone].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,k", [
    (1, 1, 1), (1, 2, 3), (1, 1000, 64), (2, 63, 8), (31, 64, 33), (32, 65, 64), (33, 127, 65), (64, 128, 128),
    (65, 129, 17), (100, 257, 40), (129, 1000, 130), (300, 777, 64), (7, 5000, 24),
])
def test_xent_sizes(dtype, n, v, k):
    check_xent(n, v, k, dtype, seed=n + v + k)
    check_xent(n, v, k, dtype, bias=False, seed=n + v + k)


@pytest.mark.parametrize("dtype", TYPES)
def test_xent_unaligned_and_every_tile(dtype):
    check_xent(40, 96, 64, dtype, offset=1)
    check_xent(2100, 2100, 24, dtype, seed=1)
    check_xent(1030, 1100, 40, dtype, seed=2)


# a few tiles of logits, each a long sum: computed in parts of the contraction
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,k", [(1, 5, 4096), (17, 1000, 2048), (76, 344, 3473), (129, 66, 5003)])
def test_xent_few_classes_and_long_rows(dtype, n, v, k):
    check_xent(n, v, k, dtype, seed=n + v + k)
    check_xent(n, v, k, dtype, bias=False, offset=1, seed=n + v)
    if v > 300:
        check_xent(n, v, k, dtype, masked=list(range(0, 260)) + [v - 1], seed=n)


@pytest.mark.parametrize("dtype", TYPES)
def test_xent_long_rows_that_are_not_finite(dtype):
    """A row with a NaN, one whose logits are all -inf and one whose target is no
    class leave the others as they are."""
    n, v, k = 70, 130, 4000
    h, w, t = rand(1, n, k, dtype=dtype), rand(2, v, k, dtype=dtype, std=0.03), targets(3, n, v, ignored=0.0)
    g = torch.full((n,), 1.0 / n)
    plain = prims.softmax_xent(dev(h), dev(w), dev(t))
    dz = prims.softmax_xent_grad(dev(h), dev(w), dev(t), plain[1], dev(g), need_dw=False)[0]
    w[:, 7], h[:, 7] = w[:, 7].abs() + 0.5, 0.0
    base = prims.softmax_xent(dev(h), dev(w), dev(t))
    h[5, 9], h[6, 7], t[8] = float("nan"), float("-inf"), v
    loss, lse = prims.softmax_xent(dev(h), dev(w), dev(t))
    dh = prims.softmax_xent_grad(dev(h), dev(w), dev(t), lse, dev(g), need_dw=False)[0]
    assert loss[5].isnan() and lse[5].isnan() and lse[6] == float("-inf") and loss[8].isnan()
    assert dh[5].isnan().all() and dh[8].isnan().all()
    kept = [i for i in range(n) if i not in (5, 6, 8)]
    assert torch.equal(loss[kept], base[0][kept]) and torch.equal(lse[kept], base[1][kept])
    assert dh[kept].isfinite().all() and dz.isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_xent_wide_logits(dtype):
    """Logits tens apart: one class has nearly all of a row, others nothing."""
    check_xent(70, 300, 64, dtype, spread=20.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_xent_masked_classes(dtype):
    """Classes left out by a bias of -inf, whole tiles of them and the first and
    the last among them, take no part and get no gradient."""
    n, v, k = 40, 700, 32
    masked = list(range(0, 260)) + [300] + list(range(690, 700))
    check_xent(n, v, k, dtype, masked=masked)
    h, w, t = rand(1, n, k, dtype=dtype), rand(2, v, k, dtype=dtype), targets(3, n, v)
    b = torch.zeros(v, dtype=dtype)
    b[masked] = float("-inf")
    t[torch.isin(t, torch.tensor(masked))] = IGNORE
    loss, lse = prims.softmax_xent(dev(h), dev(w), dev(t), bias=dev(b))
    _, dw, db = prims.softmax_xent_grad(dev(h), dev(w), dev(t), lse, torch.ones(n, device="cuda"), bias=dev(b))
    assert loss.isfinite().all() and lse.isfinite().all()
    assert not dw[masked].any() and not db[masked].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_xent_many_rows_in_pieces(dtype):
    """More rows than the statistics have room for at a time, and a gradient of
    the logits of several pieces, the last of them short and odd.  The 64-bit
    reference is computed on the GPU (its products are float64)."""
    n, v, k = 56000, 20011, 16
    h, w, b = rand(1, n, k, dtype=dtype).cuda(), rand(2, v, k, dtype=dtype, std=0.4).cuda(), rand(3, v, dtype=dtype).cuda()
    t = targets(4, n, v).cuda()
    g = torch.full((n,), 1.0 / n, device="cuda")
    loss, lse = prims.softmax_xent(h, w, t, bias=b)
    dh, dw, db = prims.softmax_xent_grad(h, w, t, lse, g, bias=b)
    hd, wd = h.double(), w.double()
    want_dw, want_db = torch.zeros_like(wd), torch.zeros(v, dtype=torch.float64, device="cuda")
    for a in range(0, n, 14000):
        part = slice(a, a + 14000)
        z = hd[part] @ wd.t() + b.double()
        l = torch.logsumexp(z, 1)
        kept = t[part] != IGNORE
        at = torch.where(kept, t[part], 0)[:, None]
        # the logits are sums of 17 terms of size up to about ten, the sum of
        # exponentials one of 20,011: 2^-19 covers both
        assert (lse[part] - l).abs().max() < 2.0 ** -19 * 16
        want = torch.where(kept, l - z.gather(1, at)[:, 0], 0.0)
        assert (loss[part] - want).abs().max() < 2.0 ** -19 * 16
        d = torch.exp(z - l[:, None])
        d.scatter_add_(1, at, torch.full_like(l, -1.0)[:, None])
        d *= (kept / n)[:, None]
        want = d @ wd
        # each term is rounded once to the type, and the result
        unit = ref.UNIT[dtype]
        room = 2 * unit * (d.abs() @ wd.abs()) + unit * want.abs() + 2.0 ** -18 * (d.abs() @ wd.abs())
        assert bool(((dh[part].double() - want).abs() <= room).all())
        want_dw += d.t() @ hd[part]
        want_db += d.sum(0)
        del z, d
    size = want_dw.abs().max()
    assert (dw.double() - want_dw).abs().max() <= (4 * ref.UNIT[dtype] + 2.0 ** -16) * size
    assert (db.double() - want_db).abs().max() <= (4 * ref.UNIT[dtype] + 2.0 ** -16) * want_db.abs().max()


def pieces_inputs(n, v, k, dtype):
    h, w, b = rand(1, n, k, dtype=dtype).cuda(), rand(2, v, k, dtype=dtype, std=1.5 * k ** -0.5).cuda(), rand(
        3, v, dtype=dtype, std=0.5).cuda()
    return h, w, b, targets(4, n, v).cuda(), (rand(5, n).abs() / n).cuda()


def check_pieces(got, want, names, rows=slice(None)):
    for name, g in got.items():
        if name in names:
            value, bound = want[name]
            one = name in ("loss", "lse", "dh")
            ref.assert_near(g[rows] if one else g, (value[rows].cpu(), bound[rows].cpu()) if one else (
                value.cpu(), bound.cpu()), name)


def all_outputs(h, w, t, g, b):
    loss, lse = prims.softmax_xent(h, w, t, bias=b)
    dh, dw, db = prims.softmax_xent_grad(h, w, t, lse, g, bias=b)
    return dict(loss=loss, lse=lse, dh=dh, dw=dw, db=db)


# Gradients of two to four pieces, the last of them shorter and odd; the 64-bit
# reference is computed on the GPU.  f32: all three products in three bf16 parts,
# rows in place or packed; dh in parts of its contraction, of which the last piece
# has fewer; the logits alone in bf16 parts; none.
@pytest.mark.parametrize("n,v,k,dtype", [
    (16384, 20011, 512, F32), (16384, 20011, 511, F32), (40000, 7003, 512, F32), (20000, 16001, 300, F32),
    (270001, 1101, 61, F32), (270001, 2103, 24, F16), (270001, 2103, 24, BF16), (100003, 6007, 40, F16),
])
def test_xent_gradients_of_several_pieces(n, v, k, dtype):
    h, w, b, t, g = pieces_inputs(n, v, k, dtype)
    want = ref.xent(h, w, b, t, IGNORE, g, dtype)
    check_pieces(all_outputs(h, w, t, g, b), want, want)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n,v,k", [(16384, 20011, 512), (16384, 20011, 511), (20000, 16001, 300)])
def test_xent_pieces_that_f32_takes_over(n, v, k):
    """A class of the last piece with an element that has no bf16 parts (all rows
    are 0 there), and a row whose target is no class: the f32 kernels take over
    in the middle of the call, and everything beside them is what it was."""
    h, w, b, t, g = pieces_inputs(n, v, k, F32)
    h[:, 3] = 0.0
    want = ref.xent(h, w, b, t, IGNORE, g, F32)
    w[v - 5, 3] = torch.finfo(F32).max
    got = all_outputs(h, w, t, g, b)
    cols = [i for i in range(k) if i != 3]
    got["dh"], want["dh"] = got["dh"][:, cols], tuple(x[:, cols] for x in want["dh"])
    check_pieces(got, want, want)
    w[v - 5, 3] = 0.0
    t[77] = v
    got = all_outputs(h, w, t, g, b)
    rows = torch.arange(n, device="cuda") != 77
    got["dh"] = got["dh"][:, cols]
    check_pieces(got, want, ("loss", "lse", "dh"), rows)
    assert got["loss"][77].isnan() and got["dh"][77].isnan().all()
    assert got["dw"].isnan().all() and got["db"].isnan().all()
    torch.cuda.empty_cache()


def test_xent_of_more_logits_than_a_launch_has_tiles_for():
    """4,300,800 rows of 128,003 classes: the loss in chunks of rows, the gradient
    in pieces of the vocabulary, neither of them a launch's worth of all tiles.
    Some rows and some classes are held to 64 bits."""
    n, v, k = 4300800, 128003, 8
    h, w = rand(1, n, k, dtype=BF16).cuda(), rand(2, v, k, dtype=BF16, std=0.4).cuda()
    t = targets(3, n, v).cuda()
    g = torch.full((n,), 1.0 / n, device="cuda")
    loss, lse = prims.softmax_xent(h, w, t)
    dh, dw, _ = prims.softmax_xent_grad(h, w, t, lse, g)
    rows = torch.cat([torch.arange(a, a + 40) for a in (0, 255 * 256, n // 2, n - 40)]).cuda()
    want = ref.xent(h[rows].cpu(), w.cpu(), None, t[rows].cpu(), IGNORE, g[rows].cpu(), BF16)
    for name, got in (("loss", loss), ("lse", lse), ("dh", dh)):
        ref.assert_near(got[rows], want[name], name)
    for c in (0, 64000, v - 32):
        p = torch.exp(h.double() @ w[c:c + 32].double().t() - lse.double()[:, None])
        hot = (t[:, None] == torch.arange(c, c + 32, device="cuda")).double()
        dz = (p - hot) * (t != IGNORE).double()[:, None] * g.double()[:, None]
        room = (2 * ref.UNIT[BF16] + ref.dot_bound(n)) * (dz.abs().t() @ h.double().abs())
        assert bool(((dw[c:c + 32].double() - dz.t() @ h.double()).abs() <= room).all())


def test_layer_of_more_outputs_than_a_launch_has_threads_for():
    """Few rows by 2^27 + 40 outputs, sixteen to a workgroup."""
    m = 2 ** 27 + 40
    w = torch.arange(m, device="cuda").remainder_(2039).half()[:, None]
    for n in (1, 17):
        x = torch.arange(1, n + 1, device="cuda").half()[:, None]
        y = prims.linear(x, w)
        assert all(torch.equal(y[i], w[:, 0] * x[i, 0]) for i in (0, n - 1))
        del y


def test_layers_and_losses_of_more_rows_than_a_launch_has_threads_for():
    """2^30 + 77 rows of eight features, 64 of them to a small tile.  Zero but for
    runs of 300 rows, of small whole numbers: every sum is exact."""
    n, k, m = 2 ** 30 + 77, 8, 8
    runs = [slice(a, a + 300) for a in (0, 2 ** 24, 2 ** 29, n - 300)]
    small = [rand(i, 4, 300, k).mul(2).round().clamp(-7, 7).to(BF16).cuda() for i in (1, 2)]
    w = rand(3, m, k).mul(2).round().clamp(-7, 7).to(BF16).cuda()
    x = torch.zeros(n, k, dtype=BF16, device="cuda")
    for r, t in zip(runs, small[0]):
        x[r].copy_(t)
    y = prims.linear(x, w)
    for r, t in zip(runs, small[0]):
        assert torch.equal(y[r].double(), (t.double() @ w.double().t()).bfloat16().double())
    assert not y[300:2 ** 24].any() and not y[2 ** 24 + 300:2 ** 24 + 3000].any()
    dy = y.zero_()
    for r, t in zip(runs, small[1]):
        dy[r].copy_(t)
    dx, dw, db = prims.linear_grad(dy, x, w)
    for r, t in zip(runs, small[1]):
        assert torch.equal(dx[r].double(), (t.double() @ w.double()).bfloat16().double())
    assert not dx[300:2 ** 24].any() and not dx[2 ** 24 + 300:2 ** 24 + 3000].any()
    flat = [t.reshape(-1, k).double() for t in small]
    assert torch.equal(dw, (flat[1].t() @ flat[0]).bfloat16()) and torch.equal(db, flat[1].sum(0).bfloat16())
    del dx, dy, y
    t = torch.zeros(n, dtype=torch.int64, device="cuda")
    loss, lse = prims.softmax_xent(x, w[:2], t)
    for r, h in zip(runs, small[0]):
        want = ref.xent(h.cpu(), w[:2].cpu(), None, t[r].cpu(), IGNORE, torch.ones(300), BF16)
        ref.assert_near(loss[r], want["loss"], "loss")
        ref.assert_near(lse[r], want["lse"], "lse")
    assert float((lse[300:2 ** 24] - 0.6931472).abs().max()) < 2.0 ** -20  # log 2 of zero rows
    del x, t, loss, lse
    torch.cuda.empty_cache()


def test_gradients_of_no_rows_and_many_classes():
    """2^28 + 40 of them: their zeros are sixteen to a workgroup."""
    w = torch.ones(2 ** 28 + 40, 1, dtype=BF16, device="cuda")
    e = torch.empty(0, device="cuda")
    dh, dw, db = prims.softmax_xent_grad(torch.empty(0, 1, dtype=BF16, device="cuda"), w,
                                         torch.empty(0, dtype=torch.int64, device="cuda"), e, e, bias=w[:, 0])
    assert dh.shape == (0, 1) and not dw.any() and not db.any()


def test_xent_target_that_is_masked_or_no_class():
    h, w = rand(1, 6, 16), rand(2, 50, 16)
    b = torch.zeros(50)
    b[4] = float("-inf")
    t = torch.tensor([4, 50, -1, 3, IGNORE, 49])
    loss, lse = prims.softmax_xent(dev(h), dev(w), dev(t), bias=dev(b))
    assert loss[0] == float("inf") and loss[1].isnan() and loss[2].isnan()
    assert loss[3:].isfinite().all() and loss[4] == 0 and lse.isfinite().all()
    dh, _, _ = prims.softmax_xent_grad(dev(h), dev(w), dev(t), lse, torch.ones(6, device="cuda"), bias=dev(b))
    assert dh[1].isnan().all() and dh[2].isnan().all() and dh[3].isfinite().all() and not dh[4].any()


def test_xent_all_rows_ignored_and_no_rows():
    for dtype in TYPES:
        h, w, b = rand(1, 20, 16, dtype=dtype), dev(rand(2, 50, 16, dtype=dtype)), dev(rand(3, 50, dtype=dtype))
        t = torch.full((20,), IGNORE)
        loss, lse = prims.softmax_xent(dev(h), w, dev(t), bias=b)
        assert not loss.any() and lse.isfinite().all()
        parts = prims.softmax_xent_grad(dev(h), w, dev(t), lse, torch.ones(20, device="cuda"), bias=b)
        assert not any(p.any() for p in parts)
        e = torch.empty(0, device="cuda")
        none = torch.empty(0, dtype=torch.int64, device="cuda")
        loss, lse = prims.softmax_xent(dev(h)[:0], w, none, bias=b)
        assert loss.shape == (0,) and lse.shape == (0,)
        dh, dw, db = prims.softmax_xent_grad(dev(h)[:0], w, none, e, e, bias=b)
        assert dh.shape == (0, 16) and dw.shape == (50, 16) and not dw.any() and not db.any()


def test_xent_rows_with_nan_stay_alone():
    h, w, t = rand(1, 70, 32), dev(rand(2, 300, 32)), dev(targets(4, 70, 300, 0.0))
    clean = prims.softmax_xent(dev(h), w, t)
    h[3, 5] = float("nan")
    loss, lse = prims.softmax_xent(dev(h), w, t)
    keep = [i for i in range(70) if i != 3]
    assert torch.equal(loss[keep], clean[0][keep]) and torch.equal(lse[keep], clean[1][keep])
    assert loss[3].isnan() and lse[3].isnan()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,k", [(70, 300, 32), (70, 130, 4000)])
def test_xent_rows_with_infinite_logits_stay_alone(dtype, n, v, k):
    h, w, t = rand(1, n, k, dtype=dtype), rand(2, v, k, dtype=dtype, std=k ** -0.5), targets(3, n, v, 0.0)
    w[:, 5] = w[:, 5].abs() + 0.1
    t[9] = IGNORE
    clean = prims.softmax_xent(dev(h), dev(w), dev(t))
    h[3, 5] = h[9, 5] = float("inf")
    loss, lse = prims.softmax_xent(dev(h), dev(w), dev(t))
    dh, _, _ = prims.softmax_xent_grad(dev(h), dev(w), dev(t), lse, torch.ones(n, device="cuda"), need_dw=False)
    keep = [i for i in range(n) if i not in (3, 9)]
    assert torch.equal(loss[keep], clean[0][keep]) and torch.equal(lse[keep], clean[1][keep])
    assert loss[3].isnan() and lse[3].isnan() and loss[9] == 0 and lse[9].isnan()
    assert dh[3].isnan().all() and not dh[9].any() and dh[keep].isfinite().all()


@pytest.mark.parametrize("size", [1e-6, 1.0, 3e4])
def test_xent_half_precision_gradient_range(size):
    """Gradients far below and above half precision's range times probabilities
    of a large vocabulary keep their accuracy; the outputs are what their type
    can hold."""
    n, v, k = 64, 3000, 64
    h, w, t = rand(1, n, k, dtype=F16), rand(2, v, k, dtype=F16, std=0.05), targets(3, n, v)
    g = torch.full((n,), size)
    _, lse = prims.softmax_xent(dev(h), dev(w), dev(t))
    dh, dw, _ = prims.softmax_xent_grad(dev(h), dev(w), dev(t), lse, dev(g))
    want = ref.xent(h, w, None, t, IGNORE, g, F16)
    ref.assert_near(dh, want["dh"], "dh")
    ref.assert_near(dw, want["dw"], "dw")


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_xent_common_gradient_is_not_rounded(dtype):
    """Rows that share a gradient g halfway between two numbers of the type, three
    of them to a target's class, and probabilities of 1 / v: a class's sum is
    -3 g but for 3 g / v.  With u the type's unit its rounding costs u / 3, as
    3 + 3 u lies a quarter of a step from 3 + 4 u; rounding p - 1 costs p at most;
    each row's g rounded by itself would cost u."""
    n, v, k = 24, 40000, 16
    unit = ref.UNIT[dtype]
    g = (1.0 + unit) / 32.0
    h, w = rand(1, n, k, dtype=dtype), rand(2, v, k, dtype=dtype, std=0.001)
    t, b = torch.arange(n) // 3 * 200, torch.zeros(v, dtype=dtype)
    _, lse = prims.softmax_xent(dev(h), dev(w), dev(t), bias=dev(b))
    _, _, db = prims.softmax_xent_grad(dev(h), dev(w), dev(t), lse, torch.full((n,), g, device="cuda"), bias=dev(b))
    classes = t.unique()
    err = (db.cpu()[classes].double() / (-3.0 * g) - 1.0).abs()
    assert float(err.max()) <= 0.5 * unit + (3 + n) / v


def test_xent_gradient_against_differences():
    n, v, k, e = 30, 90, 20, 1e-5
    h, w, b, t, c = rand(1, n, k), rand(2, v, k, std=0.3), rand(3, v), targets(4, n, v), rand(5, n)
    _, lse = prims.softmax_xent(dev(h), dev(w), dev(t), bias=dev(b))
    grads = prims.softmax_xent_grad(dev(h), dev(w), dev(t), lse, dev(c), bias=dev(b))
    kept = t != IGNORE
    for i, (x, g) in enumerate(zip((h, w, b), grads)):
        u = rand(9 + i, *x.shape).double()

        def value(s):
            a = [q.double() + (s * u if j == i else 0) for j, q in enumerate((h, w, b))]
            z = a[0] @ a[1].t() + a[2]
            rows = torch.logsumexp(z, 1) - z.gather(1, torch.where(kept, t, 0)[:, None])[:, 0]
            return float((c.double() * rows)[kept].sum())

        slope = (value(e) - value(-e)) / (2 * e)
        got = float((g.cpu().double() * u).sum())
        room = 4e-6 * float((g.cpu().double() * u).abs().sum()) + 1e-5
        assert abs(got - slope) <= room, (i, got, slope)


@pytest.mark.parametrize("dtype", TYPES)
def test_the_same_call_gives_the_same_bits_on_any_stream(dtype):
    n, v, k = 300, 700, 65
    h, w, t = dev(rand(1, n, k, dtype=dtype)), dev(rand(2, v, k, dtype=dtype)), dev(targets(3, n, v))
    g = torch.full((n,), 1.0 / n, device="cuda")

    def both():
        loss, lse = prims.softmax_xent(h, w, t)
        dh, dw, _ = prims.softmax_xent_grad(h, w, t, lse, g)
        y, z = prims.linear(h, w, activation="gelu", keep_preact=True)
        return [loss, lse, dh, dw, y, z] + list(prims.linear_grad(z, h, w, preact=y, activation="gelu"))

    first = both()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = both()
    third = both()  # its scratch is the other stream's too: the calls are ordered
    torch.cuda.synchronize()
    for a, b, c in zip(first, again, third):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_calls_alternate_between_streams():
    """Calls on the null stream and on another one, in turn and without waiting,
    share a workspace: each starts after the one before."""
    n, v, k = 2048, 30011, 256
    hs, w = [dev(rand(1 + i, n, k, dtype=BF16)) for i in range(8)], dev(rand(20, v, k, dtype=BF16, std=0.2))
    t = dev(targets(3, n, v))
    want = []
    for h in hs:
        want.append(prims.softmax_xent(h, w, t))
        torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = []
    for i, h in enumerate(hs):
        with torch.cuda.stream(side if i % 2 else torch.cuda.default_stream()):
            got.append(prims.softmax_xent(h, w, t))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# f32 products large enough to run in three bf16 parts: whole and ragged sizes,
# parts of the contraction (the gradients), rows aligned to four bytes alone
@pytest.mark.parametrize("n,k,m,offset", [(4100, 1040, 4096, 0), (4100, 1031, 4100, 0), (4099, 1040, 4101, 1)])
def test_large_f32_layers(n, k, m, offset):
    check_linear(n, k, m, F32, "gelu", offset=offset, seed=n + k)


@pytest.mark.parametrize("n,k,m,offset", [(2600, 2048, 2496, 0), (2050, 1031, 2101, 0), (2051, 1040, 2100, 1)])
def test_large_f32_layer_gradients(n, k, m, offset):
    check_grad(n, k, m, F32, "silu", offset=offset, seed=n + k)
    check_grad(n, k, m, F32, "none", offset=offset, seed=n + k, bias=False)


@pytest.mark.parametrize("n,v,k,offset", [(2048, 3080, 1024, 0), (2051, 3001, 1031, 1)])
def test_large_f32_losses(n, v, k, offset):
    check_xent(n, v, k, F32, offset=offset, seed=v)
    check_xent(n, v, k, F32, offset=offset, seed=v, bias=False)


def test_large_f32_products_keep_every_scale():
    """Columns of very different size, whose weights make up for it: each term
    has f32's relative accuracy, whatever the others of its row are."""
    n, k, m = 4100, 1040, 4100
    x, w = rand(1, n, k), rand(2, m, k)
    size = 10.0 ** torch.linspace(-18, 18, k)
    x, w = x * size, w / size
    got = prims.linear(dev(x), dev(w))
    ref.assert_near(got, ref.linear(x, w, None, "none", None)[0], "scaled columns")


def test_large_f32_infinities_and_nan():
    """Elements that have no bf16 parts: infinities, NaN, and floats that round
    to an infinity in bf16, in either operand, give what f32 arithmetic gives."""
    n, k, m = 4100, 1040, 4100
    x, w = rand(1, n, k), rand(2, m, k, std=0.03)
    big = torch.finfo(F32).max
    for where in ("x", "w"):
        xs, ws = x.clone(), w.clone()
        a = xs if where == "x" else ws
        a[5, 3], a[6, 4], a[7, 8] = float("inf"), float("nan"), big
        got = prims.linear(dev(xs), dev(ws))
        lines = got if where == "x" else got.t()
        other = ws if where == "x" else xs
        assert torch.equal(lines[5].cpu(), torch.where(other[:, 3] > 0, float("inf"), float("-inf")))
        assert lines[6].isnan().all()
        keep = [i for i in range(4100) if i not in (5, 6, 7)]
        y, off = ref.linear(x, w, None, "none", None)[0]
        y, off = (y, off) if where == "x" else (y.t(), off.t())
        ref.assert_near(lines[keep], (y[keep], off[keep]), "rows beside them")
        one = big * other[:, 8].double()
        rest = (ref.U32 * 4 * one.abs() + 1e30)
        fits = one.abs() < big * 0.99
        assert bool(((lines[7].cpu().double() - one).abs() <= rest)[fits].all())
    dy = rand(3, 2600, 2496)
    x, w = rand(4, 2600, 2048), rand(5, 2496, 2048, std=0.03)
    clean = prims.linear_grad(dev(dy), dev(x), dev(w))
    x[9, 2] = float("inf")  # a column of dw; dx does not read x
    dx, dw, db = prims.linear_grad(dev(dy), dev(x), dev(w))
    assert torch.equal(db, clean[2])
    assert (dx - clean[0]).abs().max() <= 1e-5 * clean[0].abs().max()
    assert torch.equal(dw[:, 2].cpu(), torch.where(dy[9] > 0, float("inf"), float("-inf")))
    keep = [i for i in range(2048) if i != 2]
    assert (dw[:, keep] - clean[1][:, keep]).abs().max() <= 1e-5 * clean[1].abs().max()


def test_large_f32_loss_of_a_row_with_nan():
    n, v, k = 2051, 3001, 1031
    h, w, t = rand(1, n, k), dev(rand(2, v, k, std=0.05)), dev(targets(3, n, v, 0.0))
    g = torch.full((n,), 1.0 / n, device="cuda")
    loss, lse = prims.softmax_xent(dev(h), w, t)
    dh, _, _ = prims.softmax_xent_grad(dev(h), w, t, lse, g)
    h[17, 4] = float("nan")
    loss2, lse2 = prims.softmax_xent(dev(h), w, t)
    dh2, dw2, _ = prims.softmax_xent_grad(dev(h), w, t, lse2, g)
    keep = [i for i in range(n) if i != 17]
    assert loss2[17].isnan() and dh2[17].isnan().all() and dw2.isnan().all()
    assert (loss2 - loss)[keep].abs().max() <= 1e-5 * loss.abs().max()
    assert (dh2 - dh)[keep].abs().max() <= 1e-5 * dh.abs().max()


# ---- the optimizer ----

SIZES = [1, 3, 255, 256, 257, 1000, 4096, 4097, 10007]


def opt_inputs(sizes, seed, grad_dtype=F32, std=0.01):
    out = []
    for i, n in enumerate(sizes):
        s = seed + 10 * i
        out.append((rand(s, n, std=0.1), rand(s + 1, n, std=std).to(grad_dtype), rand(s + 2, n, std=std / 3),
                    rand(s + 3, n, std=std).square()))
    return out


HY = dict(step=7, lr=3e-3, betas=(0.9, 0.995), eps=1e-7)


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("grad_dtype", TYPES)
def test_adamw_32_bits(grad_dtype, offset):
    data = opt_inputs(SIZES, 1, grad_dtype)
    ps, gs, ms, vs = ([dev(d[i], offset) for d in data] for i in range(4))
    decays = [0.1 * (i % 3) for i in range(len(SIZES))]
    scale = torch.full((1,), 0.5, device="cuda")
    prims.adamw_step(ps, gs, ms, vs, weight_decay=decays, scale=scale, **HY)
    for i, (p, g, m, v) in enumerate(data):
        want = ref.adamw(p, g.double(), m, v, HY["step"], HY["lr"], HY["betas"], HY["eps"], decays[i], 0.5)
        size = [np.abs(p.numpy()) + HY["lr"] * 4, np.abs(m.numpy()) + np.abs(g.double().numpy()),
                np.abs(v.numpy()) + np.abs(g.double().numpy()) ** 2]
        for got, w, s, name in zip((ps[i], ms[i], vs[i]), want, size, "pmv"):
            # about eight roundings, each of at most half a unit of the larger term
            assert np.all(np.abs(got.cpu().numpy() - w) <= 16 * ref.U32 * s), (i, name)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_adamw_masters(dtype):
    data = opt_inputs(SIZES, 2, dtype)
    masters = [dev(d[0]) for d in data]
    ps = [m.to(dtype) for m in masters]
    gs, ms, vs = ([dev(d[i]) for d in data] for i in (1, 2, 3))
    plain = [t.clone() for t in masters]
    pm, pv = [t.clone() for t in ms], [t.clone() for t in vs]
    prims.adamw_step(plain, gs, pm, pv, **HY)
    prims.adamw_step(ps, gs, ms, vs, masters=masters, **HY)
    for a, b in zip(plain + pm + pv, masters + ms + vs):
        assert torch.equal(a, b)
    for p, m in zip(ps, masters):
        assert torch.equal(p, m.to(dtype))


def test_adamw_more_tensors_than_a_launch():
    sizes = [(7 * i) % 300 for i in range(130)] + [5000]  # empty ones among them
    data = opt_inputs(sizes, 3)
    ps, gs, ms, vs = ([dev(d[i]) for d in data] for i in range(4))
    prims.adamw_step(ps, gs, ms, vs, **HY)
    one = [[dev(d[i]) for d in data] for i in range(4)]
    for p, g, m, v in zip(*one):
        prims.adamw_step([p], [g], [m], [v], **HY)
    for got, want in zip((ps, ms, vs), (one[0], one[2], one[3])):
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def opt8_inputs(sizes, seed):
    r = np.random.default_rng(seed)
    out = []
    for n in sizes:
        blocks = -(-n // 256)
        out.append([r.normal(0, 0.1, n).astype(np.float32), r.normal(0, 0.01, n).astype(np.float32),
                    r.integers(0, 256, n).astype(np.uint8), r.integers(0, 256, n).astype(np.uint8),
                    r.uniform(0.001, 0.01, blocks).astype(np.float32), r.uniform(0.001, 0.02, blocks).astype(np.float32)])
    return out


@pytest.mark.parametrize("offset", [0, 1])
def test_adamw_8_bits_follows_its_definition(offset):
    """Three steps, codes and scales bit for bit, from states of every code and
    from the zero state, with blocks whose gradient is zero."""
    data = opt8_inputs(SIZES, 5)
    data.append([t.copy() * (0 if i >= 2 else 1) for i, t in enumerate(opt8_inputs([3000], 6)[0])])
    data[-1][1][256:512] = 0.0
    dt = [[dev(torch.from_numpy(d[i].copy()), offset) for d in data] for i in range(6)]
    decays = [0.0 if i % 2 else 0.05 for i in range(len(data))]
    scale = torch.full((1,), 0.8, device="cuda")
    for step in (1, 2, 3):
        prims.adamw_step(dt[0], dt[1], dt[2], dt[3], step=step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
                         weight_decay=decays, avg_scales=dt[4], avg_sq_scales=dt[5], scale=scale, seed=1000 + step)
        for i, d in enumerate(data):
            d[0], d[2], d[3], d[4], d[5] = ref.adamw8(*[d[j] for j in (0, 1, 2, 3, 4, 5)], i, step, 1e-3,
                                                      (0.9, 0.999), 1e-8, decays[i], 1000 + step, np.float32(0.8))
            for j, name in ((4, "scale m"), (5, "scale root"), (2, "codes m"), (3, "codes root"), (0, "p")):
                got = dt[j][i].cpu().numpy()
                assert np.array_equal(got, d[j]), (step, i, name, int((got != d[j]).sum()), len(got))
    for i, d in enumerate(data):
        m = prims.adamw_state_values(dt[2][i], dt[4][i], "exp_avg").cpu().numpy()
        r = prims.adamw_state_values(dt[3][i], dt[5][i], "exp_avg_sq").cpu().numpy()
        n = len(d[0])
        vm = ref.code_values(d[2] & 127, 3)
        assert np.array_equal(m, np.where(d[2] > 127, -vm, vm) * np.repeat(d[4], 256)[:n])
        assert np.array_equal(r, ref.code_values(d[3], 4) * np.repeat(d[5], 256)[:n])


def test_adamw_8_bits_past_32_bits():
    """A tensor of 2^32 + 5000 elements: its last blocks, whose elements' numbers
    have a thirty-third bit."""
    n, tail = 2 ** 32 + 5000, 5000 + 512
    first = n - tail
    first -= first % 256
    d = opt8_inputs([n - first], 11)[0]
    t = [torch.zeros(n, device="cuda"), torch.zeros(n, dtype=BF16, device="cuda"),
         torch.zeros(n, dtype=torch.uint8, device="cuda"), torch.zeros(n, dtype=torch.uint8, device="cuda"),
         torch.zeros(-(-n // 256), device="cuda"), torch.zeros(-(-n // 256), device="cuda")]
    for i, x in enumerate(d):
        t[i][-len(x):] = dev(torch.from_numpy(x))
    g = t[1][first:].float().cpu().numpy()
    prims.adamw_step([t[0]], [t[1]], [t[2]], [t[3]], step=4, lr=1e-3, avg_scales=[t[4]], avg_sq_scales=[t[5]],
                     weight_decay=0.1, seed=3)
    want = ref.adamw8(d[0], g, *d[2:], 0, 4, 1e-3, (0.9, 0.999), 1e-8, 0.1, 3, first=first)
    for i, w in zip((0, 2, 3, 4, 5), want):
        assert np.array_equal(t[i][-len(w):].cpu().numpy(), w)
    assert not t[2][:first].any() and not t[0][:first].any()


def test_adamw_8_bits_half_parameters():
    d = opt8_inputs([5000], 8)[0]
    t = [dev(torch.from_numpy(x.copy())) for x in d]
    g = t[1].to(BF16)
    param = t[0].to(BF16)
    prims.adamw_step([param], [g], [t[2]], [t[3]], step=4, lr=1e-3, masters=[t[0]], avg_scales=[t[4]],
                     avg_sq_scales=[t[5]], weight_decay=0.1, seed=3)
    want = ref.adamw8(d[0], g.float().cpu().numpy(), d[2], d[3], d[4], d[5], 0, 4, 1e-3, (0.9, 0.999), 1e-8, 0.1, 3)
    assert np.array_equal(t[0].cpu().numpy(), want[0]) and np.array_equal(t[2].cpu().numpy(), want[1])
    assert torch.equal(param, t[0].to(BF16))


def test_adamw_8_bits_moves_on_average():
    """A constant gradient: the second moment's root must approach it although a
    step is far below half a code, as rounding up by chance lets it."""
    n = 1 << 16
    g = torch.full((n,), 0.01, device="cuda")
    p, m, r = torch.zeros(n, device="cuda"), *(torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2))
    ms, rs = (torch.zeros(n // 256, device="cuda") for _ in range(2))
    m[0::256] = 0
    # one element of each block has a gradient ten times as large, so that the
    # others' codes are not the block's largest
    g[0::256] = 0.1
    for step in range(1, 201):
        prims.adamw_step([p], [g], [m], [r], step=step, lr=0.0, betas=(0.9, 0.98), avg_scales=[ms],
                         avg_sq_scales=[rs], seed=step * 7919)
    root = prims.adamw_state_values(r, rs, "exp_avg_sq")
    avg = prims.adamw_state_values(m, ms, "exp_avg")
    small = torch.ones(n, dtype=torch.bool, device="cuda")
    small[0::256] = False
    want = 0.01 * (1 - 0.98 ** 200) ** 0.5
    # a code is up to 2^-4 of its value; over 65,000 elements the mean of the
    # random roundings is within a hundredth of that, and squaring a rounded
    # root adds its variance, under 2^-9, fifty times over: 2^-4 in all
    assert abs(float(root[small].mean()) / want - 1) < 2.0 ** -4
    assert abs(float(avg[small].mean()) / 0.01 - 1) < 2.0 ** -6


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("factor", [float("nan"), float("inf")])
def test_adamw_takes_no_step_with_a_factor_that_is_not_finite(bits, factor):
    d = opt8_inputs([3000], 9)[0]
    t = [dev(torch.from_numpy(x.copy())) for x in d]
    if bits == 32:
        t[2], t[3] = t[2].float(), t[3].float()
    before = [x.clone() for x in t]
    more = dict(avg_scales=[t[4]], avg_sq_scales=[t[5]]) if bits == 8 else {}
    prims.adamw_step([t[0]], [t[1]], [t[2]], [t[3]], step=2, lr=0.1, scale=torch.full((1,), factor, device="cuda"),
                     **more)
    for a, b in zip(t, before):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [0, 1])
def test_clip_scale(dtype, offset):
    sizes = SIZES + [(11 * i) % 500 for i in range(60)] + [300000]
    gs = [rand(i, n, dtype=dtype) for i, n in enumerate(sizes)]
    square = sum(float(g.double().square().sum()) for g in gs)
    for max_norm in (1.0, 1e6):
        norm, scale = prims.clip_scale([dev(g, offset) for g in gs], max_norm)
        assert abs(float(norm) / square ** 0.5 - 1) <= 16 * ref.U32
        want = min(1.0, max_norm / square ** 0.5)
        assert abs(float(scale) / want - 1) <= 16 * ref.U32


def test_clip_scale_of_more_gradients_than_a_launch():
    gs = [rand(i, (13 * i) % 300, dtype=TYPES[i % 3]) for i in range(600)]
    square = sum(float(g.double().square().sum()) for g in gs)
    norm, _ = prims.clip_scale([dev(g) for g in gs], 1.0)
    assert abs(float(norm) / square ** 0.5 - 1) <= 16 * ref.U32


def test_clip_scale_of_nothing_and_of_infinities():
    norm, scale = prims.clip_scale([torch.empty(0, device="cuda"), torch.zeros(5, device="cuda")], 1.0)
    assert float(norm) == 0.0 and float(scale) == 1.0
    for bad in (float("inf"), float("nan")):
        g = torch.ones(5000, device="cuda")
        g[4321] = bad
        norm, scale = prims.clip_scale([torch.ones(3, device="cuda"), g], 1.0)
        assert not norm.isfinite().any() and scale.isnan().all()


@pytest.mark.parametrize("dtype,size", [(F32, 1e20), (F32, 1e-25), (F32, 3e38), (BF16, 1e20), (BF16, 1e-25), (F16, 6e4)])
def test_clip_scale_of_gradients_whose_squares_f32_cannot_hold(dtype, size):
    gs = [(rand(i, n).clamp(-1, 1) * 0.01 * size).to(dtype) for i, n in enumerate((5000, 3))]
    gs[0][77] = size
    want = sum(float(g.double().square().sum()) for g in gs) ** 0.5
    norm, scale = prims.clip_scale([dev(g) for g in gs], size / 2)
    assert abs(float(norm) / want - 1) <= 16 * ref.U32
    assert abs(float(scale) / (size / 2 / want) - 1) <= 16 * ref.U32


def test_clip_scale_of_a_norm_that_f32_cannot_hold():
    norm, scale = prims.clip_scale([torch.full((100,), 3e38, device="cuda")], 1.0)
    assert float(norm) == float("inf") and scale.isnan().all()


def test_clip_scale_of_more_elements_than_a_launch_has_threads_for():
    """Many large gradients, and one by itself."""
    g = torch.ones(2 ** 32, dtype=F16, device="cuda")
    norm, _ = prims.clip_scale([g] * 17, 1.0)
    assert abs(float(norm) / (17 * 2.0 ** 32) ** 0.5 - 1) <= 16 * ref.U32
    del g
    torch.cuda.empty_cache()
    g = torch.zeros(2 ** 36 + 5000, dtype=F16, device="cuda")
    g[::2 ** 27] = 2.0
    g[-1] = 3.0
    norm, scale = prims.clip_scale([g], 1.0)
    want = (4.0 * 513 + 9.0) ** 0.5
    assert abs(float(norm) / want - 1) <= 16 * ref.U32 and abs(float(scale) * want - 1) <= 16 * ref.U32
    del g
    torch.cuda.empty_cache()
