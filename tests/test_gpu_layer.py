"""Dropout and group norm on the GPU against their formulas in 64 bits."""
import numpy as np
import pytest
import torch

import layer_reference as layer
import train_reference as ref
from mlrs_amd import _lib, prims

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def rand(seed, *shape, dtype=F32, std=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * std + mean).to(dtype)


def dev(t, offset=0):
    """On the GPU; with `offset` elements before it, so that it is aligned to its
    element size alone."""
    if t is None or not offset:
        return None if t is None else t.cuda()
    flat = torch.empty(t.numel() + offset, dtype=t.dtype, device="cuda")
    view = flat[offset:].view(t.shape)
    view.copy_(t)
    return view


# ---- dropout ----

def want_dropout(x, p, seed, offset, residual):
    """Dropped elements are 0 whatever they hold."""
    by = layer.factor(tuple(x.shape), p, seed, offset)
    y = torch.where(by > 0, x.double() * by, torch.zeros_like(by))
    off = 2 * ref.U32 * y.abs()  # the factor's rounding and the product's
    if residual is not None:
        y = y + residual.double()
        off = off + ref.U32 * y.abs()
    return y, off


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 255, 2048, 2049, 4099, 1000003])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout(dtype, n, residual):
    x, r = rand(n, n, dtype=dtype), rand(n + 1, n, dtype=dtype) if residual else None
    seed, offset = 0xFEDCBA9876543210, 0x123456789A
    got = prims.dropout(dev(x), 0.3, seed, offset, residual=dev(r))
    ref.assert_near(got, want_dropout(x, 0.3, seed, offset, r), "dropout")
    if n > 1:
        got = prims.dropout(dev(x, 1), 0.3, seed, offset, residual=dev(r, 3))
        ref.assert_near(got, want_dropout(x, 0.3, seed, offset, r), "dropout, unaligned")


@pytest.mark.parametrize("p", [0.0, 1e-9, 2.0 ** -17, 2.0 ** -16, 0.5, 0.999, 1 - 1e-9])
def test_dropout_probabilities(p):
    x = rand(1, 100, 333)
    ref.assert_near(prims.dropout(dev(x), p, 5), want_dropout(x, p, 5, 0, None), "p = %r" % p)


def test_dropout_masks_do_not_repeat():
    """One seed with several offsets, and several seeds: no two masks alike, and
    each keeps its share (standard deviation 0.0005 of it)."""
    x = torch.ones(1 << 20, device="cuda")
    masks = [prims.dropout(x, 0.5, seed, offset) > 0 for seed, offset in
             ((0, 0), (0, 1), (1, 0), (0, 1 << 32), (1 << 32, 0), (-1, 0))]
    for i, a in enumerate(masks):
        assert abs(float(a.float().mean()) - 0.5) < 0.004
        for b in masks[:i]:
            assert abs(float((a == b).float().mean()) - 0.5) < 0.004


@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_in_place_and_its_gradient(dtype):
    x, r = rand(1, 50, 41, dtype=dtype), rand(2, 50, 41, dtype=dtype)
    want = prims.dropout(dev(x), 0.4, 3, 4, residual=dev(r))
    a, b = dev(x), dev(r)
    assert prims.dropout(a, 0.4, 3, 4, residual=b, out=b) is b and torch.equal(b, want)
    b = dev(r)
    assert torch.equal(prims.dropout(a, 0.4, 3, 4, residual=b, out=a), want)
    ones = torch.ones_like(want)
    # the gradient of ones is the factor itself
    grad = prims.dropout(ones, 0.4, 3, 4)
    ref.assert_near(grad, (layer.factor((50, 41), 0.4, 3, 4), torch.full((50, 41), 1e-6, dtype=torch.float64)), "grad")


def test_dropout_drops_infinities():
    x = torch.full((1000,), float("inf"), device="cuda")
    x[::2] = float("nan")
    y = prims.dropout(x, 0.5, 1)
    drop = torch.from_numpy(layer.random_halves(1000, 1, 0) < 32768).cuda()
    assert (y[drop] == 0).all() and not y[~drop].isfinite().any()


def test_dropout_refusals():
    x = torch.zeros(8, 8, device="cuda")
    for kw in (dict(residual=x[:4]), dict(residual=x.half()), dict(out=x.half()), dict(offset=torch.zeros(1).cuda()),
               dict(offset=torch.zeros(2, dtype=torch.int64).cuda()), dict(p=1.0), dict(p=-0.5)):
        with pytest.raises((ValueError, TypeError)):
            prims.dropout(x, **{**dict(p=0.5, seed=0), **kw})
    both = torch.zeros(65, device="cuda")
    with pytest.raises(_lib.InvalidParam, match="overlaps"):
        prims.dropout(both[1:], 0.5, 0, out=both[:-1])
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        prims.dropout(x.double(), 0.5, 0)
    with pytest.raises(ValueError, match="contiguous"):
        prims.dropout(x.t()[:, 1:], 0.5, 0)


def test_dropout_of_nothing():
    assert prims.dropout(torch.empty(0, 5, device="cuda"), 0.5, 0).shape == (0, 5)


# ---- group norm ----

def check_norm(shape, groups, dtype, act, p=0.0, affine=True, offset=0, seed=0, mean=0.5, eps=1e-5, std=1.0):
    c = shape[-1]
    x = rand(seed, *shape, dtype=dtype, std=std, mean=mean)
    w = rand(seed + 1, c, dtype=dtype, std=0.3, mean=1.0) if affine else None
    b = rand(seed + 2, c, dtype=dtype, std=0.3) if affine else None
    dy = rand(seed + 3, *shape, dtype=dtype)
    drop = dict(p=p, seed=seed, offset=7)
    by = layer.factor(shape, p, seed, 7) if p else None
    want = layer.group_norm(x, groups, w, b, eps, act, by, dy)
    xd, wd, bd, dyd = (dev(t, offset) for t in (x, w, b, dy))
    got = dict(zip(("y", "mean", "rstd"), prims.group_norm(xd, groups, weight=wd, bias=bd, eps=eps, activation=act,
                                                           keep_stats=True, **drop)))
    assert torch.equal(got["y"], prims.group_norm(xd, groups, weight=wd, bias=bd, eps=eps, activation=act, **drop))
    got.update(zip(("dx", "dw", "db"), prims.group_norm_grad(dyd, xd, got["mean"], got["rstd"], weight=wd, bias=bd,
                                                             activation=act, **drop)))
    for name, t in got.items():
        if t is None:
            assert not affine and name in ("dw", "db")
            continue
        ref.assert_near(t, want[name], "%s of %s in %d groups, %s %s p=%g" % (name, shape, groups, dtype, act, p))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_norm_activations(dtype, act):
    check_norm((70, 96), 4, dtype, act, p=0.25)
    check_norm((5, 6, 96), 4, dtype, act, p=0.25)
    check_norm((2, 700, 96), 4, dtype, act, p=0.25)


# rows: from one lane of a group to a workgroup, groups that end inside eight
# channels, one group, more groups than a wave, many samples
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,c,groups", [
    (1, 8, 1), (1, 4, 2), (5, 30, 5), (3, 1000, 1), (7, 2000, 1), (6, 2500, 1), (4, 4100, 1), (2, 8192, 1),
    (3, 16384, 2), (1000, 64, 8), (333, 14, 7), (17, 130, 13), (2, 1024, 128), (5000, 24, 3), (9, 520, 8),
    (300, 4104, 1), (1, 1024, 8), (6000, 39, 3), (2, 16, 2), (401, 16, 1),
])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_norm_rows(dtype, n, c, groups, p):
    check_norm((n, c), groups, dtype, "silu", p=p, seed=n + c)


# slabs that a workgroup holds: few and many positions, slabs of one and of several
# groups, a last slab of fewer, groups that end inside eight channels
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,groups", [
    ((3, 2, 5), 5), ((5, 49, 250), 10), ((2, 10, 10, 64), 8), ((300, 4, 16), 4), ((2, 7, 2056), 1), ((4, 3, 1000), 8),
    ((1, 900, 40), 4), ((2, 256, 72), 9), ((1, 2, 8192), 1), ((2, 500, 6), 3), ((700, 2, 130), 13), ((2, 3, 600), 300),
])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_norm_slabs(dtype, shape, groups, p):
    check_norm(shape, groups, dtype, "gelu", p=p, seed=shape[0] + shape[-1])


# half a line of memory at many positions: as many as a thread has registers for, and
# one more; a last slab of fewer groups; as many samples as there is room for, and more
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,groups", [
    ((3, 1000, 100), 5), ((2, 1122, 40), 2), ((2, 1123, 40), 2), ((1, 1225, 64), 4), ((2, 1500, 64), 4),
    ((2, 1537, 64), 4), ((1, 700, 200), 4), ((90, 700, 120), 6), ((80, 600, 96), 6),
])
def test_norm_slabs_of_many_positions(dtype, shape, groups):
    check_norm(shape, groups, dtype, "silu", p=0.2, seed=shape[0] + shape[-1])


# few positions: a wave to a sample, slabs of many groups, more samples than workgroups
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,groups", [
    ((3000, 4, 18), 6), ((70000, 2, 8), 4), ((1300, 5, 1025), 41), ((2100, 3, 300), 300), ((600, 9, 777), 7),
    ((40, 8, 128), 16), ((40, 9, 128), 16), ((5, 64, 8), 1),
])
def test_norm_slabs_of_few_positions(dtype, shape, groups):
    check_norm(shape, groups, dtype, "gelu", p=0.2, seed=shape[0] + shape[-1])


# groups larger than a workgroup holds
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,groups", [
    ((2, 5000, 40), 8), ((1, 70001, 8), 2), ((2, 300, 2000), 1), ((1, 20, 16384), 2), ((2, 64, 64, 100), 20),
    ((1, 3001, 7), 7), ((3, 2500, 330), 33),
])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_norm_large_groups(dtype, shape, groups, p):
    check_norm(shape, groups, dtype, "silu", p=p, seed=shape[0] + shape[-1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,groups", [((9, 130), 13), ((40, 2056), 1), ((5, 9, 60), 6), ((2, 3000, 30), 6)])
def test_norm_unaligned(dtype, shape, groups):
    check_norm(shape, groups, dtype, "gelu_tanh", p=0.2, offset=1)
    check_norm(shape, groups, dtype, "none", offset=3, affine=False)


@pytest.mark.parametrize("shape,groups", [((20, 256), 2), ((4, 30, 64), 4), ((2, 4000, 64), 4)])
def test_norm_of_a_large_mean(shape, groups):
    """A mean of 1000 standard deviations: the squares are those about the mean."""
    check_norm(shape, groups, F32, "none", mean=1000.0)


@pytest.mark.parametrize("shape", [(3, 64), (3, 5, 64), (2, 4000, 64)])
def test_norm_of_equal_elements(shape):
    """No variance: y is the bias's activation, and rstd 1 / sqrt(eps)."""
    x = torch.full(shape, 3.0, device="cuda")
    b = dev(rand(1, 64))
    y, mean, rstd = prims.group_norm(x, 4, bias=b, eps=1e-4, keep_stats=True)
    assert torch.equal(mean, torch.full_like(mean, 3.0))
    assert torch.equal(y, b.expand(shape))
    assert (rstd - 100.0).abs().max() < 1e-4


@pytest.mark.parametrize("shape", [(6, 64), (6, 5, 64), (6, 2000, 64)])
def test_norm_nan_stays_in_its_group(shape):
    x = rand(1, *shape)
    dy = rand(2, *shape)
    clean = prims.group_norm(dev(x), 4, keep_stats=True)
    cdx = prims.group_norm_grad(dev(dy), dev(x), clean[1], clean[2])[0]
    x.view(6, -1, 64)[1, 0, 20] = float("nan")  # group 1 of sample 1
    x.view(6, -1, 64)[4, 0, 63] = float("inf")  # group 3 of sample 4
    y, mean, rstd = prims.group_norm(dev(x), 4, keep_stats=True)
    dx = prims.group_norm_grad(dev(dy), dev(x), mean, rstd)[0]
    for got, want in ((y, clean[0]), (dx, cdx)):
        got, want = got.view(6, -1, 4, 16), want.view(6, -1, 4, 16)
        bad = torch.zeros(6, 4, dtype=torch.bool)
        bad[1, 1] = bad[4, 3] = True
        for i in range(6):
            for j in range(4):
                if bad[i, j]:
                    assert got[i, :, j].isnan().any()
                else:
                    assert torch.equal(got[i, :, j], want[i, :, j])


@pytest.mark.parametrize("shape", [(6, 64), (6, 5, 64), (6, 2000, 64)])
def test_norm_parts_of_the_gradient(shape):
    """What is asked for does not change what comes."""
    x, dy, w, b = dev(rand(1, *shape)), dev(rand(2, *shape)), dev(rand(3, 64)), dev(rand(4, 64))
    y, mean, rstd = prims.group_norm(x, 4, weight=w, bias=b, activation="relu", keep_stats=True)
    dx, dw, db = prims.group_norm_grad(dy, x, mean, rstd, weight=w, bias=b, activation="relu")
    none, dw2, db2 = prims.group_norm_grad(dy, x, mean, rstd, weight=w, bias=b, activation="relu", need_dx=False)
    assert none is None and torch.equal(dw, dw2) and torch.equal(db, db2)


def test_norm_of_nothing():
    x, w = torch.empty(0, 5, 8, device="cuda"), torch.ones(8, device="cuda")
    y, mean, rstd = prims.group_norm(x, 2, weight=w, bias=w, keep_stats=True)
    assert y.shape == (0, 5, 8) and mean.shape == (0, 2)
    dx, dw, db = prims.group_norm_grad(x, x, mean, rstd, weight=w, bias=w)
    assert dx.shape == (0, 5, 8) and not dw.any() and not db.any()


def test_norm_refusals():
    x = torch.zeros(4, 6, 8, device="cuda")
    m = torch.zeros(4, 2, device="cuda")
    for call in (lambda: prims.group_norm(x, 3), lambda: prims.group_norm(x, 0),
                 lambda: prims.group_norm(x, 2, weight=torch.ones(4, device="cuda")),
                 lambda: prims.group_norm(x, 2, weight=torch.ones(8, device="cuda").half()),
                 lambda: prims.group_norm(x[0, 0], 2), lambda: prims.group_norm(x, 2, activation="tanh"),
                 lambda: prims.group_norm(x, 2, p=1.5), lambda: prims.group_norm(x, 2, eps=-1.0),
                 lambda: prims.group_norm(x.transpose(0, 1), 2), lambda: prims.group_norm(x.double(), 2),
                 lambda: prims.group_norm_grad(x[:2], x, m, m), lambda: prims.group_norm_grad(x, x, m[:2], m),
                 lambda: prims.group_norm_grad(x, x, m, m.half()), lambda: prims.group_norm_grad(x, x, m, m[:2])):
        with pytest.raises((ValueError, TypeError)):
            call()
    with pytest.raises(NotImplementedError):
        prims.group_norm(torch.zeros(2, 8200, device="cuda"), 1)


# ---- streams and graphs ----

def test_same_bits_on_any_stream():
    x, dy, w = dev(rand(1, 4, 3000, 64)), dev(rand(2, 4, 3000, 64)), dev(rand(3, 64))

    def all_of_it():
        y, mean, rstd = prims.group_norm(x, 8, weight=w, activation="gelu", p=0.1, seed=5, keep_stats=True)
        return [y, mean, rstd, prims.dropout(x, 0.2, 4, residual=y)] + list(
            prims.group_norm_grad(dy, x, mean, rstd, weight=w, activation="gelu", p=0.1, seed=5))[:2]

    first = all_of_it()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = all_of_it()
    third = all_of_it()
    torch.cuda.synchronize()
    for a, b, c in zip(first, again, third):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_captured_calls_replay():
    """Calls without a workspace in a graph: every replay draws the bits of the
    offset that is on the device then, between eager calls of the same kind."""
    x, w = dev(rand(1, 200, 256)), dev(rand(2, 256))
    step = torch.zeros(1, dtype=torch.int64, device="cuda")

    def work(offset):
        y = prims.group_norm(x, 4, weight=w, activation="silu", p=0.1, seed=9, offset=offset)
        return prims.dropout(y, 0.5, 9, offset=offset, residual=x)

    work(step)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work(step)
    for i in (3, 4, 5, 3):
        step.fill_(i)
        x.copy_(rand(10 + i, 200, 256))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, work(i))


def test_calls_with_a_workspace_are_not_captured():
    x = dev(rand(1, 2, 5000, 64))
    y, mean, rstd = prims.group_norm(x, 4, keep_stats=True)
    w = torch.ones(64, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = prims.dropout(x, 0.5, 1)
        with pytest.raises(NotImplementedError, match="cannot be captured"):
            prims.group_norm(x, 4)
        with pytest.raises(NotImplementedError, match="cannot be captured"):
            prims.group_norm_grad(x, x, mean, rstd, weight=w)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(z, prims.dropout(x, 0.5, 1))
    assert torch.equal(y, prims.group_norm(x, 4))
