"""The layer in 8-bit floating point on the GPU against its formulas in 64 bits."""
import pytest
import torch

import layer_reference as layer
import train_reference as ref
from mlrs_amd import _lib, prims
from test_gpu_layer import ACTS, BF16, F16, F32, TYPES, dev, rand

pytestmark = pytest.mark.gpu


def values(codes, scales, rows, k):
    """What codes and scales stand for, float64 (rows, k)."""
    v = codes.cpu().double()[:, :k]
    up = torch.ldexp(torch.ones(scales.shape, dtype=torch.float64), scales.cpu().to(torch.int32) - 127)
    return v * up.repeat_interleave(128, 0)[:rows].repeat_interleave(128, 1)[:, :k]


def check_codes(w):
    m, k = w.shape
    w8 = prims.fp8_weight(dev(w), backward=True)
    for codes, scales, v in ((w8.codes, w8.scales, w.double()), (w8.codes_t, w8.scales_t, w.double().t().contiguous())):
        rows, cols = v.shape
        val, q, e = layer.fp8_blocks(v, 128)
        assert codes.shape == (rows, -(-cols // 128) * 128) and scales.shape == (-(-rows // 128), -(-cols // 512) * 4)
        got, want = codes.cpu().double(), torch.nan_to_num(q, nan=1e9)
        assert torch.equal(torch.nan_to_num(got, nan=1e9), want)
        assert torch.equal(scales.cpu()[:, :e.shape[1]].to(torch.int32), (e + 127).to(torch.int32))
        assert (scales.cpu()[:, e.shape[1]:] == 127).all()
    assert prims.fp8_weight(dev(w)).codes_t is None
    return w8


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (5, 7), (128, 128), (129, 127), (16, 640), (300, 513), (257, 1030)])
def test_codes_of_weights(dtype, m, k):
    size = 10.0 ** torch.linspace(-3, 3, k)
    check_codes((rand(m + k, m, k) * size).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_codes_of_every_value(dtype):
    """Every code and the borders between two: at and beside them, in a block whose
    largest magnitude is 448; and blocks of zeros, of the smallest and the largest
    magnitudes, with infinities and NaN."""
    q = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (q[1:] + q[:-1]) / 2
    near = torch.cat([q, mid, mid * (1 - 2.0 ** -7), mid * (1 + 2.0 ** -7)])
    w = torch.zeros(256, 512, dtype=torch.float64)
    w[0, :near.numel() // 4] = near[:near.numel() // 4]
    for i in range(4):
        w[i, :near.numel() // 4 + 1] = near[i * (near.numel() // 4):][:near.numel() // 4 + 1]
    w[:8, 127] = w[:8, 126 + 128] = 448.0
    w[5] = -w[1]
    w[130, 3] = torch.finfo(dtype).smallest_normal / 4
    w[131, 200] = torch.finfo(dtype).max
    w[132, 201] = torch.finfo(dtype).max * 2.0 ** -9
    w[133, 300], w[134, 301], w[135, 302] = float("inf"), float("-inf"), 3.0
    w[136, 400], w[137, 401] = float("nan"), -5.0
    check_codes(w.to(dtype))


@pytest.mark.parametrize("top", [448.0, 449.0, 447.0, 1.75, 1.76, 2.0 ** -120, 2.0 ** -140, 3e38, 0.0])
def test_scales_of_the_largest_magnitude(top):
    w = torch.zeros(3, 5, dtype=F32)
    w[1, 2] = -top
    w[2, 2] = top / 3
    check_codes(w)


def check_linear(n, k, m, dtype, act, bias=True, residual=True, keep=True, offset=0, seed=0):
    x, w = rand(seed, n, k, dtype=dtype), rand(seed + 1, m, k, dtype=dtype, std=k ** -0.5)
    b = rand(seed + 2, m, dtype=dtype, std=0.3) if bias else None
    res = rand(seed + 3, n, m, dtype=dtype) if residual else None
    got = prims.linear_fp8(dev(x, offset), prims.fp8_weight(dev(w, offset)), bias=dev(b, offset), activation=act,
                           residual=dev(res, offset), keep_preact=keep)
    y, z = got if keep else (got, None)
    want_y, want_z = layer.linear_fp8(x, w, b, act, res)
    what = "linear_fp8 n=%d k=%d m=%d %s %s" % (n, k, m, dtype, act)
    ref.assert_near(y, want_y, what + " y")
    if keep:
        ref.assert_near(z, want_z, what + " z")


def check_grad(n, k, m, dtype, act, offset=0, seed=0, **need):
    x, w = rand(seed, n, k, dtype=dtype), rand(seed + 1, m, k, dtype=dtype, std=k ** -0.5)
    dy, z = rand(seed + 2, n, m, dtype=dtype), rand(seed + 3, n, m, dtype=dtype)
    w8 = prims.fp8_weight(dev(w, offset), backward=True)
    got = prims.linear_fp8_grad(dev(dy, offset), dev(x, offset), w8, preact=dev(z, offset), activation=act, **need)
    for name, t, want in zip(("dx", "dw", "db"), got, layer.linear_fp8_grad(dy, x, w, z, act)):
        if t is not None:
            ref.assert_near(t, want, "%s n=%d k=%d m=%d %s %s" % (name, n, k, m, dtype, act))
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("n", [3, 70])
def test_linear_activations(dtype, act, n):
    check_linear(n, 192, 80, dtype, act)


# one row and few rows; one column, one output; sizes around the widths of a block,
# a word of scales, a wave and a tile; none a multiple of the next
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,m", [
    (1, 1, 1), (1, 128, 16), (1, 1000, 33), (3, 17, 5), (15, 127, 31), (16, 2048, 130), (17, 129, 33), (32, 640, 300),
    (33, 130, 47), (63, 40, 100), (64, 512, 64), (65, 1, 65), (66, 513, 64), (127, 100, 129), (128, 256, 128),
    (129, 385, 257), (257, 257, 130), (300, 1100, 520), (1000, 33, 7),
])
def test_linear_sizes(dtype, n, k, m):
    check_linear(n, k, m, dtype, "gelu", seed=n + k + m)


# the rows from which weights of this size go in tiles, and the last before them
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [8, 16, 17, 31])
def test_linear_few_rows_of_large_weights(dtype, n):
    check_linear(n, 2100, 4100, dtype, "silu", seed=n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias,residual,keep", [(False, False, False), (True, False, True), (False, True, False)])
@pytest.mark.parametrize("n", [9, 130])
def test_linear_options(dtype, bias, residual, keep, n):
    check_linear(n, 72, 136, dtype, "silu", bias, residual, keep)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,m", [(7, 64, 40), (100, 128, 64), (131, 165, 67)])
@pytest.mark.parametrize("offset", [1, 3])
def test_linear_unaligned(dtype, n, k, m, offset):
    check_linear(n, k, m, dtype, "relu", offset=offset)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_every_tile(dtype):
    """Sizes that the rule gives the largest tile, the middle one, and parts of a
    long contraction."""
    check_linear(2100, 1100, 2100, dtype, "gelu_tanh", seed=3)
    check_linear(1100, 700, 1030, dtype, "none", seed=4)
    check_linear(130, 8200, 130, dtype, "silu", seed=5)


@pytest.mark.parametrize("n", [8, 150])
def test_scales_of_every_block_count(n):
    """Columns of very different size, whose weights make up for it."""
    k, m = 1500, 200
    x, w = rand(1, n, k), rand(2, m, k)
    size = 10.0 ** torch.linspace(-15, 15, k)
    x, w = x * size, w / size
    got = prims.linear_fp8(dev(x), prims.fp8_weight(dev(w)))
    ref.assert_near(got, layer.linear_fp8(x, w, None, "none", None)[0], "scaled columns")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [4, 100])
def test_linear_nan_stays_in_its_row(dtype, n):
    x, w = rand(5, n, 200, dtype=dtype), rand(6, 150, 200, dtype=dtype, std=0.1)
    w8 = prims.fp8_weight(dev(w))
    clean = prims.linear_fp8(dev(x), w8)
    x[1, 3], x[2, 150] = float("inf"), float("nan")
    got = prims.linear_fp8(dev(x), w8)
    keep = [i for i in range(n) if i not in (1, 2)]
    assert torch.equal(got[keep], clean[keep]) and got[[1, 2]].isnan().all()
    w[7, 9], w[140, 199] = float("-inf"), float("nan")
    got = prims.linear_fp8(dev(x), prims.fp8_weight(dev(w)))
    cols = [j for j in range(150) if j not in (7, 140)]
    assert torch.equal(got[keep][:, cols], clean[keep][:, cols]) and got[:, [7, 140]].isnan().all()


def test_linear_no_rows_and_in_place():
    w8 = prims.fp8_weight(dev(rand(1, 24, 16)), backward=True)
    none = torch.empty(0, 16, device="cuda")
    assert prims.linear_fp8(none, w8).shape == (0, 24)
    dx, dw, db = prims.linear_fp8_grad(torch.empty(0, 24, device="cuda"), none, w8)
    assert dx.shape == (0, 16) and dw.shape == (24, 16) and not dw.any() and not db.any()
    for n in (20, 90):
        x, res = rand(2, n, 16), rand(3, n, 24)
        r = dev(res)
        y = prims.linear_fp8(dev(x), w8, residual=r, out=r)
        assert y is r
        ref.assert_near(y, layer.linear_fp8(x, rand(1, 24, 16), None, "none", res)[0], "residual's buffer")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_grad_activations(dtype, act):
    check_grad(150, 192, 140, dtype, act)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,m", [
    (1, 1, 1), (1, 200, 33), (3, 17, 5), (16, 64, 32), (33, 129, 47), (127, 128, 129), (128, 256, 128), (129, 31, 257),
    (300, 72, 520), (1000, 33, 7), (513, 513, 100), (2100, 300, 260),
])
def test_grad_sizes(dtype, n, k, m):
    check_grad(n, k, m, dtype, "gelu", seed=n + k + m)


@pytest.mark.parametrize("dtype", TYPES)
def test_grad_every_tile(dtype):
    check_grad(2100, 1100, 2100, dtype, "silu", seed=3)
    check_grad(8200, 130, 140, dtype, "none", seed=4)
    check_grad(140, 150, 8200, dtype, "relu", seed=5)


@pytest.mark.parametrize("dtype", TYPES)
def test_grad_parts_and_alignment(dtype):
    whole = check_grad(200, 130, 140, dtype, "gelu")
    for i, kw in enumerate((dict(bias=False, need_dw=False), dict(bias=False, need_dx=False),
                            dict(need_dx=False, need_dw=False))):
        got = check_grad(200, 130, 140, dtype, "gelu", **kw)
        for j in range(3):
            assert got[j] is None if j != i else torch.equal(got[j], whole[j])
    check_grad(200, 130, 140, dtype, "gelu", offset=1)


def test_gradient_is_a_derivative():
    """With every operand a value that 8 bits hold, the layer is the plain one, and
    differences in x and w along values that they hold too are its slope."""
    n, k, m = 40, 130, 50
    x, w, dy = ((torch.randint(-3, 4, s, generator=torch.Generator().manual_seed(i)).to(F32)) for i, s in
                enumerate(((n, k), (m, k), (n, m))))
    w8 = prims.fp8_weight(dev(w), backward=True)
    dx, dw, db = prims.linear_fp8_grad(dev(dy), dev(x), w8)
    assert torch.equal(prims.linear_fp8(dev(x), w8).cpu(), x @ w.t())
    for i in (0, 11):
        up, down = x.clone(), x.clone()
        up[i % n, 5 * i] += 1
        down[i % n, 5 * i] -= 1
        value = [(prims.linear_fp8(dev(t), w8) * dev(dy)).sum() for t in (up, down)]
        assert float(value[0] - value[1]) / 2 == float(dx[i % n, 5 * i])
        up, down = w.clone(), w.clone()
        up[i, 7 * i] += 1
        down[i, 7 * i] -= 1
        value = [(prims.linear_fp8(dev(x), prims.fp8_weight(dev(t))) * dev(dy)).sum() for t in (up, down)]
        assert float(value[0] - value[1]) / 2 == float(dw[i, 7 * i])
    assert torch.equal(db.cpu(), dy.sum(0))


def test_refusals():
    x, w = torch.zeros(40, 64, device="cuda"), torch.zeros(48, 64, device="cuda")
    w8 = prims.fp8_weight(w)
    full = prims.fp8_weight(w, backward=True)
    dy = torch.zeros(40, 48, device="cuda")
    flat = torch.zeros(48 * 128 + 8, dtype=torch.uint8, device="cuda")
    off = flat[8:].view(torch.float8_e4m3fn).view(48, 128)
    for call in (lambda: prims.fp8_weight(w[0]), lambda: prims.fp8_weight(w.double()), lambda: prims.fp8_weight(w.t()),
                 lambda: prims.linear_fp8(x[:, :63].contiguous(), w8), lambda: prims.linear_fp8(x.double(), w8),
                 lambda: prims.linear_fp8(x, w8, bias=torch.zeros(47, device="cuda")),
                 lambda: prims.linear_fp8(x, w8, bias=torch.zeros(48, device="cuda").half()),
                 lambda: prims.linear_fp8(x, w8, activation="tanh"),
                 lambda: prims.linear_fp8(x, w8._replace(scales=w8.scales[:, :2].contiguous())),
                 lambda: prims.linear_fp8(x, w8._replace(codes=w8.codes[:, :64].contiguous())),
                 lambda: prims.linear_fp8(x, w8._replace(codes=w8.codes.view(torch.uint8))),
                 lambda: prims.linear_fp8(x, w8._replace(codes=off)),
                 lambda: prims.linear_fp8_grad(dy, x, w8), lambda: prims.linear_fp8_grad(dy, x, full, activation="relu"),
                 lambda: prims.linear_fp8_grad(dy[:, :40].contiguous(), x, full),
                 lambda: prims.linear_fp8_grad(dy.half(), x, full)):
        with pytest.raises((ValueError, TypeError)):
            call()
    with pytest.raises(_lib.InvalidParam, match="overlaps"):
        prims.linear_fp8(x, prims.fp8_weight(torch.zeros(64, 64, device="cuda")), out=x)


def test_same_bits_on_any_stream_and_in_graphs():
    n, k, m = 300, 700, 260
    x, w, dy = dev(rand(1, n, k, dtype=BF16)), dev(rand(2, m, k, dtype=BF16)), dev(rand(3, n, m, dtype=BF16))

    def all_of_it():
        w8 = prims.fp8_weight(w, backward=True)
        y, z = prims.linear_fp8(x, w8, activation="gelu", keep_preact=True)
        return [y, z] + list(prims.linear_fp8_grad(dy, x, w8, preact=z, activation="gelu"))

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
    # a few rows take no workspace: an online encoder's call in a graph
    row = x[:5].contiguous()
    w8 = prims.fp8_weight(w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = prims.linear_fp8(row, w8, activation="silu")
        with pytest.raises(NotImplementedError, match="cannot be captured"):
            prims.linear_fp8(x, w8)
    for i in range(3):
        row.copy_(x[5 * i:5 * i + 5])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, prims.linear_fp8(row, w8, activation="silu"))
