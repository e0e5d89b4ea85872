"""The layer in 8-bit floating point rejects bad arguments before anything is
launched -- CPU only."""
import ctypes

import pytest
import torch

import layer_reference as layer
from mlrs_amd import _lib, prims
from test_layer_checks import NULL, PARAM, SHAPE, SIZE, TYPES, UNSUPPORTED, apart, failed

# 4 x 130 by 5 x 130: codes 5 x 256, scales 1 x 4; transposed 130 x 128, 2 x 4
CODES, SCALES, CODES_T, SCALES_T = 5 * 256, 4, 130 * 128, 8


def weight(s, at=None, **kw):
    w, codes, scales, codes_t, scales_t = at or apart(5)
    a = dict(w=w, w_len=650, m=5, k=130, codes=codes, codes_len=CODES, scales=scales, scales_len=SCALES,
             codes_t=codes_t, codes_t_len=CODES_T, scales_t=scales_t, scales_t_len=SCALES_T)
    a.update(kw)
    return failed(getattr(_lib.load(), "mlrs_fp8_weight_" + s)(*a.values(), None))


def linear(s, at=None, **kw):
    x, codes, scales, b, r, y, z = at or apart(7)
    a = dict(x=x, x_len=520, n=4, k=130, codes=codes, codes_len=CODES, scales=scales, scales_len=SCALES, m=5, b=b,
             b_len=5, r=r, r_len=20, act=1, y=y, y_len=20, z=z, z_len=20)
    a.update(kw)
    return failed(getattr(_lib.load(), "mlrs_linear_fp8_" + s)(*a.values(), None))


def grad(s, at=None, **kw):
    dy, x, codes_t, scales_t, z, dx, dw, db = at or apart(8)
    a = dict(dy=dy, dy_len=20, x=x, x_len=520, n=4, k=130, codes_t=codes_t, codes_t_len=CODES_T, scales_t=scales_t,
             scales_t_len=SCALES_T, m=5, z=z, z_len=20, act=1, dx=dx, dx_len=520, dw=dw, dw_len=650, db=db, db_len=5)
    a.update(kw)
    return failed(getattr(_lib.load(), "mlrs_linear_fp8_grad_" + s)(*a.values(), None))


HUGE = (1 << 22) + 1


@pytest.mark.parametrize("s", TYPES)
@pytest.mark.parametrize("kw,rc,operand", [
    (dict(w_len=651), SHAPE, "w"), (dict(m=-5), SHAPE, "w"), (dict(k=0, w_len=0), SHAPE, "features"),
    (dict(m=HUGE, k=1, w_len=HUGE), UNSUPPORTED, "features"), (dict(codes_len=650), SHAPE, "codes"),
    (dict(scales_len=2), SHAPE, "scales"), (dict(codes=0x100008), PARAM, "codes"), (dict(scales=0x100002), PARAM, "scales"),
    (dict(codes_t_len=650), SHAPE, "codes_t"), (dict(scales_t_len=4), SHAPE, "scales_t"),
    (dict(codes_t=None), NULL, "codes_t"), (dict(scales_t=None), NULL, "scales_t"), (dict(w=None), NULL, "w"),
    (dict(codes=None), NULL, "codes"), (dict(scales=None), NULL, "scales"),
])
def test_weight_validation(s, kw, rc, operand):
    assert weight(s, **kw) == (rc, operand)


@pytest.mark.parametrize("s", TYPES)
@pytest.mark.parametrize("kw,rc,operand", [
    (dict(x_len=519), SHAPE, "x"), (dict(n=-4), SHAPE, "x"), (dict(m=0), SHAPE, "features"),
    (dict(n=1 << 31, x_len=130 << 31), UNSUPPORTED, "rows"), (dict(codes_len=650), SHAPE, "codes"),
    (dict(scales_len=8), SHAPE, "scales"), (dict(codes=0x100001), PARAM, "codes"), (dict(scales=0x100001), PARAM, "scales"),
    (dict(b_len=4), SHAPE, "bias"), (dict(b=None), SHAPE, "bias"), (dict(r_len=19), SHAPE, "residual"),
    (dict(y_len=21), SHAPE, "out"), (dict(z_len=19), SHAPE, "preact"), (dict(z=None), SHAPE, "preact"),
    (dict(act=7), UNSUPPORTED, "activation"), (dict(x=None), NULL, "x"), (dict(codes=None), NULL, "codes"),
    (dict(scales=None), NULL, "scales"), (dict(y=None), NULL, "out"),
])
def test_linear_validation(s, kw, rc, operand):
    assert linear(s, **kw) == (rc, operand)


@pytest.mark.parametrize("s", TYPES)
@pytest.mark.parametrize("kw,rc,operand", [
    (dict(x_len=519), SHAPE, "x"), (dict(codes_t_len=650), SHAPE, "codes_t"), (dict(scales_t_len=4), SHAPE, "scales_t"),
    (dict(codes_t=0x100004), PARAM, "codes_t"), (dict(dy_len=19), SHAPE, "dy"), (dict(dx_len=519), SHAPE, "dx"),
    (dict(dw_len=649), SHAPE, "dw"), (dict(dw=None), SHAPE, "dw"), (dict(db_len=4), SHAPE, "dbias"),
    (dict(act=-1), UNSUPPORTED, "activation"), (dict(act=0), SHAPE, "preact"), (dict(z_len=0), SHAPE, "preact"),
    (dict(dy=None), NULL, "dy"), (dict(x=None), NULL, "x"), (dict(z=None), NULL, "preact"),
    (dict(codes_t=None), NULL, "codes_t"), (dict(codes_t=None, codes_t_len=0, scales_t=None, scales_t_len=0), NULL, "codes_t"),
    (dict(n=HUGE, x_len=130 * HUGE, dy_len=5 * HUGE, z_len=5 * HUGE, dx_len=130 * HUGE), UNSUPPORTED, "rows"),
])
def test_grad_validation(s, kw, rc, operand):
    assert grad(s, **kw) == (rc, operand)


@pytest.mark.parametrize("s", TYPES)
def test_outputs_overlap_no_operand(s):
    e = SIZE[s]
    for call, outs, lens in (
            (weight, {1: "codes", 2: "scales", 3: "codes_t", 4: "scales_t"}, [650 * e, CODES, SCALES, CODES_T, SCALES_T]),
            (linear, {5: "out", 6: "preact"}, [520 * e, CODES, SCALES, 5 * e, 20 * e, 20 * e, 20 * e]),
            (grad, {5: "dx", 6: "dw", 7: "dbias"},
             [20 * e, 520 * e, CODES_T, SCALES_T, 20 * e, 520 * e, 650 * e, 5 * e])):
        for out in outs:
            for other in range(len(lens)):
                if other == out:
                    continue
                at = apart(len(lens))
                at[out] = at[other] + (lens[other] - 1) // 16 * 16
                got = call(s, at)
                assert got[0] == PARAM and got[1] in outs.values(), (call.__name__, out, other, got)


def test_nothing_to_do_touches_no_device():
    assert linear("f32", n=0, x=None, x_len=0, r_len=0, y_len=0, z_len=0)[0] == _lib.MLRS_OK
    assert grad("f32", dx=None, dx_len=0, dw=None, dw_len=0, db=None, db_len=0)[0] == _lib.MLRS_OK


def test_prims_checks():
    w = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="device tensors"):
        prims.fp8_weight(w)
    w8 = prims.Fp8Weight(torch.zeros(4, 128, dtype=torch.float8_e4m3fn), torch.zeros(1, 4, dtype=torch.uint8), None,
                         None, 8)
    with pytest.raises(ValueError, match="device tensors"):
        prims.linear_fp8(w, w8)
    with pytest.raises(ValueError, match="needs the transposed weights"):
        prims.linear_fp8_grad(w, w, w8)
    with pytest.raises(ValueError, match="needs preact"):
        prims.linear_fp8_grad(w, w, w8, activation="gelu")


def test_reference_codes_are_those_of_the_type():
    """The reference's rounding against torch's conversion, at scale 1."""
    v = torch.cat([torch.linspace(-448, 448, 100001, dtype=torch.float64),
                   torch.linspace(-0.02, 0.02, 10001, dtype=torch.float64)]).float()
    assert torch.equal(layer.e4m3(v.double()), v.to(torch.float8_e4m3fn).double())
