"""Dropout and group norm reject bad arguments before anything is launched --
CPU only: the C ABI's checks run on sizes, the prims' on tensor metadata."""
import ctypes

import pytest
import torch

from mlrs_amd import _lib, prims

P = ctypes.c_void_p(0x1000)  # never dereferenced: validation fails first
SHAPE, UNSUPPORTED, NULL, PARAM = (_lib.MLRS_ERR_SHAPE_MISMATCH, _lib.MLRS_ERR_UNSUPPORTED,
                                   _lib.MLRS_ERR_NULL_POINTER, _lib.MLRS_ERR_INVALID_PARAM)
TYPES = ["f32", "f16", "bf16"]
SIZE = dict(f32=4, f16=2, bf16=2)
NAN = float("nan")


def failed(rc):
    e = _lib.ErrorInfo()
    _lib.load().mlrs_last_error(ctypes.byref(e))
    return rc, e.operand.decode()


def dropout(s, **kw):
    a = dict(x=P, x_len=20, p=0.5, seed=1, offset=2, step=None, r=ctypes.c_void_p(0x2000), r_len=20,
             y=ctypes.c_void_p(0x3000), y_len=20)
    a.update(kw)
    return failed(getattr(_lib.load(), "mlrs_dropout_" + s)(*a.values(), None))


@pytest.mark.parametrize("s", TYPES)
@pytest.mark.parametrize("kw,rc,operand", [
    (dict(x_len=-1), SHAPE, "x"), (dict(r_len=19), SHAPE, "residual"), (dict(r=None), SHAPE, "residual"),
    (dict(y_len=21), SHAPE, "out"), (dict(p=1.0), PARAM, "p"), (dict(p=-0.1), PARAM, "p"), (dict(p=NAN), PARAM, "p"),
    (dict(x=None), NULL, "x"), (dict(y=None), NULL, "out"), (dict(y=0x1004), PARAM, "out"),
    (dict(y=0x1FFE), PARAM, "out"), (dict(step=0x3004), PARAM, "out"),
])
def test_dropout_validation(s, kw, rc, operand):
    assert dropout(s, **kw) == (rc, operand)


def test_dropout_of_nothing():
    assert dropout("f32", x=None, x_len=0, r=None, r_len=0, y=None, y_len=0)[0] == _lib.MLRS_OK


def apart(count):
    return [0x100000 + i * (1 << 20) for i in range(count)]


NORM = dict(n=2, positions=3, c=8, g=4)


def norm(s, at=None, **kw):
    x, w, b, y, mean, rstd = at or apart(6)
    a = dict(x=x, x_len=48, **NORM, w=w, w_len=8, b=b, b_len=8, eps=1e-5, act=1, p=0.1, seed=0, offset=0, step=None,
             y=y, y_len=48, mean=mean, rstd=rstd, stats_len=8)
    a.update(kw)
    return failed(getattr(_lib.load(), "mlrs_group_norm_" + s)(*a.values(), None))


def norm_grad(s, at=None, **kw):
    dy, x, w, b, mean, rstd, dx, dw, db = at or apart(9)
    a = dict(dy=dy, dy_len=48, x=x, x_len=48, **NORM, w=w, w_len=8, b=b, b_len=8, mean=mean, rstd=rstd, stats_len=8,
             act=1, p=0.1, seed=0, offset=0, step=None, dx=dx, dx_len=48, dw=dw, dw_len=8, db=db, db_len=8)
    a.update(kw)
    return failed(getattr(_lib.load(), "mlrs_group_norm_grad_" + s)(*a.values(), None))


BOTH = [
    (dict(x_len=47), SHAPE, "x"), (dict(n=-2), SHAPE, "x"), (dict(positions=0, x_len=0), SHAPE, "features"),
    (dict(c=0, x_len=0), SHAPE, "features"), (dict(g=0), SHAPE, "groups"), (dict(g=3), SHAPE, "groups"),
    (dict(g=-4), SHAPE, "groups"), (dict(c=8194, g=1, x_len=6 * 8194), UNSUPPORTED, "groups"),
    (dict(n=0, c=(1 << 22) + 4, g=1 << 21, x_len=0), SHAPE, "groups"),
    (dict(n=0, c=1 << 23, g=1 << 21, x_len=0), UNSUPPORTED, "features"),
    (dict(n=0, positions=(1 << 31) + 1, x_len=0), UNSUPPORTED, "features"),
    (dict(w_len=7), SHAPE, "weight"), (dict(w=None), SHAPE, "weight"), (dict(b_len=9), SHAPE, "bias"),
    (dict(b=None), SHAPE, "bias"), (dict(stats_len=7), SHAPE, "stats"), (dict(act=5), UNSUPPORTED, "activation"),
    (dict(p=1.0), PARAM, "p"), (dict(p=NAN), PARAM, "p"), (dict(x=None), NULL, "x"),
]


@pytest.mark.parametrize("s", TYPES)
@pytest.mark.parametrize("kw,rc,operand", BOTH + [
    (dict(y_len=49), SHAPE, "out"), (dict(mean=None, rstd=None), SHAPE, "stats"), (dict(mean=None), NULL, "stats"),
    (dict(eps=-1.0), PARAM, "eps"), (dict(eps=NAN), PARAM, "eps"), (dict(eps=float("inf")), PARAM, "eps"),
    (dict(y=None), NULL, "out"),
])
def test_group_norm_validation(s, kw, rc, operand):
    assert norm(s, **kw) == (rc, operand)


@pytest.mark.parametrize("s", TYPES)
@pytest.mark.parametrize("kw,rc,operand", BOTH + [
    (dict(dy_len=47), SHAPE, "dy"), (dict(dx_len=47), SHAPE, "dx"), (dict(dx=None), SHAPE, "dx"),
    (dict(dw_len=7), SHAPE, "dweight"), (dict(db=None), SHAPE, "dbias"), (dict(dy=None), NULL, "dy"),
    (dict(mean=None), NULL, "stats"), (dict(rstd=None), NULL, "stats"),
])
def test_group_norm_grad_validation(s, kw, rc, operand):
    assert norm_grad(s, **kw) == (rc, operand)


@pytest.mark.parametrize("s", TYPES)
def test_group_norm_outputs_overlap_no_operand(s):
    size = SIZE[s]
    lens = [48 * size, 8 * size, 8 * size, 48 * size, 32, 32]
    for out, name in ((3, "out"), (4, "stats"), (5, "stats")):
        for other in range(6):
            if other == out:
                continue
            at = apart(6)
            at[out] = at[other] + lens[other] - 1
            got = norm(s, at)
            assert got[0] == PARAM and got[1] in (name, "out", "stats"), (out, other, got)
        assert norm(s, step=apart(6)[out] + 4)[0] == PARAM
    lens = [48 * size] * 2 + [8 * size] * 2 + [32] * 2 + [48 * size] + [8 * size] * 2
    for out, name in ((6, "dx"), (7, "dweight"), (8, "dbias")):
        for other in range(9):
            if other == out:
                continue
            at = apart(9)
            at[out] = at[other] + lens[other] - 1
            got = norm_grad(s, at)
            assert got[0] == PARAM and got[1] in (name, "dx", "dweight", "dbias"), (out, other, got)


def test_nothing_to_do_touches_no_device():
    none = dict(n=0, x_len=0, x=None, stats_len=0)
    assert norm("f32", y_len=0, y=None, **none)[0] == _lib.MLRS_OK
    assert norm_grad("f32", dx=None, dx_len=0, dw=None, dw_len=0, db=None, db_len=0)[0] == _lib.MLRS_OK


def test_prims_checks():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="device tensors"):
        prims.dropout(x, 0.1, 0)
    with pytest.raises(ValueError, match="device tensors"):
        prims.group_norm(x, 2)
    with pytest.raises(ValueError, match="device tensors"):
        prims.group_norm_grad(x, x, torch.zeros(4, 2), torch.zeros(4, 2))
