"""The training operators reject bad arguments before anything is launched --
CPU only: the C ABI's checks run on sizes, the prims' on tensor metadata."""
import ctypes

import numpy as np
import pytest
import torch

import train_reference as ref
from mlrs_amd import _lib, prims

P = ctypes.c_void_p(0x1000)  # never dereferenced: validation fails first
SHAPE, UNSUPPORTED, NULL, PARAM = (_lib.MLRS_ERR_SHAPE_MISMATCH, _lib.MLRS_ERR_UNSUPPORTED,
                                   _lib.MLRS_ERR_NULL_POINTER, _lib.MLRS_ERR_INVALID_PARAM)
TYPES = ["f32", "f16", "bf16"]


def failed(rc):
    e = _lib.ErrorInfo()
    _lib.load().mlrs_last_error(ctypes.byref(e))
    return rc, e.operand.decode(), (e.rows, e.cols, e.len)


def linear(s="f32", x_len=None, n=4, k=3, w_len=None, m=5, b=P, b_len=5, r=P, r_len=20, act=0, y=P, y_len=20, z=P,
           z_len=20, x=P, w=P):
    return failed(getattr(_lib.load(), "mlrs_linear_" + s)(
        x, n * k if x_len is None else x_len, n, k, w, m * k if w_len is None else w_len, m, b, b_len, r, r_len, act,
        y, y_len, z, z_len, None))


@pytest.mark.parametrize("s", TYPES)
@pytest.mark.parametrize("kw,rc,operand", [
    (dict(x_len=11), SHAPE, "x"), (dict(n=-1, x_len=-3), SHAPE, "x"), (dict(w_len=16), SHAPE, "w"),
    (dict(k=0), SHAPE, "features"), (dict(m=0), SHAPE, "features"),
    (dict(k=1 << 22, b_len=5), UNSUPPORTED, "features"), (dict(n=(1 << 31), y_len=0), UNSUPPORTED, "rows"),
    (dict(b_len=4), SHAPE, "bias"), (dict(b=None), SHAPE, "bias"), (dict(r_len=19), SHAPE, "residual"),
    (dict(r=None), SHAPE, "residual"), (dict(y_len=21), SHAPE, "out"), (dict(z_len=19), SHAPE, "preact"),
    (dict(z=None), SHAPE, "preact"), (dict(act=5), UNSUPPORTED, "activation"), (dict(act=-1), UNSUPPORTED, "activation"),
    (dict(x=None), NULL, "x"), (dict(w=None), NULL, "w"), (dict(y=None), NULL, "out"),
])
def test_linear_validation(s, kw, rc, operand):
    got = linear(s, **kw)
    assert got[:2] == (rc, operand)


def test_linear_with_nothing_to_do_touches_no_device():
    assert linear(n=0, r_len=0, y_len=0, z_len=0, x=None)[0] == _lib.MLRS_OK


def apart(count, step=1 << 20):
    return [0x100000 + i * step for i in range(count)]


SIZE = dict(f32=4, f16=2, bf16=2)


@pytest.mark.parametrize("s", TYPES)
def test_linear_outputs_overlap_no_operand(s):
    """4 x 3 by 3 x 5: each output a byte into, or a byte short of leaving, each
    operand; the residual's own buffer is refused only where it is another's too."""
    x, w, b, r, y, z = apart(6)
    at = dict(x=(x, 12), w=(w, 15), b=(b, 5), r=(r, 20), y=(y, 20), z=(z, 20))
    for out, name in (("y", "out"), ("z", "preact")):
        for other, (start, n) in at.items():
            if other == out:
                continue
            size = 20 * SIZE[s]
            for p in (start - size + 1, start + n * SIZE[s] - 1) + ((start,) if (out, other) != ("y", "r") else ()):
                got = linear(s, **{**dict(x=x, w=w, b=b, r=r, y=y, z=z), out: p})
                assert got[0] == PARAM and got[1] == (name if other != "z" else "preact"), (out, other, got)


@pytest.mark.parametrize("s", TYPES)
def test_gradients_overlap_no_operand(s):
    lib = _lib.load()
    names = ["dy", "x", "w", "z", "dx", "dw", "db"]
    lens = dict(dy=20, x=12, w=15, z=20, dx=12, dw=15, db=5)
    base = dict(zip(names, apart(7)))
    for out, name in (("dx", "dx"), ("dw", "dw"), ("db", "dbias")):
        for other in names:
            if other != out:
                p = {**base, out: base[other] + (lens[other] - 1) * SIZE[s]}
                got = failed(getattr(lib, "mlrs_linear_grad_" + s)(
                    p["dy"], 20, p["x"], 12, 4, 3, p["w"], 15, 5, p["z"], 20, 1, p["dx"], 12, p["dw"], 15, p["db"], 5,
                    None))
                assert got[0] == PARAM and got[1] in (name, "dx", "dw", "dbias"), (out, other, got)
    names = ["h", "w", "b", "t", "lse", "g", "dh", "dw", "db"]
    size = {**{n: SIZE[s] for n in names}, "t": 8, "lse": 4, "g": 4}
    lens = dict(h=12, w=15, b=5, t=4, lse=4, g=4, dh=12, dw=15, db=5)
    base = dict(zip(names, apart(9)))
    for out in ("dh", "dw", "db"):
        for other in names:
            if other != out:
                p = {**base, out: base[other] + lens[other] * size[other] - 1}
                got = failed(getattr(lib, "mlrs_softmax_xent_grad_" + s)(
                    p["h"], 12, 4, 3, p["w"], 15, 5, p["b"], 5, p["t"], 4, -100, p["lse"], p["g"], 4, p["dh"], 12,
                    p["dw"], 15, p["db"], 5, None))
                assert got[0] == PARAM and got[1] in ("dh", "dw", "dbias"), (out, other, got)
    names = ["h", "w", "b", "t", "loss", "lse"]
    base = dict(zip(names, apart(6)))
    for out in ("loss", "lse"):
        for other in names:
            if other != out:
                p = {**base, out: base[other] - 15}
                got = failed(getattr(lib, "mlrs_softmax_xent_" + s)(
                    p["h"], 12, 4, 3, p["w"], 15, 5, p["b"], 5, p["t"], 4, -100, p["loss"], p["lse"], 4, None))
                assert got[0] == PARAM and got[1] == "out", (out, other, got)


@pytest.mark.parametrize("s", TYPES)
@pytest.mark.parametrize("kw,rc,operand", [
    (dict(x_len=13), SHAPE, "x"), (dict(w_len=14), SHAPE, "w"), (dict(k=0, x_len=0, w_len=0), SHAPE, "features"),
    (dict(dy_len=19), SHAPE, "dy"), (dict(dx_len=13), SHAPE, "dx"), (dict(dx=None), SHAPE, "dx"),
    (dict(dw_len=16), SHAPE, "dw"), (dict(db_len=6), SHAPE, "dbias"), (dict(act=9), UNSUPPORTED, "activation"),
    (dict(act=0), SHAPE, "preact"), (dict(z_len=0), SHAPE, "preact"), (dict(dy=None), NULL, "dy"),
    (dict(x=None), NULL, "x"), (dict(z=None), NULL, "preact"), (dict(w=None), NULL, "w"),
])
def test_linear_grad_validation(s, kw, rc, operand):
    a = dict(dy=P, dy_len=20, x=P, x_len=12, n=4, k=3, w=P, w_len=15, m=5, z=P, z_len=20, act=1, dx=P, dx_len=12,
             dw=P, dw_len=15, db=P, db_len=5)
    a.update(kw)
    got = failed(getattr(_lib.load(), "mlrs_linear_grad_" + s)(*a.values(), None))
    assert got[:2] == (rc, operand)


@pytest.mark.parametrize("s", TYPES)
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("kw,rc,operand", [
    (dict(h_len=13), SHAPE, "h"), (dict(w_len=14), SHAPE, "w"), (dict(v=0, w_len=0, b_len=0), SHAPE, "features"),
    (dict(b_len=6), SHAPE, "bias"), (dict(b=None), SHAPE, "bias"), (dict(t_len=3), SHAPE, "target"),
    (dict(out_len=5), SHAPE, "out"), (dict(h=None), NULL, "h"), (dict(w=None), NULL, "w"), (dict(t=None), NULL, "target"),
])
def test_softmax_xent_validation(s, grad, kw, rc, operand):
    a = dict(h=P, h_len=12, n=4, d=3, w=P, w_len=15, v=5, b=P, b_len=5, t=P, t_len=4, ignore=-100)
    tail = dict(lse=P, grad=P, out_len=4, dh=P, dh_len=12, dw=P, dw_len=15, db=P, db_len=5) if grad else dict(
        loss=P, lse=P, out_len=4)
    a.update(tail)
    a.update(kw)
    f = getattr(_lib.load(), ("mlrs_softmax_xent_grad_" if grad else "mlrs_softmax_xent_") + s)
    assert failed(f(*a.values(), None))[:2] == (rc, operand)


@pytest.mark.parametrize("kw,operand", [(dict(dh_len=11), "dh"), (dict(dw_len=16), "dw"), (dict(db_len=4), "dbias"),
                                        (dict(dh=None), "dh")])
def test_softmax_xent_grad_outputs(kw, operand):
    a = dict(h=P, h_len=12, n=4, d=3, w=P, w_len=15, v=5, b=P, b_len=5, t=P, t_len=4, ignore=-100, lse=P, grad=P,
             out_len=4, dh=P, dh_len=12, dw=P, dw_len=15, db=P, db_len=5)
    a.update(kw)
    assert failed(_lib.load().mlrs_softmax_xent_grad_f32(*a.values(), None))[:2] == (SHAPE, operand)


def adamw(count=1, bits=32, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, step=1, tensors=True, **kw):
    t = _lib.AdamwTensor(param=0x1000, grad=0x1000, exp_avg=0x1000, exp_avg_sq=0x1000, len=5, weight_decay=0.1)
    for name, v in kw.items():
        setattr(t, name, v)
    items = (_lib.AdamwTensor * 1)(t) if tensors else None
    return failed(_lib.load().mlrs_adamw_step(items, count, bits, lr, b1, b2, eps, step, None, 0, None))


@pytest.mark.parametrize("kw,rc,operand", [
    (dict(count=-1), SHAPE, "tensors"), (dict(tensors=False), NULL, "tensors"), (dict(bits=16), UNSUPPORTED, "state_bits"),
    (dict(lr=-1.0), PARAM, "lr"), (dict(lr=float("nan")), PARAM, "lr"), (dict(b1=1.0), PARAM, "betas"),
    (dict(b2=-0.1), PARAM, "betas"), (dict(eps=-1e-8), PARAM, "eps"), (dict(step=0), PARAM, "step"),
    (dict(len=-1), SHAPE, "tensors"), (dict(param_dtype=3), UNSUPPORTED, "dtype"), (dict(grad_dtype=-1), UNSUPPORTED, "dtype"),
    (dict(weight_decay=-0.1), PARAM, "weight_decay"), (dict(weight_decay=float("inf")), PARAM, "weight_decay"),
    (dict(grad=None), NULL, "tensors"), (dict(param_dtype=1), NULL, "master"), (dict(bits=8), NULL, "scales"),
])
def test_adamw_validation(kw, rc, operand):
    assert adamw(**kw)[:2] == (rc, operand)


def test_adamw_of_more_elements_than_a_launch_has_threads_for():
    assert adamw(len=2 ** 36 - 4095)[:2] == (UNSUPPORTED, "tensors")


def test_adamw_with_nothing_to_do_touches_no_device():
    assert adamw(count=0, tensors=False)[0] == _lib.MLRS_OK
    assert adamw(len=0, param=None)[0] == _lib.MLRS_OK


@pytest.mark.parametrize("kw,rc,operand", [
    (dict(count=-1), SHAPE, "tensors"), (dict(tensors=False), NULL, "tensors"), (dict(len=-2), SHAPE, "tensors"),
    (dict(dtype=7), UNSUPPORTED, "dtype"), (dict(grad=None), NULL, "grad"), (dict(max_norm=0.0), PARAM, "max_norm"),
    (dict(max_norm=float("nan")), PARAM, "max_norm"), (dict(norm=None), NULL, "out"),
])
def test_clip_scale_validation(kw, rc, operand):
    a = dict(count=1, max_norm=1.0, norm=P, tensors=True, grad=0x1000, len=5, dtype=0)
    a.update(kw)
    items = (_lib.GradTensor * 1)(_lib.GradTensor(grad=a["grad"], len=a["len"], dtype=a["dtype"]))
    got = failed(_lib.load().mlrs_grad_clip_scale(items if a["tensors"] else None, a["count"], a["max_norm"],
                                                  a["norm"], P, None))
    assert got[:2] == (rc, operand)


@pytest.mark.parametrize("args,rc,operand", [
    ((P, -1, P, 0, 0, P, -1), SHAPE, "codes"), ((P, 257, P, 1, 0, P, 257), SHAPE, "scales"),
    ((P, 256, P, 1, 0, P, 255), SHAPE, "out"), ((P, 256, P, 1, 2, P, 256), UNSUPPORTED, "which"),
    ((None, 256, P, 1, 0, P, 256), NULL, "codes"),
])
def test_state_values_validation(args, rc, operand):
    assert failed(_lib.load().mlrs_adamw_state_values(*args, None))[:2] == (rc, operand)


def test_prims_refuse_what_the_library_does_not_take():
    x, w = torch.zeros(4, 3), torch.zeros(5, 3)
    t = torch.zeros(4, dtype=torch.int64)
    for call in (lambda: prims.linear(x, w), lambda: prims.linear_grad(x, x, w), lambda: prims.softmax_xent(x, w, t),
                 lambda: prims.clip_scale([x], 1.0), lambda: prims.adamw_step([x], [x], [x], [x], 1, 1e-3),
                 lambda: prims.adamw_state_values(x, x, "exp_avg")):
        with pytest.raises(ValueError, match="device tensors"):
            call()
    with pytest.raises(ValueError, match="at least one"):
        prims.clip_scale([], 1.0)
    with pytest.raises(ValueError, match="a tensor for each of the 2"):
        prims.adamw_step([x, x], [x], [x, x], [x, x], 1, 1e-3)
    with pytest.raises(ValueError, match="8-bit states need"):
        prims.adamw_step([x], [x], [x.byte()], [x.byte()], 1, 1e-3)
    with pytest.raises(ValueError, match="go with uint8"):
        prims.adamw_step([x], [x], [x], [x], 1, 1e-3, avg_scales=[x])
    with pytest.raises(ValueError, match="a number for each"):
        prims.adamw_step([x], [x], [x], [x], 1, 1e-3, weight_decay=[0.1, 0.2])
    with pytest.raises(TypeError, match="must hold tensors"):
        prims.adamw_step([1.0], [x], [x], [x], 1, 1e-3)
    with pytest.raises(ValueError, match="which should be"):
        prims.adamw_state_values(x, x, "m")
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        prims._train_suffix(x.double())
    with pytest.raises(ValueError, match="unknown activation"):
        prims._activation_id("tanh")


def test_the_codes_are_what_they_stand_for():
    """Every code is its own nearest value, whatever the random part; values
    between two codes go to either, as often as they are near it."""
    for mant in (3, 4):
        codes = np.arange(16 << mant)
        values = ref.code_values(codes, mant)
        assert np.all(np.diff(values) > 0) and values[0] == 0 and values[-1] == 2 - 2.0 ** -mant
        for r in (0, 1, 65535):
            assert np.array_equal(ref.codes_of(values, np.full(len(codes), r), mant), codes)
        y = 0.75 * values[:-1].astype(np.float64) + 0.25 * values[1:]
        r = np.arange(0, 65536, 16)
        up = np.mean([ref.codes_of(y, np.full(len(y), q), mant) - codes[:-1] for q in r], axis=0)
        # a quarter of the draws, within one draw of them
        assert np.all(np.abs(up - 0.25) <= 1.5 / len(r))


def test_the_hash_is_even():
    """Sixteen bits of it, of consecutive elements, as a mean and a variance of
    uniform numbers: within five standard deviations of them."""
    n = 1 << 16
    for key in (0, 1, 0x9E3779B1, 123456789):
        u = ref.mix32(np.arange(n, dtype=np.uint64) ^ ref.mix32(key))
        assert len(np.unique(u)) == n  # a bijection
        for part in (u & np.uint64(0xFFFF), u >> np.uint64(16)):
            f = part.astype(np.float64) / 65536
            assert abs(f.mean() - 0.5) < 5 * (1 / 12 / n) ** 0.5
            assert abs(f.var() - 1 / 12) < 5 * (1 / 180 / n) ** 0.5
            lag = np.corrcoef(f[:-1], f[1:])[0, 1]
            assert abs(lag) < 5 / n ** 0.5
