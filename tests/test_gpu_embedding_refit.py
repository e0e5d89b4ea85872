"""An EmbeddingEncoder whose fit did not end has the weights it got to, in 8 bits too:
never an earlier fit's."""
import numpy as np
import pytest
import torch

from mlrs_amd import prims
from mlrs_amd.embedding import EmbeddingEncoder
from test_gpu_embedding import rows

pytestmark = pytest.mark.gpu


class Stop(Exception):
    pass


def stop_after(e, steps):
    """Lets a fit of `e` take some steps and then ends it."""
    inner = EmbeddingEncoder._loss_and_grads
    left = [steps]

    def step(*args):
        if not left[0]:
            raise Stop
        left[0] -= 1
        return inner(e, *args)

    e._loss_and_grads = step


def encoded(e, x):
    """transform, from the encoder's weights as they are."""
    h = torch.from_numpy(x).cuda()
    for i in range(0, len(e._params) - 2, 2):
        w8 = prims.fp8_weight(e._params[i])
        h = prims.linear_fp8(h, w8, bias=e._params[i + 1], activation="gelu" if i < len(e._params) - 4 else "none")
    return h.cpu().numpy()


def encoder(**kw):
    return EmbeddingEncoder(n_components=4, hidden=(16,), epochs=1, batch_size=100, products="fp8", **kw)


def test_a_stopped_refit_keeps_no_codes():
    x, y = rows(1, 500)
    e = encoder().fit(x, y)
    first = e.transform(x)
    e.random_state = 7
    stop_after(e, 3)
    with pytest.raises(Stop):
        e.fit(x, y)
    h = e.transform(x)
    assert np.array_equal(h, encoded(e, x)) and not np.array_equal(h, first)
    assert np.array_equal(h, e.transform(x)) and e.predict(x[:5]).shape == (5,)


def test_a_stopped_first_fit():
    x, y = rows(1, 500)
    e = encoder()
    stop_after(e, 2)
    with pytest.raises(Stop):
        e.fit(x, y)
    assert np.array_equal(e.transform(x), encoded(e, x))


def test_a_refused_refit_leaves_the_fit():
    x, y = rows(1, 500)
    e = encoder().fit(x, y)
    first, labels = e.transform(x), e.predict(x)
    e.state_bits = 7
    with pytest.raises(ValueError):
        e.fit(x[:, :5], y + 10)
    assert np.array_equal(e.transform(x), first) and np.array_equal(e.predict(x), labels)


def test_products_that_change_after_the_fit():
    """The layers take the products that the encoder has when they are computed."""
    x, y = rows(1, 500)
    e = encoder().fit(x, y)
    eight = e.transform(x)
    assert np.array_equal(eight, encoded(e, x))
    e.products = "native"
    native = e.transform(x)
    assert not np.array_equal(native, eight)
    e = encoder(random_state=2)
    e.products = "native"
    e.fit(x, y)
    e.products = "fp8"
    assert np.array_equal(e.transform(x), encoded(e, x))
