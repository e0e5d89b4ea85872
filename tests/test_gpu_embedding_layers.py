"""EmbeddingEncoder with group norm, dropout and 8-bit products: its gradients
against automatic differentiation in 64 bits, and runs of them together."""
import numpy as np
import pytest
import torch

import layer_reference as layer
import train_reference as ref
from mlrs_amd import prims
from mlrs_amd.embedding import EmbeddingEncoder
from mlrs_amd.neighbors import KNeighborsClassifier
from test_gpu_embedding import rows

pytestmark = pytest.mark.gpu


class Product8(torch.autograd.Function):
    """x w^T of what 8 bits hold of both, and the gradient that goes with it."""

    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x, w)
        return layer.fp8_blocks(x)[0] @ layer.fp8_blocks(w, 128)[0].t()

    @staticmethod
    def backward(ctx, dz):
        x, w = ctx.saved_tensors
        dx = layer.fp8_blocks(dz)[0] @ layer.fp8_blocks(w, 128)[0]
        dzt, xt = (layer.fp8_blocks(v.t().contiguous())[0] for v in (dz, x))
        return dx, dzt @ xt.t()


def want_of(e, x, t, weight, seed, step, hidden):
    """(loss, gradients) of the same network in 64 bits."""
    params = [p.double().cpu().requires_grad_() for p in e._params]
    h, at, layers = x.double().cpu(), 0, hidden + 1
    for i in range(layers):
        w, b = params[at:at + 2]
        at += 2
        y = (Product8.apply(h, w) if e.products == "fp8" else h @ w.t()) + b
        if i < hidden:
            if e.norm_groups is not None:
                g, n = e.norm_groups, len(y)
                v = y.view(n, g, -1)
                v = v - v.mean(2, keepdim=True)
                v = v / torch.sqrt((v * v).mean(2, keepdim=True) + 1e-5)
                y = v.reshape(n, -1) * params[at] + params[at + 1]
                at += 2
            y = torch.nn.functional.gelu(y)
            if e.dropout:
                y = y * layer.factor(tuple(y.shape), e.dropout, seed, step * layers + i)
            y = y + h if y.shape == h.shape else y
        h = y
    z = h @ params[at].t() + params[at + 1]
    loss = torch.nn.functional.cross_entropy(z, t.cpu(), reduction="none", ignore_index=-100)
    (loss * weight.double().cpu()).sum().backward()
    return loss.detach(), [p.grad for p in params]


def setup(dtype, **kw):
    e = EmbeddingEncoder(n_components=12, hidden=(24, 24, 40), activation="gelu", dtype=dtype, **kw)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    e._params = e._init_params(20, e._validate(), 7, torch.device("cuda"), gen)
    for p in e._params:
        if p.dim() == 1:
            p += 0.2 * torch.randn(p.shape, device="cuda", generator=gen).to(p.dtype)
    x = torch.randn(50, 20, device="cuda", generator=gen).to(e._params[0].dtype)
    t = torch.randint(0, 7, (50,), device="cuda", generator=gen)
    t[3] = -100
    return e, x, t, torch.rand(50, device="cuda", generator=gen)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("groups,p", [(None, 0.3), (4, 0.0), (4, 0.3), (1, 0.1)])
def test_gradients_against_autograd(dtype, groups, p):
    e, x, t, weight = setup(dtype, norm_groups=groups, dropout=p)
    loss, grads = e._loss_and_grads(x, t, weight, seed=11, step=5)
    want, want_grads = want_of(e, x, t, weight, 11, 5, 3)
    # as without them, some twenty-five roundings of independent sign; where a norm
    # divides by a group's spread, its input's rounding counts 1 / spread times: of
    # sums of variance near 1 that is 2 at most over groups of six
    room = 50 * ref.UNIT[x.dtype] + 128 * ref.U32
    assert (loss.cpu().double() - want).norm() <= room * want.norm()
    assert len(grads) == len(want_grads)
    for g, w in zip(grads, want_grads):
        assert g.shape == w.shape and (g.cpu().double() - w).norm() <= room * w.norm()


@pytest.mark.parametrize("groups,p", [(None, 0.0), (4, 0.3)])
def test_gradients_of_8_bit_products(groups, p):
    """In float32 the values in 8 bits are those of the reference but where one lies
    within 2^-18 of the border of two codes: 2^-3 of it is a code's step, so one in
    2^14 elements, each a step off, in fewer than 2^13 of them a layer: room for four
    in the some 2,000 of a matrix here, 2^-4 sqrt(4 / 2000)."""
    e, x, t, weight = setup("float32", norm_groups=groups, dropout=p, products="fp8")
    loss, grads = e._loss_and_grads(x, t, weight, seed=11, step=5)
    want, want_grads = want_of(e, x, t, weight, 11, 5, 3)
    assert (loss.cpu().double() - want).norm() <= 3e-3 * want.norm()
    for g, w in zip(grads, want_grads):
        assert (g.cpu().double() - w).norm() <= 3e-3 * w.norm()


@pytest.mark.parametrize("dtype,products", [("float32", "fp8"), ("bfloat16", "fp8"), ("float16", "fp8"),
                                            ("bfloat16", "native")])
def test_everything_together(dtype, products):
    """Norm, dropout, 8-bit products and 8-bit states in one fit, repeatable, and a
    search over what it learned."""
    x, y = rows(1, 3000)
    kw = dict(n_components=8, hidden=(64, 64), epochs=3, batch_size=500, learning_rate=3e-3, dtype=dtype, state_bits=8,
              random_state=3, norm_groups=4, dropout=0.1, products=products)
    e = EmbeddingEncoder(**kw)
    h = e.fit_transform(x, y)
    assert np.isfinite(h).all() and np.isfinite(e.loss_curve_).all() and len(e.loss_curve_) == 3
    again = EmbeddingEncoder(**kw).fit(x, y)
    assert again.loss_curve_ == e.loss_curve_ and np.array_equal(again.transform(x), h)
    KNeighborsClassifier(n_neighbors=5).fit(h, y).predict(e.transform(x[:100]))
    assert e.predict(x[:10]).shape == (10,) and np.isfinite(e.score(x, y))
    # one row, as an online encoder answers a request, is its row of the table up to
    # the order of sums
    one = e.transform(x[:1])
    assert np.abs(one - h[:1]).max() <= 0.1 * np.abs(h).max()


def test_dropout_is_for_fitting_alone():
    x, y = rows(2, 500)
    e = EmbeddingEncoder(n_components=4, hidden=(16,), epochs=1, batch_size=100, dropout=0.5).fit(x, y)
    assert np.array_equal(e.transform(x), e.transform(x))
    w, b = e._params[:2]
    xd = torch.from_numpy(x).cuda()
    h = prims.linear(prims.linear(xd, w, bias=b, activation="gelu"), e._params[2], bias=e._params[3])
    assert np.array_equal(e.transform(x), h.cpu().numpy())
