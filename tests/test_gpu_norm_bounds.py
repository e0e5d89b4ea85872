"""Group norm and its gradient within bounds that follow the kernels' sums."""
import pytest
import torch

import layer_reference as layer
import norm_bounds
import train_reference as ref
from mlrs_amd import prims

pytestmark = pytest.mark.gpu


def check(seed, shape, groups, dtype, act, p=0.0, affine=True, mean=0.5):
    x, w, b, dy = norm_bounds.inputs(seed, shape, groups, dtype, mean=mean)
    if not affine:
        w = b = None
    by = layer.factor(shape, p, 3, 7) if p else None
    want = norm_bounds.group_norm(x, groups, w, b, 1e-5, act, by, dy, norm_bounds.split(shape, groups, dtype))
    x, w, b, dy = (t if t is None else t.cuda() for t in (x, w, b, dy))
    kw = dict(weight=w, bias=b, activation=act, p=p, seed=3, offset=7)
    y, m, rstd = prims.group_norm(x, groups, keep_stats=True, **kw)
    got = [y, m, rstd, *prims.group_norm_grad(dy, x, m, rstd, **kw)]
    for name, t in zip(("y", "mean", "rstd", "dx", "dw", "db"), got):
        if t is not None:
            ref.assert_near(t, want[name], "%s of %s in %d groups, %s %s" % (name, shape, groups, dtype, act))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("shape,groups", norm_bounds.SHAPES)
def test_within_the_sums_bounds(dtype, act, shape, groups):
    check(1, shape, groups, dtype, act)
    check(3, shape, groups, dtype, act, p=0.3)


@pytest.mark.parametrize("shape,groups", norm_bounds.SHAPES)
def test_of_a_large_mean(shape, groups):
    check(2, shape, groups, torch.float32, "none", affine=False, mean=1000.0)
