"""The formulas of tests/layer_reference.py against differentiation -- CPU only."""
import numpy as np
import pytest
import torch

import layer_reference as layer
import train_reference as ref


@pytest.mark.parametrize("act", ["none", "gelu", "gelu_tanh", "silu"])
def test_group_norm_gradient_is_the_derivative(act):
    g = torch.Generator().manual_seed(1)
    n, s, c, groups = 3, 5, 12, 4
    x, w, b, dy = (torch.randn(*k, generator=g, dtype=torch.float64) for k in ((n, s, c), (c,), (c,), (n, s, c)))
    by = layer.factor((n, s, c), 0.3, 7, 9)
    got = layer.group_norm(x, groups, w, b, 1e-3, act, by, dy)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    v = leaves[0].view(n, s, groups, -1)
    far = v - v.mean((1, 3), keepdim=True)
    xh = far / torch.sqrt((far ** 2).mean((1, 3), keepdim=True) + 1e-3)
    y = ref.act(xh.reshape(n, s, c) * leaves[1] + leaves[2], act)[0] * by
    for name, want in zip(("dx", "dw", "db"), torch.autograd.grad((y * dy).sum(), leaves)):
        assert torch.allclose(got[name][0], want, rtol=1e-9, atol=1e-12), name
    # and against differences
    e = 1e-6
    for i in (0, 17, 100):
        step = torch.zeros(n * s * c, dtype=torch.float64)
        step[i] = e
        value = [(layer.group_norm(x + k * step.view(n, s, c), groups, w, b, 1e-3, act, by)["y"][0] * dy).sum()
                 for k in (1, -1)]
        assert abs(float(value[0] - value[1]) / (2 * e) - float(got["dx"][0].view(-1)[i])) < 1e-6


def test_random_halves_are_uniform():
    """65,536 times eight: a bin of 256 holds 2048 on average, with a standard
    deviation of 45; seven of them on either side."""
    u = layer.random_halves(1 << 19, 0x123456789ABCDEF, 5)
    counts = np.bincount((u >> np.uint64(8)).astype(np.int64), minlength=256)
    assert abs(counts - 2048).max() < 7 * 45.3
    again = layer.random_halves(1 << 19, 0x123456789ABCDEF, 6)
    # equal halves of two offsets: one in 65536, 8 on average
    assert (u == again).sum() < 30
