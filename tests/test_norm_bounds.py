"""The bounds of tests/norm_bounds.py are narrow enough to show a term that is left out
or a sum kept in 16 bits -- CPU only."""
import pytest
import torch

import norm_bounds
import train_reference as ref

TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,groups", norm_bounds.SHAPES)
def test_what_the_bounds_show(dtype, shape, groups):
    x, w, b, dy = norm_bounds.inputs(1, shape, groups, dtype)

    def result(change=None):
        return norm_bounds.group_norm(x, groups, w, b, 1e-5, "silu", None, dy,
                                      norm_bounds.split(shape, groups, dtype), change)

    want = result()
    kept = dict(mean=torch.float32, rstd=torch.float32)
    for name, (value, _) in want.items():
        ref.assert_near(value.to(kept.get(name, dtype)), want[name], name)
    for change, name in (("m1", "dx"), ("m2", "dx"), ("rstd", "rstd")):
        value = result(change)[name][0]
        with pytest.raises(AssertionError, match="out of bounds"):
            ref.assert_near(value.to(kept.get(name, dtype)), want[name], change)
    if dtype == torch.float32:
        for name in ("y", "dx", "dw", "db", "rstd"):
            with pytest.raises(AssertionError, match="out of bounds"):
                ref.assert_near(want[name][0].to(torch.bfloat16).float(), want[name], name)
            # and f16's eleven bits
            with pytest.raises(AssertionError, match="out of bounds"):
                ref.assert_near(want[name][0].to(torch.float16).float(), want[name], name)


@pytest.mark.parametrize("shape,groups", norm_bounds.SHAPES)
def test_a_large_mean_shows(shape, groups):
    """With a mean of 1000 standard deviations a shift of 0.03 of one is seen."""
    x, w, b, dy = norm_bounds.inputs(2, shape, groups, torch.float32, mean=1000.0)
    want = norm_bounds.group_norm(x, groups, None, None, 1e-5, "none", None, dy,
                                  norm_bounds.split(shape, groups, torch.float32))
    for name in ("mean", "y"):
        with pytest.raises(AssertionError, match="out of bounds"):
            ref.assert_near((want[name][0] + 0.03).float(), want[name], name)
