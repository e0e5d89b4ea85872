"""Group norm's gelu and its slope, value by value.

With weights of 0, z is the bias itself, whatever x holds, and the bias's gradient of a
dy that is 1 at one position is act'(z).  gelu is held to the accuracy of the other
layers' (2^-20 of z, 2^-20 (1 + z^2) of the slope: tests/train_reference.py) and one
rounding: more than that shows where an exact result lies near the middle of two
values, which some of all 16-bit values' do."""
import pytest
import torch

import train_reference as ref
from mlrs_amd import prims

pytestmark = pytest.mark.gpu


def values(dtype):
    """Every 16-bit value up to 12 in magnitude, or 65536 float32 ones."""
    if dtype == torch.float32:
        return 3 * torch.randn(1 << 16, generator=torch.Generator().manual_seed(1))
    z = torch.arange(-(1 << 15), 1 << 15, dtype=torch.int32).to(torch.int16).view(dtype)
    z = z[z.float().abs() <= 12]
    return torch.cat([z, torch.zeros(-len(z) % 512, dtype=dtype)])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("positions,every", [(1, 1), (2, 1), (3000, 8)])  # rows, slabs, runs
def test_gelu_and_its_slope(dtype, positions, every):
    for first in range(every):
        z = values(dtype)[first::every].contiguous()
        c = len(z)
        x = torch.randn(1, positions, c, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
        zd, wd = z.cuda(), torch.zeros(c, dtype=dtype, device="cuda")
        y, mean, rstd = prims.group_norm(x, c // 64, weight=wd, bias=zd, activation="gelu", keep_stats=True)
        want, slope = ref.act(z.double(), "gelu")
        assert torch.equal(y, y[:, :1].expand_as(y))
        ref.assert_near(y[0, positions // 2], (want, ref.FUN * z.double().abs()), "gelu")
        dy = torch.zeros_like(x)
        dy[0, positions // 2] = 1
        _, _, db = prims.group_norm_grad(dy, x, mean, rstd, weight=wd, bias=zd, activation="gelu")
        ref.assert_near(db, (slope, ref.FUN * (1 + z.double() ** 2)), "slope")
