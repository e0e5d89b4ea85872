"""Group norm where one workgroup's slab has more groups than threads: a wave alone
takes up to 256 groups of a sample, a thread several of them."""
import pytest
import torch

from test_gpu_layer import check_norm

pytestmark = pytest.mark.gpu


# either side of 64 groups, whole octs and not, as many groups as a slab may have,
# more samples than workgroups
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", [
    ((3, 4, 64), 64), ((3, 8, 65), 65), ((3, 4, 128), 128), ((3, 2, 256), 128), ((2, 2, 512), 128), ((2, 2, 256), 256),
    ((2, 2, 510), 255), ((3, 2, 3, 195), 65), ((1000, 4, 200), 100), ((5000, 2, 96), 96),
])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_norm_many_groups_of_a_wave(dtype, shape, groups, p):
    check_norm(shape, groups, dtype, "silu", p=p, seed=shape[0] + groups)
