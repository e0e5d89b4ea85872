"""Group norm of infinities, NaN and squares past float32's range, wherever in a group
they stand: rows, slabs in registers and groups split into runs give what the
definition does, and all three alike."""
import pytest
import torch

from mlrs_amd import prims

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")
# one position; a slab of a few; runs of positions, of one channel and of several
SHAPES = [(3, 64), (3, 5, 64), (3, 2000, 64), (3, 9000, 4), (3, 600, 4100)]
GROUPS = {4: 4, 64: 4, 4100: 2}


def normal(shape, dtype):
    g = torch.Generator().manual_seed(len(shape) + shape[1])
    return torch.randn(shape, generator=g, dtype=torch.float64).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("place", [0.0, 0.01, 0.5, 0.999])
@pytest.mark.parametrize("bad", [INF, -INF, NAN, "both"])
def test_nothing_of_such_a_group_is_a_number(dtype, shape, place, bad):
    """The mean of a group with an infinity is that infinity, of both or a NaN NaN; its
    variance, rstd and all of its y and dx are NaN; the other groups stay as they are."""
    n, c = shape[0], shape[-1]
    g = GROUPS[c]
    x, dy = normal(shape, dtype).cuda(), normal(shape, dtype).cuda()
    y0, mean0, rstd0 = prims.group_norm(x, g, keep_stats=True)
    dx0, _, _ = prims.group_norm_grad(dy, x, mean0, rstd0)
    v = x.view(n, -1, g, c // g)
    s = v.shape[1]
    at = int(place * s)
    v[1, at, g - 1, (c // g) // 2] = INF if bad == "both" else bad
    if bad == "both":
        v[1, s - 1 - at, g - 1, 0] = -INF
    others = torch.ones(n, g, dtype=torch.bool, device="cuda")
    others[1, g - 1] = False

    def check(t, t0):
        t, t0 = (u.view(n, -1, g, c // g).transpose(1, 2) for u in (t, t0))
        assert t[1, g - 1].isnan().all()
        assert torch.equal(t[others], t0[others])

    for act in ("none", "relu", "gelu", "silu"):
        y, mean, rstd = prims.group_norm(x, g, activation=act, keep_stats=True)
        want = prims.group_norm(torch.nan_to_num(x), g, activation=act)
        assert mean[1, g - 1].isnan() if bad in (NAN, "both") else mean[1, g - 1] == bad
        assert rstd[1, g - 1].isnan()
        assert torch.equal(mean[others], mean0[others]) and torch.equal(rstd[others], rstd0[others])
        check(y, want)
    check(prims.group_norm_grad(dy, x, mean, rstd)[0], dx0)


@pytest.mark.parametrize("shape", SHAPES)
def test_squares_past_the_range(shape):
    """Deviations near 1e25, whose squares are infinite in float32: rstd is 0 and y the
    bias, on every way."""
    c = shape[-1]
    x = normal(shape, torch.float32).cuda() * 1e25
    b = normal((1, c), torch.float32).cuda()[0]
    y, mean, rstd = prims.group_norm(x, GROUPS[c], bias=b, keep_stats=True)
    assert mean.isfinite().all() and not rstd.any()
    assert torch.equal(y, b.expand(shape))
