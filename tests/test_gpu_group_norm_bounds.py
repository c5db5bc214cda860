"""GPU: s2_group_norm within what 32-bit statistics and one rounding to the output's type may be off, whatever the
activation and the type."""
import pytest
import torch

from tests import operator_oracles as oracles
from tests.test_gpu_group_norm import DT, _affine, _x

pytestmark = pytest.mark.gpu


def _want(x, groups, gamma, beta, act, dtype, rows_a_thread=24):
    """(out, bound).  The oracle's bound of an fp32 result, whose statistics count 24 rows a thread; more rows in one
    thread's sums raise that part in proportion.  Then the rounding to dtype."""
    y, bound = oracles.group_norm(x, groups, gamma, beta, 1e-6, act, torch.float32)
    bound = bound * max(1.0, rows_a_thread / 24)
    return y, bound + oracles.half_step(dtype) * (y.abs() + bound) + 1e-37


@pytest.mark.parametrize("size", [(1, 256, 512, 32), (3, 1185, 320, 32), (2, 333, 30, 3), (1, 6000, 512, 32), (2, 9000, 256, 32)], ids=str)
@pytest.mark.parametrize("tin", ["bf16", "f32"])
@pytest.mark.parametrize("tout", ["bf16", "f32"])
@pytest.mark.parametrize("act", oracles.ACTS)
def test_each_activation_and_type(s2lib, gpu_ctx, size, tin, tout, act):
    """gamma and beta wide enough that z reaches -30, where a result is far smaller than its argument."""
    i, r, c, g = size
    x = _x(r, i, r, c, DT[tin])
    gamma, beta = _affine(c, c)
    gamma, beta = gamma * 3, beta * 20
    got = s2lib.group_norm(gpu_ctx, x, g, gamma, beta, act=oracles.ACTS.index(act), out=torch.empty_like(x, dtype=DT[tout]))
    assert gpu_ctx.status() == 0
    oracles.check(got, *_want(x, g, gamma, beta, act, DT[tout]), f"{size} {tin} {tout} {act}")


# type, instances, rows, channels, groups, the channels' distance from zero, rows in one thread's sums (those of a
# part over 256 threads of one vector each)
LONG = [("f32", 1, 60000, 128, 32, 1.5, 17), ("bf16", 2, 100000, 64, 2, 30.0, 15), ("bf16", 1, 921600, 128, 32, 1.5, 130)]


@pytest.mark.parametrize("case", LONG, ids=str)
@pytest.mark.parametrize("act", ["none", "silu"])
def test_long_sums(s2lib, gpu_ctx, case, act):
    """Large x, read twice."""
    tin, i, r, c, g, far, rows = case
    x = _x(1, i, r, c, DT[tin], far)
    gamma, beta = _affine(2, c)
    got = s2lib.group_norm(gpu_ctx, x, g, gamma, beta, act=oracles.ACTS.index(act))
    assert gpu_ctx.status() == 0
    oracles.check(got, *_want(x, g, gamma, beta, act, DT[tin], rows), f"{case} {act}")
