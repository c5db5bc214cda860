"""GPU: the sums of s2_linear's fp32 results, and values that are not finite next to activated ones."""
import pytest
import torch

from tests import operator_oracles as oracles
from tests.test_gpu_linear import _case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 40, 300, 2500])
@pytest.mark.parametrize("k", [960, 1024, 10240])
def test_fp32_sums(s2lib, gpu_ctx, rows, k):
    """The tensor core drops some 6.2e-8 of a sum for each K block of 64; one sum has 14 of them at most: 8.7e-7 of the
    result in the 2-norm (sums of 24 blocks lost 1.5e-6)."""
    a, w, _, _, _ = _case(rows + k, rows, 384, k, bias=False, out="f32")
    got = s2lib.linear(gpu_ctx, a, w, out_dtype=s2lib.S2_DTYPE_F32).double()
    want = a.double() @ w.double().t()
    assert float((got - want).norm() / want.norm()) < 1.0e-6


@pytest.mark.parametrize("rows", [40, 200, 6000])
@pytest.mark.parametrize("k", [136, 1000])
@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("act", oracles.ACTS[1:])
def test_nonfinite_values_stay_apart(s2lib, gpu_ctx, rows, k, out, act):
    """NaN and infinities of either sign in some rows and in the bias of some columns: no other value changes."""
    n = 261
    a, w, b, _, _ = _case(k, rows, n, k)
    code = s2lib.S2_DTYPE_F32 if out == "f32" else s2lib.S2_DTYPE_BF16
    run = lambda a, b: s2lib.linear(gpu_ctx, a, w, b, act=oracles.ACTS.index(act), out_dtype=code)  # noqa: E731
    good = run(a, b)
    bad_a, bad_b = a.clone(), b.clone()
    hit = torch.zeros(rows, n, dtype=torch.bool, device="cuda")
    for r, v in ((0, float("nan")), (rows // 3, float("inf")), (rows - 1, -float("inf"))):
        bad_a[r, 5] = v
        hit[r] = True
    for c, v in ((0, float("nan")), (6, float("inf")), (130, -float("inf")), (n - 1, float("nan"))):
        bad_b[c] = v
        hit[:, c] = True
    got = run(bad_a, bad_b)
    assert gpu_ctx.status() == 0
    assert torch.equal(got[~hit], good[~hit])
    assert bool(torch.isnan(got[:, 0]).all()) and bool(torch.isnan(got[:, n - 1]).all())
    assert bool(torch.isinf(got[1:rows // 3, 6]).all()) and bool(torch.isnan(got[1:rows // 3, 130]).all())
