"""GPU: the activations of s2_linear, s2_grouped_linear and s2_group_norm over all of their argument's range, next to
values that are not finite, through each kernel that applies them."""
import math

import pytest
import torch

from tests import operator_oracles as oracles

pytestmark = pytest.mark.gpu

U = oracles.U


def _values():
    """Arguments of the activation: dense where the result bends, sparse far out, with what is not finite between
    them.  An odd number of them, so that every kernel's last vector is cut."""
    near = torch.cat([torch.linspace(-16, 16, 1025, dtype=torch.float64), torch.linspace(-130, -16, 229, dtype=torch.float64)])
    far = torch.logspace(2, 30, 57, dtype=torch.float64)
    bad = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, -1e-30, 1e-30, 2e38, -2e38], dtype=torch.float64)
    v = torch.cat([near, far, -far, bad]).float()
    order = torch.randperm(v.numel(), generator=torch.Generator().manual_seed(3))
    return v[order].cuda()


def _want(x, act, dtype):
    """(act(x), bound) of the formula in 64 bits.  Beside what oracles.activated() counts of the sigmoid forms: a
    sigmoid below 2^-126 is zero.

    GELU with erf is max(x, 0) - a q, a = |x|, q = erfc(a / sqrt 2) / 2 = r P(6 r - 1) exp(-a^2 / 2), r = 1 / (a + 3).
    Relative to q in units of U: r 3 (a sum, a reciprocal of one ulp), which counts 1 + 6 r P' / P <= 2.4 times, 7; the
    argument of P rounded once, times P' / P, 1; P's own steps 3 and its fit 1; the exponent's three roundings
    3 a^2 / 2, the exponential 4 (two ulp); two products and one with a 3.  Together 19 + 1.5 a^2; then the sum."""
    x = x.double()
    y, bound = oracles.activated(x, torch.zeros_like(x), act)
    if act == "gelu_erf":
        a = x.abs().clamp(max=40)
        bound = (20 + 2 * a**2) * U * a * torch.special.erfc(a / math.sqrt(2)) / 2 + 2 * U * y.abs()
    bound = bound + 2.0**-126 * x.abs()
    return y, bound + oracles.half_step(dtype) * (y.abs() + bound) + 1e-37


def _check(got, x, act, dtype, what):
    want, bound = _want(x, act, dtype)
    want = want.expand(got.shape)
    oracles.check(got, want, bound.expand(got.shape), what)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(got.double()[inf], want[inf]), f"{what}: other infinities"


ACTS = ["silu", "gelu_tanh", "gelu_erf"]

# rows, K: the transposed product, single CTAs, CTA pairs; with fp32 results the two K of 15 blocks sum in registers
LINEAR = [(1, 8), (40, 8), (700, 8), (6000, 8), (700, 960), (6000, 960)]


@pytest.mark.parametrize("rows,k", LINEAR)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("act", ACTS)
def test_linear(s2lib, gpu_ctx, rows, k, dtype, act):
    """The product is zero, so that the bias is the argument to the last bit."""
    x = _values()
    a = torch.zeros(rows, k, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(x.numel(), k, device="cuda", dtype=torch.bfloat16)
    out = torch.empty(rows, x.numel(), device="cuda", dtype=dtype)
    s2lib.linear(gpu_ctx, a, w, x, act=oracles.ACTS.index(act), out=out)
    assert gpu_ctx.status() == 0
    _check(out, x, act, dtype, f"{rows} x {k} {act}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("act", ACTS)
def test_grouped_linear(s2lib, gpu_ctx, dtype, act):
    x = _values()
    a = torch.zeros(90, 8, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(2, x.numel(), 8, device="cuda", dtype=torch.bfloat16)
    off = torch.tensor([0, 31, 90], dtype=torch.int32, device="cuda")
    out = torch.empty(90, x.numel(), device="cuda", dtype=dtype)
    s2lib.grouped_linear(gpu_ctx, a, w, off, torch.stack([x, x.flip(0)]), act=oracles.ACTS.index(act), out=out)
    assert gpu_ctx.status() == 0
    _check(out[:31], x, act, dtype, act)
    _check(out[31:], x.flip(0), act, dtype, act)


# instances, rows: one CTA a slab, clusters, clusters of more rows a thread, two kernels
NORM = [(1, 5), (2, 700), (1, 6000), (2, 30000)]


@pytest.mark.parametrize("tin", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("tout", [torch.bfloat16, torch.float32], ids=["to_bf16", "to_f32"])
@pytest.mark.parametrize("instances,rows", NORM)
@pytest.mark.parametrize("whole", [True, False], ids=["vectors", "single"])
@pytest.mark.parametrize("act", ACTS)
def test_group_norm(s2lib, gpu_ctx, instances, rows, tin, tout, whole, act):
    """A scale of zero leaves the shift, to the last bit, as the argument."""
    beta = _values()
    if whole:
        beta = torch.cat([beta, beta[: -beta.numel() % 8]])
    c = beta.numel()
    x = torch.randn(instances, rows, c, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(tin)
    out = torch.empty(instances, rows, c, device="cuda", dtype=tout)
    s2lib.group_norm(gpu_ctx, x, c, torch.zeros(c, device="cuda"), beta, act=oracles.ACTS.index(act), out=out)
    assert gpu_ctx.status() == 0
    _check(out[:, :2], beta, act, tout, f"{instances} x {rows} {act}")
    first = out[:1, :1].expand_as(out)
    assert torch.equal(torch.isnan(out), torch.isnan(first)) and torch.equal(out.nan_to_num(), first.nan_to_num())
