"""Linear, grouped linear and group norm in 64 bits, with an elementwise bound
on what an fp32 evaluation rounded once to the output's type may be off."""
import math

import torch

U = 2.0**-24  # half a step of fp32, relative
ACTS = ("none", "silu", "gelu_tanh", "gelu_erf")  # in the order of S2_ACT_*


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def activate(x, act):
    """(act(x), the sigmoid's argument) in x's type."""
    if act == "silu":
        return x * torch.sigmoid(x), x
    if act == "gelu_tanh":
        t = 2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x**3)
        return x * torch.sigmoid(t), t
    if act == "gelu_erf":
        return x * 0.5 * torch.special.erfc(-x / math.sqrt(2)), None
    return x, None


def activated(x, dx, act, fast=False):
    """act(x) and its bound, x known within dx.  The slopes of all three are at most 1.13.  The sigmoid forms cost
    an exponential (2 units plus the rounding of its argument t: |t| units), an addition, a division and a product;
    0.5 x (1 + erf) an absolute error of a few units of x.  fast: sigmoid(t) = (1 + tanh(t / 2)) / 2 with the device's
    tanh.approx, whose relative error is 2^-11 at most: half of that on the sigmoid, times |x|."""
    y, t = activate(x, act)
    if act == "none":
        return y, dx
    own = (16 + 4 * t.abs()) * U * y.abs() if t is not None else 8 * U * x.abs()
    if fast and t is not None:
        own = own + 2.0**-12 * x.abs()
    return y, 1.13 * dx + own + 1e-37


def linear(a, w, bias, act, gate, residual, dtype):
    """(out, bound).  Products of bf16 are exact in fp32; the tensor core adds K of them in steps of 16 into an fp32
    accumulator, each step off by at most a whole step (2 U) of the partial sum, which sum |a| |w| bounds; splitting
    the sum only shortens that."""
    a, w = a.double(), w.double()
    x = a @ w.t()
    s = a.abs() @ w.abs().t()
    dx = (math.ceil(a.shape[1] / 16) + 8) * 2 * U * s
    if bias is not None:
        x = x + bias.double()
        dx = dx + U * x.abs()
    y, dy = activated(x, dx, act)
    if gate is not None:
        y, dy = y * gate.double(), (dy + U * y.abs()) * gate.double().abs()
    if residual is not None:
        y = y + residual.double()
        dy = dy + U * y.abs()
    return y, dy + half_step(dtype) * (y.abs() + dy) + 1e-37


def grouped_linear(a, w, offsets, bias, act, gate, residual, dtype, before):
    out, bound = before.double().clone(), torch.zeros_like(before, dtype=torch.float64)
    for g, (lo, hi) in enumerate(zip(offsets, offsets[1:])):
        if lo < hi:
            out[lo:hi], bound[lo:hi] = linear(a[lo:hi], w[g], None if bias is None else bias[g], act,
                                              None if gate is None else gate[g],
                                              None if residual is None else residual[lo:hi], dtype)
    return out, bound


def group_norm(x, groups, gamma, beta, eps, act, dtype):
    """(out, bound) for x [instances, rows, channels].  A thread sums at most 24 rows of the tests' sizes: sums of
    squares around a value of the data (twice the variance on average) are within 2 * 2 * 24 units, their root
    within half of that, the mean within 40 units of the deviation; then a difference, two products and a sum."""
    i, r, c = x.shape
    v = x.double().reshape(i, r, groups, c // groups)
    mean = v.mean(dim=(1, 3), keepdim=True)
    var = ((v - mean) ** 2).mean(dim=(1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    z = ((v - mean) * rstd).reshape(i, r, c)
    off = (mean.abs() * rstd).expand(v.shape).reshape(i, r, c)
    g = torch.ones(c, dtype=torch.float64, device=x.device) if gamma is None else gamma.double()
    b = torch.zeros(c, dtype=torch.float64, device=x.device) if beta is None else beta.double()
    y = z * g + b
    dy = U * (g.abs() * (64 * z.abs() + 64 + 4 * off) + 4 * b.abs())
    y, dy = activated(y, dy, act, fast=dtype == torch.bfloat16)
    return y, dy + half_step(dtype) * (y.abs() + dy) + 1e-37


def check(got, want, bound, what=""):
    """Elementwise: |got - want| <= bound, and NaN or Inf exactly where want has them."""
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)), f"{what}: non-finite values in other places"
    over = ((got - want).abs() - bound)[fine]
    if over.numel() and float(over.max()) > 0:
        k = int(over.argmax())
        raise AssertionError(f"{what}: {int((over > 0).sum())} of {over.numel()} values off by more than the bound, "
                             f"worst {float(got[fine][k])} for {float(want[fine][k])} (bound {float(bound[fine][k])})")
