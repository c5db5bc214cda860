"""GPU: calls of the operators as a program writes them."""
import pytest
import torch

from tests import operator_oracles as oracles
from tests.test_gpu_group_norm_bounds import _want as bounds

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("channels", [1375, 64, 2048])
def test_group_norm_of_vectors_made_in_the_call(s2lib, gpu_ctx, channels):
    """gamma and beta that only the call holds, in front of a workspace: it must not lie where they are."""
    gen = torch.Generator(device="cuda").manual_seed(channels)
    x = torch.randn(2, 2 ** 24 // channels, channels, device="cuda", generator=gen).bfloat16()
    gamma, beta = (torch.randn(channels, device="cuda", generator=gen).double() for _ in range(2))
    assert s2lib.lib().s2_group_norm_workspace(2, x.shape[1], channels, channels) > 0
    kept = gamma.float(), beta.float()
    out = torch.empty_like(x)
    want = s2lib.group_norm(gpu_ctx, x, channels, *kept)
    del kept
    for _ in range(3):
        torch.cuda.empty_cache()
        got = s2lib.group_norm(gpu_ctx, x, channels, gamma.float(), beta.float(), out=out)
        assert gpu_ctx.status() == 0 and torch.equal(got, want)


def _rows_apart(rows):
    """A few rows at each end, and around the one whose first element is the 2^31st."""
    return torch.cat([torch.arange(0, 3), torch.arange(rows // 2, rows // 2 + 3), torch.arange(rows - 130, rows)]).cuda()


@pytest.mark.parametrize("long", ["operand", "result"])
@pytest.mark.parametrize("grouped", [False, True])
def test_linear_past_two_to_the_31_elements(s2lib, gpu_ctx, long, grouped):
    rows = 2**18 + 77
    n, k = (24, 8200) if long == "operand" else (8200, 24)
    gen = torch.Generator(device="cuda").manual_seed(1)
    a = torch.empty(rows, k, device="cuda", dtype=torch.bfloat16).normal_(generator=gen)
    w = torch.empty(n, k, device="cuda", dtype=torch.bfloat16).normal_(generator=gen).mul_(k**-0.5)
    bias = torch.randn(n, device="cuda", generator=gen)
    out = torch.full((rows, n), 3.0, device="cuda", dtype=torch.bfloat16)
    assert max(a.numel(), out.numel()) > 2**31
    if grouped:
        off = torch.tensor([0, 5, rows - 100, rows], dtype=torch.int32, device="cuda")
        s2lib.grouped_linear(gpu_ctx, a, w.expand(3, n, k).contiguous(), off, bias.expand(3, n).contiguous(), residual=out, out=out)
    else:
        s2lib.linear(gpu_ctx, a, w, bias, residual=out, out=out)
    assert gpu_ctx.status() == 0
    at = _rows_apart(rows)
    three = torch.full((at.numel(), n), 3.0, device="cuda", dtype=torch.bfloat16)
    oracles.check(out[at], *oracles.linear(a[at], w, bias, "none", None, three, torch.bfloat16))


@pytest.mark.parametrize("kind", ["two kernels", "slabs"])
def test_group_norm_past_two_to_the_31_elements(s2lib, gpu_ctx, kind):
    """Rows 8,200 channels apart: all of them, or a few channels of each."""
    rows, pitch = 2**18 + 77, 8200
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.empty(rows, pitch, device="cuda", dtype=torch.bfloat16).normal_(generator=gen)
    view = x.view(1, rows, pitch) if kind == "two kernels" else x.view(rows, 1, pitch)[:, :, :8]
    out = torch.empty(rows, pitch, device="cuda", dtype=torch.bfloat16).view(view.shape[0], view.shape[1], pitch)[..., :view.shape[2]]
    groups = view.shape[-1] // 8 if kind == "two kernels" else 2
    s2lib.group_norm(gpu_ctx, view, groups, out=out)
    assert gpu_ctx.status() == 0
    if kind == "slabs":
        want, bound = oracles.group_norm(view[-130:], groups, None, None, 1e-6, "none", torch.bfloat16)
        oracles.check(out[-130:], want, bound)
    else:
        for g in (0, 511, groups - 1):
            c = slice(8 * g, 8 * g + 8)
            # slices of 40 channels, two parts of the rows each: 51 rows at once, 2,571 in a thread's sums
            want, bound = bounds(view[:, :, c], 1, None, None, "none", torch.bfloat16, 2571)
            at = _rows_apart(rows)
            oracles.check(out[0, at, c], want[0, at], bound[0, at])
