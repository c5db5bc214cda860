"""GPU: calls of the operators as a program writes them."""
import pytest
import torch

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
