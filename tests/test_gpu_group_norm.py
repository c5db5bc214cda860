"""GPU: s2_group_norm against the 64-bit formula, and the three operators
together as a VAE block and a two-stream MLP use them."""
import pytest
import torch

from tests import operator_oracles as oracles

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _x(seed, i, r, c, dtype, far=1.5):
    gen = _gen(seed)
    x = torch.randn(i, r, c, device="cuda", generator=gen)
    x = x * (torch.rand(c, device="cuda", generator=gen) * 2 + 0.2) + torch.randn(c, device="cuda", generator=gen) * far
    return x.to(dtype)


def _affine(seed, c):
    gen = _gen(seed)
    return torch.randn(c, device="cuda", generator=gen) * 0.3 + 1, torch.randn(c, device="cuda", generator=gen) * 0.3


# instances, rows, channels, groups
SIZES = [(1, 1, 8, 1), (1, 1, 64, 8), (2, 2, 32, 32), (1, 256, 512, 32), (3, 7, 320, 32), (3, 1185, 320, 32),
         (2, 100, 7, 7), (2, 333, 30, 3), (1, 50, 1000, 1), (2, 65, 2048, 1), (1, 40, 4104, 1), (24, 5, 96, 32),
         (1, 20000, 64, 32), (5, 3600, 256, 32), (1, 3000, 1536, 32), (40, 17, 128, 8), (1, 9, 2047, 23),
         (2, 19, 4096, 4096), (2, 3000, 660, 20), (40, 100, 660, 20), (3, 2500, 20, 5), (9, 4000, 39, 1),
         (300, 7, 12, 3), (5, 1200, 1980, 60)]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("form", [("bf16", "bf16", "silu", True), ("f32", "f32", "none", True),
                                  ("f32", "bf16", "gelu_tanh", False), ("bf16", "f32", "gelu_erf", True)],
                         ids=lambda f: f"{f[0]}-{f[1]}-{f[2]}")
def test_group_norm(s2lib, gpu_ctx, size, form):
    i, r, c, g = size
    tin, tout, act, affine = form
    x = _x(r + c, i, r, c, DT[tin])
    gamma, beta = _affine(c, c) if affine else (None, None)
    got = s2lib.group_norm(gpu_ctx, x, g, gamma, beta, eps=1e-5, act=oracles.ACTS.index(act),
                           out_dtype=s2lib.S2_DTYPE_F32 if tout == "f32" else s2lib.S2_DTYPE_BF16)
    assert gpu_ctx.status() == 0 and got.shape == x.shape
    oracles.check(got, *oracles.group_norm(x, g, gamma, beta, 1e-5, act, DT[tout]), f"{size} {form}")


@pytest.mark.parametrize("size", [(6, 4282, 128, 32), (1, 6000, 512, 32), (1, 5001, 512, 32), (1, 12288, 512, 32),
                                  (1, 4000, 33, 33), (1, 6100, 36, 4), (2, 6529, 20, 1)], ids=str)
@pytest.mark.parametrize("types", [("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32"), ("f32", "f32")],
                         ids=lambda t: "-".join(t))
def test_clusters_of_any_size(s2lib, gpu_ctx, size, types):
    """Rows that more than eight a thread of a cluster hold."""
    i, r, c, g = size
    x = _x(r + c, i, r, c, DT[types[0]])
    gamma, beta = _affine(c, c)
    got = s2lib.group_norm(gpu_ctx, x, g, gamma, beta, act=s2lib.S2_ACT_SILU,
                           out_dtype=s2lib.S2_DTYPE_F32 if types[1] == "f32" else s2lib.S2_DTYPE_BF16)
    assert gpu_ctx.status() == 0
    oracles.check(got, *oracles.group_norm(x, g, gamma, beta, 1e-6, "silu", DT[types[1]]), f"{size} {types}")


def test_large_slabs(s2lib, gpu_ctx):
    """More rows than the cluster's shared memory keeps: the rest is read again."""
    for tin, i, r, c, g, far in (("f32", 1, 60000, 128, 32, 1.5), ("bf16", 2, 100000, 64, 2, 30.0)):
        x = _x(1, i, r, c, DT[tin], far)
        gamma, beta = _affine(2, c)
        got = s2lib.group_norm(gpu_ctx, x, g, gamma, beta, act=s2lib.S2_ACT_SILU)
        want, bound = oracles.group_norm(x, g, gamma, beta, 1e-6, "silu", DT[tin])
        # up to 512 rows a thread here against the 24 the bound counts: the sums' units grow with them
        oracles.check(got, want, bound + 512 / 24 * (bound - oracles.half_step(DT[tin]) * want.abs()))


def test_channels_far_from_zero(s2lib, gpu_ctx):
    """A mean of 1000 deviations: sums of x^2 in 32 bits would leave nothing of the variance."""
    x = torch.randn(2, 500, 64, device="cuda", generator=_gen(3)) + 1000.0
    got = s2lib.group_norm(gpu_ctx, x, 8)
    oracles.check(got, *oracles.group_norm(x, 8, None, None, 1e-6, "none", torch.float32))


@pytest.mark.parametrize("shift", [0, 1])
def test_strides_and_in_place(s2lib, gpu_ctx, shift):
    i, r, c, g = 2, 77, 96, 8
    for dtype in DT.values():
        wide = _x(5, i, r, c + 24, dtype)
        out = torch.full((i, r, c + 40), 7.0, device="cuda", dtype=dtype)
        x, y = wide[:, :, 8 + shift:8 + shift + c], out[:, :, 16 + shift:16 + shift + c]
        gamma, beta = _affine(4, c)
        want = oracles.group_norm(x, g, gamma, beta, 1e-6, "silu", dtype)
        s2lib.group_norm(gpu_ctx, x, g, gamma, beta, act=s2lib.S2_ACT_SILU, out=y)
        oracles.check(y, *want)
        y.fill_(7.0)
        assert bool((out == 7.0).all()), "the columns around the output stay"
        kept = wide.clone()
        s2lib.group_norm(gpu_ctx, x, g, gamma, beta, act=s2lib.S2_ACT_SILU, out=x)
        oracles.check(x, *want)
        x.copy_(kept[:, :, 8 + shift:8 + shift + c])
        assert torch.equal(wide, kept)


def test_nonfinite_stays_in_its_group(s2lib, gpu_ctx):
    x = _x(6, 3, 400, 64, torch.float32)
    good = s2lib.group_norm(gpu_ctx, x, 8)
    x[1, 7, 9] = float("nan")
    x[2, 399, 63] = float("inf")
    got = s2lib.group_norm(gpu_ctx, x, 8)
    hit = torch.zeros_like(x, dtype=torch.bool)
    hit[1, :, 8:16] = True
    hit[2, :, 56:64] = True
    assert torch.equal(got[~hit], good[~hit]) and bool(torch.isnan(got[hit]).all())


def test_constant_and_empty(s2lib, gpu_ctx):
    x = torch.full((2, 30, 16), -3.25, device="cuda")
    gamma, beta = _affine(1, 16)
    got = s2lib.group_norm(gpu_ctx, x, 2, gamma, beta)
    assert torch.equal(got, beta.expand_as(got)), "no variance: the shift alone"
    for shape in ((0, 5, 16), (2, 0, 16)):
        assert s2lib.group_norm(gpu_ctx, torch.empty(shape, device="cuda"), 4).shape == shape


def test_repeats_and_replays(s2lib, gpu_ctx):
    x = _x(8, 2, 5000, 128, torch.bfloat16)
    gamma, beta = _affine(2, 128)
    out = torch.empty_like(x)
    want = s2lib.group_norm(gpu_ctx, x, 32, gamma, beta)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    home = gpu_ctx.stream
    with torch.cuda.graph(graph):
        gpu_ctx.set_stream(torch.cuda.current_stream())
        s2lib.group_norm(gpu_ctx, x, 32, gamma, beta, out=out)
    gpu_ctx.set_stream(home)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    x.copy_(_x(9, 2, 5000, 128, torch.bfloat16))
    graph.replay()
    torch.cuda.synchronize()
    oracles.check(out, *oracles.group_norm(x, 32, gamma, beta, 1e-6, "none", torch.bfloat16))
    del graph


def test_residual_block(s2lib, gpu_ctx):
    """Norm + SiLU, product, norm + SiLU, product onto the 1x1 shortcut: each step checked on the values that the
    step before it wrote."""
    frames, rows, cin, cout = 2, 900, 256, 384
    x = _x(11, frames, rows, cin, torch.bfloat16)
    gen = _gen(12)
    w1, w2, ws = (torch.randn(cout, k, device="cuda", generator=gen).mul_(k**-0.5).bfloat16() for k in (cin, cout, cin))
    b1, b2, bs = (torch.randn(cout, device="cuda", generator=gen) for _ in range(3))
    g1, t1 = _affine(1, cin)
    g2, t2 = _affine(2, cout)
    flat = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
    h1 = s2lib.group_norm(gpu_ctx, x, 32, g1, t1, act=s2lib.S2_ACT_SILU)
    y1 = s2lib.linear(gpu_ctx, flat(h1), w1, b1).view(frames, rows, cout)
    h2 = s2lib.group_norm(gpu_ctx, y1, 32, g2, t2, act=s2lib.S2_ACT_SILU)
    y2 = s2lib.linear(gpu_ctx, flat(h2), w2, b2)
    out = s2lib.linear(gpu_ctx, flat(x), ws, bs, residual=y2, out=y2.clone())
    assert gpu_ctx.status() == 0
    oracles.check(h1, *oracles.group_norm(x, 32, g1, t1, 1e-6, "silu", torch.bfloat16))
    oracles.check(flat(y1), *oracles.linear(flat(h1), w1, b1, "none", None, None, torch.bfloat16))
    oracles.check(h2, *oracles.group_norm(y1, 32, g2, t2, 1e-6, "silu", torch.bfloat16))
    oracles.check(y2, *oracles.linear(flat(h2), w2, b2, "none", None, None, torch.bfloat16))
    oracles.check(out, *oracles.linear(flat(x), ws, bs, "none", None, y2, torch.bfloat16))


def test_attention_block(s2lib, gpu_ctx):
    """Norm in front of the VAE's attention layer, its output added back by a product with one epilogue."""
    import numpy as np

    tokens, E = 300, 128
    rng = np.random.default_rng(0)
    weights = (rng.standard_normal(4 * (E * E + E)) * E**-0.5).astype(np.float32)
    x = _x(13, 1, tokens, E, torch.float32)
    gamma, beta = _affine(3, E)
    h = s2lib.group_norm(gpu_ctx, x, 32, gamma, beta)
    oracles.check(h, *oracles.group_norm(x, 32, gamma, beta, 1e-6, "none", torch.float32))
    mha = s2lib.VaeMha(gpu_ctx, E, 1, E**-0.5, weights)
    y = mha.forward(h[0])
    eye = torch.eye(E, device="cuda", dtype=torch.bfloat16)
    out = s2lib.linear(gpu_ctx, y.bfloat16(), eye, residual=x[0], out_dtype=s2lib.S2_DTYPE_F32)
    assert gpu_ctx.status() == 0
    assert torch.equal(out, y.bfloat16().float() + x[0])
    mha.close()


def test_two_stream_mlp(s2lib, gpu_ctx):
    """Up and down projections with separate video and text weights, the second onto the gated fp32 residual in place,
    against the same through one linear per stream: the same tiles, so the same bits where the sizes choose them."""
    video, text, D, F = 700, 58, 256, 1024
    rows = video + text
    gen = _gen(14)
    x = torch.randn(rows, D, device="cuda", generator=gen)
    h = s2lib.ada_rmsnorm(gpu_ctx, x, 1e-5, torch.zeros(D, device="cuda"), torch.ones(D, device="cuda"))
    up = torch.randn(2, F, D, device="cuda", generator=gen).mul_(D**-0.5).bfloat16()
    down = torch.randn(2, D, F, device="cuda", generator=gen).mul_(F**-0.5).bfloat16()
    bu, bd, gate = (torch.randn(2, n, device="cuda", generator=gen) for n in (F, D, D))
    off = torch.tensor([0, video, rows], dtype=torch.int32, device="cuda")
    u = s2lib.grouped_linear(gpu_ctx, h, up, off, bu, act=s2lib.S2_ACT_GELU_TANH)
    y = x.clone()
    s2lib.grouped_linear(gpu_ctx, u, down, off, bd, gate=gate, residual=y, out=y)
    assert gpu_ctx.status() == 0
    oracles.check(u, *oracles.grouped_linear(h, up, off.tolist(), bu, "gelu_tanh", None, None, torch.bfloat16, u))
    oracles.check(y, *oracles.grouped_linear(u, down, off.tolist(), bd, "none", gate, x, torch.float32, x))
    for g, (lo, hi) in enumerate(((0, video), (video, rows))):
        one = s2lib.linear(gpu_ctx, h[lo:hi], up[g], bu[g], act=s2lib.S2_ACT_GELU_TANH)
        oracles.check(one, *oracles.linear(h[lo:hi], up[g], bu[g], "gelu_tanh", None, None, torch.bfloat16))
