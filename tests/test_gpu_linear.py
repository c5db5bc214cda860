"""GPU: s2_linear and s2_grouped_linear against the 64-bit formula, at the
sizes, strides, alignments and group layouts where a tile can go wrong."""
import ctypes as C

import pytest
import torch

from tests import operator_oracles as oracles

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(gen, rows, k, pad=0, scale=1.0):
    """bf16 rows with NaN between their end and the stride."""
    pitch = (k + 7) // 8 * 8 + pad
    full = torch.full((rows, pitch), float("nan"), device="cuda", dtype=torch.bfloat16)
    full[:, :k] = (torch.randn(rows, k, device="cuda", generator=gen) * scale).bfloat16()
    return full[:, :k]


def _case(seed, rows, n, k, *, groups=None, bias=True, gate=False, residual=False, out="bf16", pad=0):
    gen = _gen(seed)
    G = groups or 1
    vec = (G, n) if groups else (n,)
    a = _rows(gen, rows, k, pad)
    w = _rows(gen, G * n, k, pad, k**-0.5)
    w = w.unflatten(0, (G, n)) if groups else w
    b = torch.randn(vec, device="cuda", generator=gen) if bias else None
    gt = torch.randn(vec, device="cuda", generator=gen) if gate else None
    res = torch.randn(rows, n, device="cuda", generator=gen).to(DT[out]) if residual else None
    return a, w, b, gt, res


SIZES = [(1, 8, 8), (1, 1, 1), (1, 2560, 2560), (3, 130, 72), (16, 128, 64), (17, 1001, 131), (58, 640, 2560),
         (64, 129, 65), (65, 129, 65), (128, 128, 128), (200, 96, 40), (300, 515, 1000), (1000, 1536, 520),
         (2049, 2560, 128), (4001, 1304, 264), (6000, 1023, 72), (20000, 256, 192),
         (40, 200, 5000), (150, 1300, 2050), (2049, 2560, 1096), (2500, 2055, 1030)]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("form", [("none", True, False, False, "bf16"), ("gelu_tanh", True, True, True, "f32"),
                                  ("silu", False, False, True, "bf16"), ("gelu_erf", True, False, False, "f32")],
                         ids=lambda f: f[0])
def test_linear(s2lib, gpu_ctx, size, form):
    act, bias, gate, residual, out = form
    m, n, k = size
    a, w, b, gt, res = _case(m * 7 + n, m, n, k, bias=bias, gate=gate, residual=residual, out=out)
    got = s2lib.linear(gpu_ctx, a, w, b, act=oracles.ACTS.index(act), gate=gt, residual=res,
                       out_dtype=s2lib.S2_DTYPE_F32 if out == "f32" else s2lib.S2_DTYPE_BF16)
    assert gpu_ctx.status() == 0
    oracles.check(got, *oracles.linear(a, w, b, act, gt, res, DT[out]), f"{size} {form}")


@pytest.mark.parametrize("rows", [5, 150, 5000])
@pytest.mark.parametrize("shift", [0, 1])
def test_linear_strides_and_alignment(s2lib, gpu_ctx, rows, shift):
    """Padded inputs, an output and a residual inside wider buffers, off 16 bytes with shift 1; what surrounds the
    output stays as it was."""
    n, k = 520, 200
    a, w, b, gt, _ = _case(3, rows, n, k, gate=True, pad=16)
    for dtype, code in ((torch.bfloat16, s2lib.S2_DTYPE_BF16), (torch.float32, s2lib.S2_DTYPE_F32)):
        wide = torch.randn(rows, n + 24, device="cuda", generator=_gen(8)).to(dtype)
        res = torch.randn(rows, n + 40, device="cuda", generator=_gen(9)).to(dtype)[:, shift:n + shift]
        out = wide[:, 8 + shift:8 + shift + n]
        before = wide.clone()
        s2lib.linear(gpu_ctx, a, w, b, act=s2lib.S2_ACT_SILU, gate=gt, residual=res, out=out)
        oracles.check(out, *oracles.linear(a, w, b, "silu", gt, res, dtype))
        before[:, 8 + shift:8 + shift + n] = out
        assert torch.equal(before, wide)
        # in place: the residual is the output
        acc = wide.clone()
        view = acc[:, 8 + shift:8 + shift + n]
        want = oracles.linear(a, w, b, "none", gt, view, dtype)
        s2lib.linear(gpu_ctx, a, w, b, gate=gt, residual=view, out=view)
        oracles.check(view, *want)
        assert torch.equal(acc[:, :8 + shift], wide[:, :8 + shift])
    assert gpu_ctx.status() == 0


@pytest.mark.parametrize("rows", [40, 200, 6000])
def test_linear_nonfinite_rows_stay_apart(s2lib, gpu_ctx, rows):
    a, w, b, _, _ = _case(4, rows, 264, 136)
    bad = a.clone()
    bad[rows // 3, 5] = float("nan")
    bad[rows // 2, 7] = float("inf")
    x, y = s2lib.linear(gpu_ctx, a, w, b), s2lib.linear(gpu_ctx, bad, w, b)
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    keep[rows // 3] = keep[rows // 2] = False
    assert torch.equal(x[keep], y[keep]) and bool(torch.isnan(y[rows // 3]).all())
    assert not bool(torch.isfinite(y[rows // 2]).any())


def test_linear_repeats_bit_for_bit(s2lib, gpu_ctx):
    for rows, n, k in ((1, 2560, 2560), (58, 1280, 2560), (4001, 1304, 264)):
        a, w, b, _, res = _case(5, rows, n, k, residual=True, out="f32")
        first = s2lib.linear(gpu_ctx, a, w, b, residual=res, out_dtype=s2lib.S2_DTYPE_F32)
        for _ in range(5):
            assert torch.equal(first, s2lib.linear(gpu_ctx, a, w, b, residual=res, out_dtype=s2lib.S2_DTYPE_F32))


def test_linear_no_rows(s2lib, gpu_ctx):
    a = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.zeros(16, 64, device="cuda", dtype=torch.bfloat16)
    assert s2lib.linear(gpu_ctx, a, w).shape == (0, 16)
    off = torch.zeros(2, device="cuda", dtype=torch.int32)
    assert s2lib.grouped_linear(gpu_ctx, a, w[None], off).shape == (0, 16)


LAYOUTS = [
    ([0, 1], 1), ([0, 0, 1, 1], 1), ([0, 58, 700], 700), ([3, 3, 20, 20, 21, 37], 50), ([0, 0, 0], 5),
    ([0, 130, 130, 131, 387, 900, 901], 930), ([0, 6000, 6058], 6058), (list(range(0, 130, 2)), 140),
    ([0] + [40] * 63 + [41], 44), ([0] + [300 * i + 7 for i in range(1, 17)], 5000), ([0] * 1024 + [70], 90),
    (list(range(1025)), 1024),
]


@pytest.mark.parametrize("layout", LAYOUTS, ids=lambda v: f"{len(v[0]) - 1}x{v[1]}")
@pytest.mark.parametrize("form", [(136, 200, "gelu_tanh", True, False, False, "bf16"), (1001, 72, "none", True, True, True, "f32"),
                                  (640, 328, "silu", False, False, True, "bf16")], ids=lambda f: f[2])
def test_grouped_linear(s2lib, gpu_ctx, layout, form):
    offsets, rows = layout
    n, k, act, bias, gate, residual, out = form
    groups = len(offsets) - 1
    a, w, b, gt, res = _case(rows + n, rows, n, k, groups=groups, bias=bias, gate=gate, residual=residual, out=out)
    before = torch.randn(rows, n, device="cuda", generator=_gen(2)).to(DT[out])
    got = before.clone()
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    s2lib.grouped_linear(gpu_ctx, a, w, off, b, act=oracles.ACTS.index(act), gate=gt, residual=res, out=got)
    assert gpu_ctx.status() == 0
    oracles.check(got, *oracles.grouped_linear(a, w, offsets, b, act, gt, res, DT[out], before), f"{layout} {form}")


@pytest.mark.parametrize("layout", [([0, 58, 700], 700), ([3, 3, 20, 20, 21, 37], 50), ([0, 130, 130, 131, 387, 900, 901], 930),
                                    ([0, 6000, 6058], 6058), ([0] + [300 * i + 7 for i in range(1, 17)], 5000)],
                         ids=lambda v: f"{len(v[0]) - 1}x{v[1]}")
@pytest.mark.parametrize("n", [640, 643])
def test_grouped_linear_long_sums(s2lib, gpu_ctx, layout, n):
    """fp32 results over more K than one accumulator sums (17 blocks of 64: two sums)."""
    offsets, rows = layout
    a, w, b, gt, res = _case(rows, rows, n, 1030, groups=len(offsets) - 1, gate=True, residual=True, out="f32")
    got = torch.full((rows, n), 2.0, device="cuda")
    before = got.clone()
    s2lib.grouped_linear(gpu_ctx, a, w, torch.tensor(offsets, dtype=torch.int32, device="cuda"), b,
                         act=s2lib.S2_ACT_GELU_ERF, gate=gt, residual=res, out=got)
    assert gpu_ctx.status() == 0
    oracles.check(got, *oracles.grouped_linear(a, w, offsets, b, "gelu_erf", gt, res, torch.float32, before))


@pytest.mark.parametrize("rows", [1, 40, 300, 2500])
def test_fp32_results_keep_their_precision(s2lib, gpu_ctx, rows):
    """K = 10,240 without a residual: the 2-norm of the error stays at 2e-6 of the result's (sums of 14 blocks of 64
    lose some 6e-8 a block, whatever K is; one sum of 160 blocks lost 1.1e-5)."""
    a, w, _, _, _ = _case(9, rows, 384, 10240, bias=False, out="f32")
    got = s2lib.linear(gpu_ctx, a, w, out_dtype=s2lib.S2_DTYPE_F32).double()
    want = a.double() @ w.double().t()
    assert float((got - want).norm() / want.norm()) < 2e-6


def test_linear_captured(s2lib, gpu_ctx):
    """Each kernel of the product in one graph, replayed on other values."""
    cases = [_case(30 + i, *size, residual=True, out="f32") for i, size in enumerate(
        ((3, 260, 520), (200, 640, 1400), (5000, 640, 1400), (5000, 643, 200)))]
    outs = [torch.zeros_like(c[4]) for c in cases]
    run = lambda: [s2lib.linear(gpu_ctx, c[0], c[1], c[2], residual=c[4], out=o) for c, o in zip(cases, outs)]  # noqa: E731
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    home = gpu_ctx.stream
    with torch.cuda.graph(graph):
        gpu_ctx.set_stream(torch.cuda.current_stream())
        run()
    gpu_ctx.set_stream(home)
    for c in cases:
        c[4].mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    got = [o.clone() for o in outs]
    run()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, outs))
    del graph


@pytest.mark.parametrize("rows", [30, 4000])
def test_grouped_linear_bad_offsets_stay_inside(s2lib, gpu_ctx, rows):
    """Offsets out of range or order are clamped in the kernel: rows past the buffer are not written, the status
    says so and the context goes on working."""
    n, k, groups = 256, 64, 3
    a, w, b, _, _ = _case(6, rows, n, k, groups=groups)
    whole = torch.zeros(rows + 600, n, device="cuda", dtype=torch.bfloat16)
    for offsets in ([-5, 10, 20, rows], [0, 10, 2**31 - 1, 2**31 - 1], [0, rows, 5, rows], [-2**31, -1, rows + 500, 3]):
        off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
        s2lib.grouped_linear(gpu_ctx, a, w, off, b, out=whole[:rows])
        assert gpu_ctx.status() == s2lib.S2_ERR_INVALID, offsets
        assert not bool(whole[rows:].any())
    off = torch.tensor([0, 10, 20, rows], dtype=torch.int32, device="cuda")
    got = s2lib.grouped_linear(gpu_ctx, a, w, off, b)
    assert gpu_ctx.status() == 0
    oracles.check(got, *oracles.grouped_linear(a, w, off.tolist(), b, "none", None, None, torch.bfloat16, got))


def test_grouped_linear_reads_offsets_when_it_runs(s2lib, gpu_ctx):
    """Captured once, replayed with other offsets and other rows in the same buffers."""
    rows, n, k, groups = 600, 192, 128, 4
    a, w, b, _, _ = _case(7, rows, n, k, groups=groups)
    off = torch.tensor([0, 100, 100, 300, 600], dtype=torch.int32, device="cuda")
    out = torch.zeros(rows, n, device="cuda", dtype=torch.bfloat16)
    few = torch.zeros(20, n, device="cuda", dtype=torch.bfloat16)
    few_off = torch.tensor([0, 5, 9, 9, 20], dtype=torch.int32, device="cuda")
    s2lib.grouped_linear(gpu_ctx, a, w, off, b, out=out)  # first use outside the capture
    s2lib.grouped_linear(gpu_ctx, a[:20], w, few_off, b, out=few)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    home = gpu_ctx.stream
    with torch.cuda.graph(graph):
        gpu_ctx.set_stream(torch.cuda.current_stream())
        s2lib.grouped_linear(gpu_ctx, a, w, off, b, out=out)
        s2lib.grouped_linear(gpu_ctx, a[:20], w, few_off, b, out=few)
    gpu_ctx.set_stream(home)
    for offsets, small in (([0, 1, 2, 3, 600], [0, 0, 20, 20, 20]), ([50, 180, 400, 400, 599], [1, 2, 3, 4, 5])):
        off.copy_(torch.tensor(offsets, dtype=torch.int32))
        few_off.copy_(torch.tensor(small, dtype=torch.int32))
        a.copy_(torch.randn(rows, k, device="cuda").bfloat16())
        out.fill_(3)
        few.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        three = torch.full((rows, n), 3.0, device="cuda")
        oracles.check(out, *oracles.grouped_linear(a, w, offsets, b, "none", None, None, torch.bfloat16, three))
        oracles.check(few, *oracles.grouped_linear(a[:20], w, small, b, "none", None, None, torch.bfloat16, three[:20]))
    del graph


def test_two_contexts_on_two_streams(s2lib, gpu_ctx):
    """Calls in flight at once on two streams do not share anything."""
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    ctxs = [s2lib.Context(0, s) for s in streams]
    cases = [_case(20 + i, rows, 640, 520) for i, rows in enumerate((3000, 40))]
    wants = [s2lib.linear(gpu_ctx, c[0], c[1], c[2]) for c in cases]
    torch.cuda.synchronize()
    outs = [[torch.zeros_like(wants[i]) for _ in range(4)] for i in range(2)]
    torch.cuda.synchronize()
    for j in range(4):
        for i in range(2):
            s2lib.linear(ctxs[i], cases[i][0], cases[i][1], cases[i][2], out=outs[i][j])
    for i in range(2):
        assert ctxs[i].status() == 0
        assert all(torch.equal(o, wants[i]) for o in outs[i])
        ctxs[i].close()


def test_memory_of_a_call_on_another_stream(s2lib, gpu_ctx):
    """The memory that a call on its own stream gets is not one that torch's current stream has yet to write to."""
    a, w, b, _, _ = _case(7, 900, 640, 520)
    x = torch.randn(2, 20000, 128, device="cuda").bfloat16()
    want, want_norm = s2lib.linear(gpu_ctx, a, w, b), s2lib.group_norm(gpu_ctx, x, 32)
    need = s2lib.lib().s2_group_norm_workspace(2, 20000, 128, 32)
    assert need > 0
    stream = torch.cuda.Stream()
    ctx = s2lib.Context(0, stream)
    torch.cuda.synchronize()
    for _ in range(2):
        torch.cuda._sleep(20_000_000)
        for like in (want, want_norm):
            torch.full_like(like, 7)
        torch.full((need,), 255, dtype=torch.uint8, device="cuda")  # all three freed with their writes to come
        y, y_norm = s2lib.linear(ctx, a, w, b), s2lib.group_norm(ctx, x, 32)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(y_norm, want_norm)
        del y, y_norm
    assert ctx.status() == 0
    ctx.close()


def test_wrapper_refuses(s2lib, gpu_ctx):
    a, w, b, _, _ = _case(1, 8, 16, 16)
    bad = [lambda: s2lib.linear(gpu_ctx, a.float(), w), lambda: s2lib.linear(gpu_ctx, a, w.float()),
           lambda: s2lib.linear(gpu_ctx, a, w[:, :8]), lambda: s2lib.linear(gpu_ctx, a.cpu(), w),
           lambda: s2lib.linear(gpu_ctx, a, w, b.bfloat16()), lambda: s2lib.linear(gpu_ctx, a, w, b[:8]),
           lambda: s2lib.linear(gpu_ctx, a.t(), w[:, :8]), lambda: s2lib.linear(gpu_ctx, a, w, act=9),
           lambda: s2lib.linear(gpu_ctx, a, w, residual=torch.zeros(8, 16, device="cuda")),
           lambda: s2lib.linear(gpu_ctx, a, w, out=torch.zeros(8, 15, device="cuda")),
           lambda: s2lib.grouped_linear(gpu_ctx, a, w[None], torch.tensor([0, 8], device="cuda")),
           lambda: s2lib.grouped_linear(gpu_ctx, a, w[None], torch.tensor([0], dtype=torch.int32, device="cuda"))]
    for call in bad:
        with pytest.raises(s2lib.S2Error) as e:
            call()
        assert e.value.code == s2lib.S2_ERR_INVALID
    # the library's own check through the C ABI: a stride off 8
    e = s2lib.LinearEpilogue()
    out = torch.zeros(8, 16, device="cuda", dtype=torch.bfloat16)
    assert s2lib.lib().s2_linear(gpu_ctx.handle, 8, 16, 16, a.data_ptr(), 20, w.data_ptr(), 16, C.byref(e),
                                 s2lib.S2_DTYPE_BF16, out.data_ptr(), 16) == s2lib.S2_ERR_INVALID
