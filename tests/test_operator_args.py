"""CPU: the argument checks of s2_linear, s2_grouped_linear and s2_group_norm
come before anything touches the context or a device, so they are driven here
with addresses that are never followed; a call they accept goes on to select
the device and, without one, returns the CUDA error."""
import ctypes as C

import pytest
import torch

from tests import operator_oracles as oracles

BASE = 1 << 20  # an aligned address
OUT = 1 << 24


@pytest.fixture()
def ctx():
    if torch.cuda.is_available():
        pytest.skip("for machines without a GPU")
    return C.create_string_buffer(1 << 16)


def _linear(s2lib, ctx, *, M=4, N=16, K=16, A=BASE, lda=16, W=BASE, ldw=16, act=0, bias=None, gate=None, residual=None,
            residual_ld=16, dtype=1, out=OUT, ldo=16, groups=None, offsets=None):
    e = s2lib.LinearEpilogue(act, bias, gate, residual, residual_ld)
    if groups is None:
        return s2lib.lib().s2_linear(ctx, M, N, K, A, lda, W, ldw, C.byref(e), dtype, out, ldo)
    return s2lib.lib().s2_grouped_linear(ctx, M, groups, offsets, N, K, A, lda, W, ldw, C.byref(e), dtype, out, ldo)


BAD_LINEAR = [
    {"M": -1}, {"N": 0}, {"N": -8}, {"K": 0}, {"A": None}, {"W": None}, {"out": None}, {"lda": 8}, {"ldw": 8}, {"ldo": 15},
    {"lda": 20}, {"ldw": 20}, {"A": BASE + 2}, {"W": BASE + 8}, {"out": OUT + 1}, {"out": OUT + 2, "dtype": 0},
    {"act": -1}, {"act": 4}, {"dtype": 2}, {"dtype": -1}, {"bias": BASE + 2}, {"gate": BASE + 1},
    {"residual": OUT + 1}, {"residual": BASE, "residual_ld": 8}, {"residual": OUT, "residual_ld": 24},
    {"M": 2**31 - 1},
]


@pytest.mark.parametrize("bad", BAD_LINEAR, ids=str)
def test_linear_refuses(s2lib, ctx, bad):
    assert _linear(s2lib, ctx, **bad) == s2lib.S2_ERR_INVALID
    assert _linear(s2lib, ctx, groups=2, offsets=BASE, **bad) == s2lib.S2_ERR_INVALID


def test_grouped_linear_refuses(s2lib, ctx):
    for bad in ({"groups": 0}, {"groups": -1}, {"groups": 1025}, {"offsets": None}, {"offsets": BASE + 2},
                {"N": 2**24, "ldo": 2**24, "groups": 512}):
        args = {"groups": 2, "offsets": BASE, **bad}
        assert _linear(s2lib, ctx, **args) == s2lib.S2_ERR_INVALID, bad


def test_linear_accepts(s2lib, ctx):
    for good in ({}, {"N": 15, "ldo": 15, "out": OUT + 2}, {"K": 11}, {"residual": OUT}, {"residual": BASE + 2},
                 {"bias": BASE + 4, "gate": BASE + 4}, {"groups": 1024, "offsets": BASE + 4}):
        assert _linear(s2lib, ctx, **good) == s2lib.S2_ERR_CUDA, good
    assert _linear(s2lib, ctx, M=0) == s2lib.S2_OK
    assert s2lib.lib().s2_linear(ctx, 4, 16, 16, BASE, 16, BASE, 16, None, 1, OUT, 16) == s2lib.S2_ERR_CUDA
    assert s2lib.lib().s2_linear(None, 4, 16, 16, BASE, 16, BASE, 16, None, 1, OUT, 16) == s2lib.S2_ERR_INVALID


def _norm(s2lib, ctx, *, instances=2, rows=5, channels=32, groups=4, in_dtype=1, x=BASE, ldx=32, gamma=None, beta=None,
          eps=1e-6, act=0, out_dtype=1, out=OUT, ldo=32, ws=1 << 28, ws_bytes=1 << 30):
    return s2lib.lib().s2_group_norm(ctx, instances, rows, channels, groups, in_dtype, x, ldx, gamma, beta, eps, act,
                                     out_dtype, out, ldo, ws, ws_bytes)


BAD_NORM = [
    {"instances": -1}, {"rows": -1}, {"rows": 2**30 + 1}, {"channels": 0}, {"groups": 0}, {"groups": 5}, {"groups": 64},
    {"ldx": 31}, {"ldo": 31}, {"x": None}, {"out": None}, {"x": BASE + 1}, {"x": BASE + 2, "in_dtype": 0},
    {"out": OUT + 1}, {"out": OUT + 2, "out_dtype": 0}, {"in_dtype": 2}, {"out_dtype": -1}, {"act": 4}, {"act": -1},
    {"eps": -1.0}, {"eps": float("nan")}, {"gamma": BASE + 2}, {"beta": BASE + 1}, {"out": BASE, "out_dtype": 0},
    {"out": BASE, "ldo": 40}, {"channels": 65568, "ldx": 65568, "ldo": 65568}, {"ws": (1 << 28) + 4},
    {"rows": 10**6, "ws": None}, {"rows": 10**6, "ws_bytes": 8},
]


@pytest.mark.parametrize("bad", BAD_NORM, ids=str)
def test_group_norm_refuses(s2lib, ctx, bad):
    assert _norm(s2lib, ctx, **bad) == s2lib.S2_ERR_INVALID


def test_group_norm_accepts(s2lib, ctx):
    for good in ({}, {"out": BASE}, {"x": BASE + 2, "out": OUT + 6}, {"groups": 32}, {"groups": 1}, {"eps": 0.0},
                 {"gamma": BASE + 4, "beta": BASE + 8}, {"in_dtype": 0}, {"out_dtype": 0}):
        assert _norm(s2lib, ctx, **good) == s2lib.S2_ERR_CUDA, good
    for empty in ({"instances": 0}, {"rows": 0}):
        assert _norm(s2lib, ctx, **empty) == s2lib.S2_OK


def test_group_norm_workspace(s2lib, ctx):
    size = s2lib.lib().s2_group_norm_workspace
    assert size(1, 256, 512, 32) == 0 and size(0, 5, 8, 1) == 0 and size(1, 5, 8, 3) == 0
    assert _norm(s2lib, ctx, ws=None, ws_bytes=0) == s2lib.S2_ERR_CUDA, "small x needs none"
    for shape in ((6, 14400, 512, 32), (1, 10**9, 8, 8), (1000, 3, 4096, 4096), (70000, 1, 32, 1)):
        i, r, c, g = shape
        need = size(*shape)
        assert need % 8 == 0 and 8 * i * g <= need <= 8 * g * max(i, 444)
        args = dict(instances=i, rows=r, channels=c, groups=g, ldx=c, ldo=c)
        assert _norm(s2lib, ctx, ws_bytes=need, **args) == s2lib.S2_ERR_CUDA
        assert _norm(s2lib, ctx, ws_bytes=need - 1, **args) == s2lib.S2_ERR_INVALID


def test_row_strides(s2lib):
    stride = lambda t: s2lib._row_stride(t, "t")  # noqa: E731
    assert stride(torch.empty(3, 4, 5, 8)) == 8
    assert stride(torch.empty(3, 4, 16)[:, :, :8]) == 16
    assert stride(torch.empty(1, 1, 8)) == 8
    assert stride(torch.empty(4, 1, 8)) == 8
    assert stride(torch.empty(2, 0, 16)) == 16 and stride(torch.empty(0, 5, 16)) == 16
    for bad in (torch.empty(3, 8, 4).transpose(1, 2), torch.empty(3, 6, 8)[:, :4], torch.empty(3, 4, 16)[:, :, ::2]):
        with pytest.raises(s2lib.S2Error):
            stride(bad)


def test_operand_strides(s2lib):
    stride = lambda t: s2lib._operand_stride(t, t.shape, -1, "t")  # noqa: E731
    rows = lambda *shape: torch.empty(shape, dtype=torch.bfloat16)  # noqa: E731
    assert stride(rows(4, 16)) == 16 and stride(rows(4, 24)[:, :13]) == 24
    assert stride(rows(1, 13)) == 16 and stride(rows(4, 24)[2:3, :13]) == 16, "a row of its own has no stride"
    assert stride(rows(0, 13)) == 16 and stride(rows(4, 24)[:0, :13]) == 16, "nor have no rows"
    assert stride(rows(3, 1)[:1]) == 8
    for bad in (rows(13, 4).t()[:1], rows(1, 26)[:, ::2], rows(4, 26)[:, ::2]):
        with pytest.raises(s2lib.S2Error):
            stride(bad)


class _Sized:
    """The size of a tensor and an address that is never followed."""

    def __init__(self, shape, dtype, address):
        self.meta, self.address = torch.empty(shape, dtype=dtype, device="meta"), address
        self.shape, self.dtype = self.meta.shape, dtype

    def __getattr__(self, name):
        return getattr(self.meta, name)

    def get_device(self):
        return -1

    def data_ptr(self):
        return self.address


def test_wrappers_refuse_what_a_c_int_does_not_hold(s2lib, ctx):
    class Ctx:
        handle, device = ctx, -1

    bf16 = lambda shape, at: _Sized(shape, torch.bfloat16, at)  # noqa: E731

    def linear(m, n, k):
        s2lib.linear(Ctx, bf16((m, k), BASE), bf16((n, k), BASE), out=bf16((m, n), OUT))

    def norm(instances, groups, channels=32):
        x = bf16((instances, 5, channels), BASE)
        s2lib.group_norm(Ctx, x, groups, out=bf16(x.shape, OUT))

    for call, good, bad in ((linear, (5, 16, 16), [(2**32 + 5, 16, 16), (5, 2**32 + 16, 16), (5, 16, 2**32 + 16)]),
                            (norm, (2, 4), [(2**32 + 2, 4), (2, 2**32 + 4), (2, 4, 2**32 + 32), (2, 0), (2, -4)])):
        with pytest.raises(s2lib.S2Error) as e:
            call(*good)
        assert e.value.code == s2lib.S2_ERR_CUDA
        for args in bad:
            with pytest.raises(s2lib.S2Error) as e:
                call(*args)
            assert e.value.code == s2lib.S2_ERR_INVALID, args


def test_oracles_agree_with_torch():
    """The 64-bit restatements against torch's own layers."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 7, 12, generator=g, dtype=torch.float64) * 3 + 1
    gamma, beta = torch.randn(12, generator=g, dtype=torch.float64), torch.randn(12, generator=g, dtype=torch.float64)
    y, bound = oracles.group_norm(x, 4, gamma, beta, 1e-5, "silu", torch.float32)
    want = torch.nn.functional.silu(torch.nn.functional.group_norm(x.transpose(1, 2), 4, gamma, beta, 1e-5)).transpose(1, 2)
    assert torch.allclose(y, want, rtol=1e-12, atol=1e-12) and float(bound.max()) < 1e-4
    v = torch.linspace(-12, 12, 97, dtype=torch.float64)
    assert torch.allclose(oracles.activate(v, "gelu_tanh")[0], torch.nn.functional.gelu(v, approximate="tanh"), atol=1e-12)
    assert torch.allclose(oracles.activate(v, "gelu_erf")[0], torch.nn.functional.gelu(v), atol=1e-12)
    # a mistake of one part in a thousand in the oracle's input is outside the bound
    a, w = torch.randn(5, 40, generator=g), torch.randn(6, 40, generator=g)
    y, bound = oracles.linear(a, w, None, "none", None, None, torch.float32)
    oracles.check((a.double() @ w.double().t()).float(), y, bound)
    with pytest.raises(AssertionError):
        oracles.check((a.double() @ w.double().t() * 1.001).float(), y, bound)
