"""CPU: a result's type is one of the library's, or the call is refused (a torch type among them: it would be taken for
another number)."""
import ctypes as C

import pytest
import torch

from tests.test_operator_lifetimes import BASE, _Sized

BAD = [torch.float32, torch.bfloat16, torch.float16, 2, -1, "f32"]


@pytest.fixture()
def made(s2lib, monkeypatch):
    """The types that the calls allocate; the library is not reached."""
    types = []

    def new(ctx, shape, dtype):
        types.append(dtype)
        return _Sized((shape,) if isinstance(shape, int) else shape, dtype, BASE * 8)

    class Library:
        def __getattr__(self, name):
            return lambda *args: b"refused" if name == "s2_error_string" else 0

    monkeypatch.setattr(s2lib, "_new", new)
    monkeypatch.setattr(s2lib, "lib", Library)
    return types


class _Ctx:
    device, handle = -1, C.c_void_p()


def _calls(s2lib):
    bf16 = lambda *shape: _Sized(shape, torch.bfloat16, BASE)  # noqa: E731
    return {"linear": lambda **kw: s2lib.linear(_Ctx, bf16(4, 16), bf16(8, 16), **kw),
            "grouped": lambda **kw: s2lib.grouped_linear(_Ctx, bf16(4, 16), bf16(2, 8, 16), _Sized((3,), torch.int32, BASE), **kw),
            "norm": lambda **kw: s2lib.group_norm(_Ctx, bf16(2, 5, 32), 4, **kw)}


@pytest.mark.parametrize("call", ["linear", "grouped", "norm"])
def test_known_types(s2lib, made, call):
    f = _calls(s2lib)[call]
    assert f(out_dtype=s2lib.S2_DTYPE_F32).dtype == torch.float32
    assert f(out_dtype=s2lib.S2_DTYPE_BF16).dtype == torch.bfloat16
    assert f().dtype == torch.bfloat16
    assert made == [torch.float32, torch.bfloat16, torch.bfloat16]


@pytest.mark.parametrize("call", ["linear", "grouped", "norm"])
@pytest.mark.parametrize("bad", BAD, ids=str)
def test_others_are_refused(s2lib, made, call, bad):
    with pytest.raises(s2lib.S2Error) as e:
        _calls(s2lib)[call](out_dtype=bad)
    assert e.value.code == s2lib.S2_ERR_INVALID and not made
