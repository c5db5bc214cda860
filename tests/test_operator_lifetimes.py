"""CPU: what a call was given stays alive until the library has been called, even where the caller keeps no other
reference to it (a tensor cast in the call's own expression)."""
import ctypes as C
import weakref

import pytest
import torch

BASE = 1 << 20  # an aligned address, never followed


class _Sized:
    """The size of a tensor and an address; where it still lives is seen through a weak reference."""

    def __init__(self, shape, dtype, address, seen=None):
        self.meta, self.address = torch.empty(shape, dtype=dtype, device="meta"), address
        self.shape, self.dtype = self.meta.shape, dtype
        if seen is not None:
            seen.append(weakref.ref(self))

    def __getattr__(self, name):
        return getattr(self.meta, name)

    def get_device(self):
        return -1

    def data_ptr(self):
        return self.address


class _Ctx:
    device = -1


@pytest.fixture()
def ctx(s2lib, monkeypatch):
    if torch.cuda.is_available():
        pytest.skip("for machines without a GPU")
    _Ctx.handle = C.create_string_buffer(1 << 16)
    return _Ctx


def test_group_norm_keeps_its_vectors(s2lib, ctx, monkeypatch):
    """The workspace is allocated after gamma and beta were checked: their memory must not be free by then."""
    seen, alive = [], []

    def new(ctx, shape, dtype):
        alive.append([r() is not None for r in seen])
        return _Sized((shape,) if isinstance(shape, int) else shape, dtype, BASE * 64)

    monkeypatch.setattr(s2lib, "_new", new)
    shape = (2, 30000, 64)
    assert s2lib.lib().s2_group_norm_workspace(2, 30000, 64, 32) > 0
    with pytest.raises(s2lib.S2Error) as e:  # accepted, then no device
        s2lib.group_norm(ctx, _Sized(shape, torch.float32, BASE, seen), 32, _Sized((64,), torch.float32, BASE * 2, seen),
                         _Sized((64,), torch.float32, BASE * 3, seen))
    assert e.value.code == s2lib.S2_ERR_CUDA
    assert alive == [[True] * 3] * 2, "output, then workspace"


@pytest.mark.parametrize("grouped", [False, True])
def test_linear_keeps_its_operands(s2lib, ctx, monkeypatch, grouped):
    seen, alive = [], []
    bf16, f32 = torch.bfloat16, torch.float32
    lead = (3,) if grouped else ()

    class Library:
        def __getattr__(self, name):
            alive.append([r() is not None for r in seen])
            return lambda *args: s2lib.S2_OK

    monkeypatch.setattr(s2lib, "lib", Library)
    call = s2lib.grouped_linear if grouped else s2lib.linear
    offsets = (_Sized((4,), torch.int32, BASE, seen),) if grouped else ()
    call(ctx, _Sized((5, 16), bf16, BASE, seen), _Sized((*lead, 24, 16), bf16, BASE, seen), *offsets,
         _Sized((*lead, 24), f32, BASE, seen), gate=_Sized((*lead, 24), f32, BASE, seen),
         residual=_Sized((5, 24), bf16, BASE, seen), out=_Sized((5, 24), bf16, BASE, seen))
    assert alive == [[True] * (7 if grouped else 6)]
