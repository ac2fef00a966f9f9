"""Lists of tensors as the entry points take them: addresses side by side."""
import ctypes

import pytest


class _Stub(object):
    def __init__(self, kind, a):
        self.kind, self.a = kind, a


def test_addresses_of_a_list():
    _fastcall = pytest.importorskip("cutorch_amd._fastcall")
    stubs = [_Stub("float", 16 * i + 2 ** 47) for i in range(300)] + [_Stub("float", 2 ** 64 - 8)]
    for these in (stubs, tuple(stubs), iter(stubs)):
        held, where = _fastcall.addresses(these, "float")
        assert len(held) == 8 * len(stubs)
        assert list((ctypes.c_uint64 * len(stubs)).from_address(where)) == [s.a for s in stubs]
    assert len(_fastcall.addresses([], "float")[0]) == 0
    assert len(_fastcall.addresses(stubs, "".join(["flo", "at"]))[0]) == 8 * len(stubs)      # equal, not the same object


def test_addresses_refuses():
    _fastcall = pytest.importorskip("cutorch_amd._fastcall")
    with pytest.raises(ValueError, match="another type than half"):
        _fastcall.addresses([_Stub("half", 8), _Stub("float", 16)], "half")
    with pytest.raises(AttributeError):
        _fastcall.addresses([3], "half")
    for bad in ((3, "half"), ([],), ([_Stub("half", "8")], "half")):
        with pytest.raises(TypeError):
            _fastcall.addresses(*bad)
    with pytest.raises(OverflowError):
        _fastcall.addresses([_Stub("half", -1)], "half")
