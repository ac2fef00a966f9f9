"""A list of tensors that changes while its addresses are taken."""
import ctypes

import pytest


def test_addresses_of_a_list_that_is_emptied():
    _fastcall = pytest.importorskip("cutorch_amd._fastcall")
    stubs = []

    class _Stub(object):
        a = 16

        @property
        def kind(self):
            del stubs[:]
            return "float"

    stubs.extend(_Stub() for _ in range(50))
    held, where = _fastcall.addresses(stubs, "float")
    assert stubs == [] and list((ctypes.c_uint64 * 50).from_address(where)) == [16] * 50 and len(held) == 400
