"""What orthogonalising takes besides its operands: nothing for matrices that one launch takes through all steps."""
import ctypes as C

import numpy as np
import pytest

from tests.util import assert_bit_equal

pytestmark = pytest.mark.gpu


class _Allocator(C.Structure):
    _fields_ = [("malloc", C.c_void_p), ("realloc", C.c_void_p), ("free", C.c_void_p), ("emptyCache", C.CFUNCTYPE(C.c_int, C.c_void_p)),
                ("cacheInfo", C.c_void_p), ("state", C.c_void_p)]


def _free():
    """The device's own free memory, without blocks that are parked."""
    hip = C.CDLL("libamdhip64.so")
    free, total = C.c_size_t(0), C.c_size_t(0)
    assert hip.hipMemGetInfo(C.byref(free), C.byref(total)) == 0
    return free.value


@pytest.mark.parametrize("rows,cols", [(40, 60), (60, 40), (128, 128)])
def test_matrices_of_one_launch_take_no_workspace(thc, rows, cols):
    rng = np.random.default_rng(rows)
    one = rng.standard_normal((rows, cols)).astype(np.float32)
    t = thc.Tensor.from_numpy
    want = thc.Tensor("float").orthogonalize(t(one)).numpy()
    count = (1 << 28) // (rows * cols * 4)
    many = thc.Tensor("float").resize((count, rows, cols))
    many.copy(t(one).view_as_strided(0, (count, rows, cols), (0, cols, 1)))
    thc.synchronize()
    cache = C.cast(thc.lib().THCCachingAllocator_get(), C.POINTER(_Allocator)).contents
    assert cache.emptyCache(cache.state) == 0
    before = _free()
    many.orthogonalize(many)
    thc.synchronize()
    # what it had taken would be parked now
    assert before - _free() <= 64 << 20
    got = many.numpy()
    assert_bit_equal(got[0], want)
    assert_bit_equal(got[-1], want)
