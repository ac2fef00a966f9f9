"""The binding's calls of a decoder's operators and of the optimizer of matrices, without a GPU."""
import ctypes

import pytest

import cutorch_amd as thc


def test_fast_calls_serve_the_entry_points():
    _fastcall = pytest.importorskip("cutorch_amd._fastcall")
    lib = thc.lib()
    names = [T + name for T in ("THCudaTensor_", "THCudaHalfTensor_") for name in ("layerNorm", "layerNormGrad", "rotary", "orthogonalize", "muon")]
    for name in names + ["THCudaDoubleTensor_rotaryFrequencies"]:
        f = getattr(lib, name)
        signature = "".join(thc._CODES.get(t, "?") for t in [f.restype] + list(f.argtypes[1:]))
        assert _fastcall.bind(ctypes.cast(f, ctypes.c_void_p).value, signature, 0) is not None, (name, signature)


class _Stub(object):
    def __init__(self, kind, a, shape=(2, 2)):
        self.kind, self.a, self.shape = kind, a, shape


def test_lists_of_the_optimizer():
    p, g, m = [_Stub("float", 16), _Stub("float", 32)], [_Stub("float", 48), _Stub("float", 64)], [_Stub("float", 80), _Stub("float", 96)]
    opt = thc.Muon(iter(p), g, momentum=m)
    assert opt.params == tuple(p) and opt.grads == tuple(g) and opt.momentum == tuple(m) and opt.master is None
    assert [list((ctypes.c_uint64 * 2).from_address(a)) for a in opt._args] == [[16, 32], [48, 64], [80, 96]]
    other = [_Stub("float", 112), _Stub("float", 128)]
    opt.grads = other
    assert opt.grads == tuple(other) and list((ctypes.c_uint64 * 2).from_address(opt._args[1])) == [112, 128]
    for name, bad, match in (("grads", p[:1], "1 tensors for 2 parameters"), ("grads", [_Stub("half", 1), _Stub("float", 2)], "another type"),
                             ("master", p, "have no master"), ("momentum", [_Stub("half", 1)] * 2, "another type")):
        with pytest.raises(ValueError, match=match):
            setattr(opt, name, bad)
    assert opt.grads == tuple(other) and opt.momentum == tuple(m)
    half = [_Stub("half", 16)]
    opt = thc.Muon(half, half, master=[_Stub("float", 32)], momentum=[_Stub("float", 48)])
    assert [list((ctypes.c_uint64 * 1).from_address(a)) for a in opt._args] == [[16], [32], [16], [48]]
    opt.master = None
    assert opt._args[1] == 0 and opt.master is None
    with pytest.raises(ValueError, match="all float or all half"):
        thc.Muon([_Stub("float", 1), _Stub("half", 2)], [])
    with pytest.raises(ValueError, match="copies are of half"):
        thc.Muon(p, g, master=p, momentum=m)
