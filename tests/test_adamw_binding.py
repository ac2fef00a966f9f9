"""The optimizer's lists of tensors on the host, with stand-ins for tensors and entry points: what a step is given, and that it is alive."""
import ctypes
import gc
import weakref

import pytest

import cutorch_amd as thc


class _Stub(object):
    """What the optimizer asks of a tensor."""

    def __init__(self, kind="float", shape=(4,)):
        self.kind, self.shape, self.address = kind, shape, id(self)
        self.a = self.address

    def numel(self):
        return self.shape[0]

    def resize(self, shape):
        self.shape = shape
        return self

    def zero(self):
        return self


@pytest.fixture
def made(monkeypatch):
    """Steps and moments as (entry point, addresses by list): nothing is called."""
    calls = []

    def entry(name):
        def call(count, *args):
            lists = [a for a in args if isinstance(a, int) and a > 1 << 20]
            calls.append((name, [list((ctypes.c_uint64 * count).from_address(a)) for a in lists]))
        return call

    class _Entries(dict):
        def __missing__(self, name):
            return entry(name)

    monkeypatch.setattr(thc, "Tensor", _Stub)
    monkeypatch.setattr(thc, "_CALLS", {kind: _Entries() for kind in ("float", "half")})
    return calls


def test_a_replaced_list_reaches_the_step(made):
    opt = thc.AdamW([_Stub(), _Stub()], [_Stub(), _Stub()])
    opt.step()
    assert made[-1] == ("adamW", [[t.a for t in l] for l in (opt.params, opt.grads, opt.mean, opt.square)])
    for name in ("grads", "mean", "square", "params"):
        new = [_Stub(), _Stub()]
        setattr(opt, name, new)
        opt.step()
        assert made[-1] == ("adamW", [[t.a for t in l] for l in (opt.params, opt.grads, opt.mean, opt.square)])
        assert [t.a for t in new] in made[-1][1]
    opt = thc.AdamW([_Stub("half")], [_Stub("half")], master=[_Stub()], bits=8)
    for name, kind in (("master", "float"), ("mean", "char"), ("mean_scale", "float"), ("square", "byte"), ("square_scale", "float")):
        setattr(opt, name, [_Stub(kind)])
        opt.step()
        assert made[-1] == ("adamW8", [[t.a for t in l] for l in (opt.params, opt.master, opt.grads, opt.mean, opt.mean_scale, opt.square,
                                                                 opt.square_scale)])
    opt.master = None          # from now on the halves themselves are stepped
    opt.step()
    assert len(made[-1][1]) == 6 and opt.master is None


def test_what_a_step_is_given_is_alive(made):
    opt = thc.AdamW([_Stub()], [_Stub()])
    seen = weakref.ref(opt.grads[0])
    with pytest.raises(TypeError):
        opt.grads[0] = _Stub()
    with pytest.raises(AttributeError):
        opt.grads.append(_Stub())
    gc.collect()
    opt.step()
    assert seen() is not None and made[-1][1][1] == [seen().a]
    opt.grads = [_Stub()]
    gc.collect()
    assert seen() is None
    # lists that the caller goes on using are the caller's
    mine = [_Stub()]
    opt.grads = mine
    seen = weakref.ref(mine[0])
    mine[0] = _Stub()
    gc.collect()
    opt.step()
    assert seen() is not None and made[-1][1][1] == [seen().a]


def test_a_list_that_does_not_fit_changes_nothing(made):
    opt = thc.AdamW([_Stub()], [_Stub()])
    held = opt.grads
    for name, bad in (("grads", [_Stub("half")]), ("grads", []), ("grads", [_Stub(), _Stub()]), ("params", [_Stub("half")]), ("params", []),
                      ("mean", [_Stub("char")]), ("master", [_Stub()]), ("mean_scale", [_Stub()]), ("square_scale", [_Stub()])):
        with pytest.raises(ValueError):
            setattr(opt, name, bad)
    with pytest.raises(TypeError):
        opt.grads = None
    opt.step()
    assert opt.grads is held and made[-1] == ("adamW", [[t.a for t in l] for l in (opt.params, opt.grads, opt.mean, opt.square)])


def test_parameters_may_come_from_a_generator(made):
    opt = thc.AdamW((p for p in [_Stub("half"), _Stub("half")]), (g for g in [_Stub("half"), _Stub("half")]))
    assert len(opt.params) == 2 and opt.kind == "half"
    opt.step()
    assert len(made[-1][1][0]) == 2


@pytest.mark.parametrize("bits,names", [(32, ("mean", "square")), (8, ("mean", "mean_scale", "square", "square_scale"))])
def test_an_earlier_run_is_resumed_with_all_its_states(made, bits, names):
    kinds = {"mean": "char" if bits == 8 else "float", "square": "byte" if bits == 8 else "float", "mean_scale": "float", "square_scale": "float"}
    for some in range(2 ** len(names)):
        states = {n: [_Stub(kinds[n])] for i, n in enumerate(names) if some >> i & 1}
        if len(states) == len(names):
            opt = thc.AdamW([_Stub()], [_Stub()], bits=bits, step=3, **states)
            assert opt.steps == 3 and all(getattr(opt, n) == tuple(states[n]) for n in names)
        else:
            with pytest.raises(ValueError, match="without all of"):
                thc.AdamW([_Stub()], [_Stub()], bits=bits, step=3, **states)
        # before the first step all of them are zeros, whoever makes them
        assert thc.AdamW([_Stub()], [_Stub()], bits=bits, **states).steps == 0
