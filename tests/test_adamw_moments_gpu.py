"""The outputs of adamW8Moments on shared storages, across tensors: side by side and in gaps they are what they are apart, on another
tensor's scales or outputs they are refused."""
import numpy as np
import pytest

from tests.test_adamw_gpu import HYPER, _problem, _put
from tests.util import assert_bit_equal

pytestmark = pytest.mark.gpu
SIZES = [(300,), (7, 100), (300,), (5,)]


def _stepped(thc, scales=None):
    """An optimizer after a step; `scales` takes a list of scales to the tensors that hold them."""
    p, g = _problem(np.random.default_rng(9), SIZES, "float")
    kept = {}
    if scales is not None:
        kept = dict(zip(("mean_scale", "square_scale"), scales([-(-int(np.prod(s)) // 256) for s in SIZES])))
    opt = thc.AdamW(_put(thc, p), _put(thc, g), bits=8, **kept, **HYPER)
    opt.step()
    return opt


def _new(thc):
    return [thc.Tensor("float") for _ in SIZES]


def test_outputs_on_another_tensors_are_refused(thc):
    opt = _stepped(thc)
    scales = [x.numpy() for x in opt.mean_scale + opt.square_scale]
    room = thc.Tensor("float").resize((2000,)).fill(7)
    for first, second, match in ((room.narrow(0, 0, 300), room.narrow(0, 299, 300), "tensor 3 lies on tensor 1's moments"),
                                 (room.narrow(0, 500, 300), room.narrow(0, 300, 300), "tensor 1 lies on tensor 3's moments"),
                                 (room.narrow(0, 500, 300), room.narrow(0, 500, 300), "lies on tensor .'s moments")):
        for squares in (False, True):
            mean, square = _new(thc), _new(thc)
            (square if squares else mean)[0], mean[2] = first, second
            with pytest.raises(thc.THCError, match=match):
                opt.moments(mean, square)
    for at, on in ((0, opt.mean_scale[1]), (1, opt.square_scale[0]), (2, opt.mean_scale[0])):
        for squares in (False, True):
            mean, square = _new(thc), _new(thc)
            # the output grows over the storage that begins with the scales
            (square if squares else mean)[at] = on.view_as_strided(0, (1,), (1,))
            with pytest.raises(thc.THCError, match="tensor %d lies on tensor .'s scales" % (at + 1)):
                opt.moments(mean, square)
    assert np.all(room.numpy() == 7)
    for x, was in zip(opt.mean_scale + opt.square_scale, scales):
        assert_bit_equal(x.numpy(), was)


def test_outputs_side_by_side_and_in_gaps(thc):
    plain = _stepped(thc)
    want = [[x.numpy() for x in l] for l in plain.moments()]
    # all outputs and scales on one storage, in an order of their own
    room = thc.Tensor("float").resize((4000,)).zero()

    def scales(blocks):
        ends = np.cumsum([0] + blocks + blocks)
        parts = [room.narrow(0, 3900 + int(a), n) for a, n in zip(ends, blocks + blocks)]
        return parts[:len(blocks)], parts[len(blocks):]

    opt = _stepped(thc, scales)
    at, outs = 0, []
    for n in [int(np.prod(s)) for s in SIZES + SIZES]:
        outs.append(room.narrow(0, at, n))
        at += n
    mean, square = opt.moments(outs[4:], outs[:4])
    for a, b in zip(mean + square, want[0] + want[1]):
        assert_bit_equal(a.numpy(), b)
    # every second element, and the scales in their gaps
    room = thc.Tensor("float").resize((8000,)).zero()

    def odd(blocks):
        ends = np.cumsum([0] + blocks + blocks)
        parts = [room.view_as_strided(2 * int(a) + 1, (n,), (2,)) for a, n in zip(ends, blocks + blocks)]
        return parts[:len(blocks)], parts[len(blocks):]

    opt = _stepped(thc, odd)
    at, outs = 0, []
    for s in SIZES + SIZES:
        outs.append(room.view_as_strided(2 * at, s, (2,) if len(s) == 1 else (2 * s[1], 2)))
        at += int(np.prod(s))
    outs[0], outs[4] = thc.Tensor("float"), thc.Tensor("float")
    outs[1], outs[5], outs[3], outs[7] = (thc.Tensor("float") for _ in range(4))
    mean, square = opt.moments(outs[:4], outs[4:])
    for a, b in zip(mean + square, want[0] + want[1]):
        assert_bit_equal(a.numpy(), b)


def test_32_bit_moments_in_the_tensors_given(thc):
    rng = np.random.default_rng(10)
    shapes = SIZES + [()]
    p, g = _problem(rng, SIZES, "float")
    opt = thc.AdamW(_put(thc, p) + [thc.Tensor("float")], _put(thc, g) + [thc.Tensor("float")], **HYPER)
    opt.step()
    states = [[x.numpy() for x in l[:4]] for l in (opt.mean, opt.square)]      # (the last one has no elements)
    # new ones, one of another size, and every second column of something wider
    wide = thc.Tensor("float").resize((7, 200)).fill(7)
    mean, square = ([thc.Tensor("float") for _ in shapes] for _ in range(2))
    mean[0].resize((9, 9))
    mean[1] = wide.view_as_strided(0, (7, 100), (200, 2))
    got = opt.moments(mean, square)
    assert got[0] is mean and got[1] is square
    for given, held in zip(got, states):
        assert given[4].numel() == 0
        for a, b in zip(given, held):
            assert_bit_equal(a.numpy(), b)
    assert np.all(wide.numpy()[:, 1::2] == 7)
    opt.step()
    assert_bit_equal(mean[0].numpy(), states[0][0])         # the run has gone on, the copies have not
    # those not given are the states themselves, and the states may be given
    mean, square = opt.moments(square=square)
    assert [x.a for x in mean] == [x.a for x in opt.mean] and not np.array_equal(square[0].numpy(), states[1][0])
    assert_bit_equal(opt.moments(opt.mean)[0][0].numpy(), mean[0].numpy())
    for bad in ([thc.Tensor("float")], [thc.Tensor("half") for _ in shapes]):
        with pytest.raises(ValueError):
            opt.moments(bad)


def test_a_tensors_two_moments_as_columns(thc):
    """Mean and square side by side for each element, and in the gaps of the tensor's own scales: spans that meet, elements that do not."""
    plain = _stepped(thc)
    want = [[x.numpy() for x in l] for l in plain.moments()]
    room = thc.Tensor("float").resize((300, 4)).fill(7)

    def beside(blocks):
        return ([room.view_as_strided(2, (blocks[0],), (4,))] + [thc.Tensor("float").resize((n,)).zero() for n in blocks[1:]],
                [room.view_as_strided(3, (blocks[0],), (4,))] + [thc.Tensor("float").resize((n,)).zero() for n in blocks[1:]])

    opt = _stepped(thc, lambda blocks: [[t.zero() for t in l] for l in beside(blocks)])
    mean, square = _new(thc), _new(thc)
    mean[0], square[0] = room.select(1, 0), room.select(1, 1)
    opt.moments(mean, square)
    for a, b in zip(mean + square, want[0] + want[1]):
        assert_bit_equal(a.numpy(), b)
    held = room.numpy()[:, 2:]
    assert_bit_equal(held[:2, 0].copy(), plain.mean_scale[0].numpy())
    assert_bit_equal(held[:2, 1].copy(), plain.square_scale[0].numpy())
    assert np.all(held[2:] == 7)
