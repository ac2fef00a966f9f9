"""AdamW with second moments of every size, down to the smallest float: bit for bit against the same operations in numpy, which keeps
subnormal numbers as the kernels do."""
import numpy as np
import pytest

from tests.test_adamw_gpu import _blocks, _f, _numpy_step, _put
from tests.util import assert_bit_equal

pytestmark = pytest.mark.gpu
NOTHING = dict(lr=2e-3, beta1=0.9, beta2=0.97, eps=0.0, weight_decay=0.05)


def _every_size(rng, per=64):
    """Floats of every exponent, subnormal ones by their leading bit."""
    normal = (rng.integers(0, 1 << 23, (254, per)) | (np.arange(1, 255)[:, None] << 23)).astype(np.uint32)
    bits = np.arange(23)[:, None]
    subnormal = ((1 << bits) | (rng.integers(0, 1 << 23, (23, per)) & ((1 << bits) - 1))).astype(np.uint32)
    return np.concatenate([subnormal.reshape(-1), normal.reshape(-1)]).view(np.float32)


@pytest.mark.parametrize("eps", [0.0, 1e-30])
@pytest.mark.parametrize("kind,master", [("float", False), ("half", True)])
def test_roots_of_second_moments_of_every_size(thc, kind, master, eps):
    """The moments given, no gradient: the parameter moves by the mean over the root."""
    rng = np.random.default_rng(1)
    h = dict(NOTHING, beta2=0.5, eps=eps)
    v = _every_size(rng)
    v = v[v.view(np.uint32) > 1]           # (half of the smallest would be zero)
    m = rng.uniform(0.5, 1, v.size).astype(np.float32) * np.sqrt(v)
    p = rng.standard_normal(v.size).astype(np.float32)
    q = p.astype(np.float16 if kind == "half" else np.float32)
    g = np.zeros_like(q)
    copies = _put(thc, [p]) if master else None
    dp, dm, dv = _put(thc, [q]), _put(thc, [m]), _put(thc, [v])
    thc.AdamW(dp, _put(thc, [g]), master=copies, mean=dm, square=dv, step=2, **h).step()
    p, m, v = _numpy_step(p, g, m, v, 3, 1.0, h)
    assert_bit_equal(dm[0].numpy(), m)
    assert_bit_equal(dv[0].numpy(), v)
    assert_bit_equal((copies or dp)[0].numpy(), p)
    assert_bit_equal(dp[0].numpy(), p.astype(q.dtype))


@pytest.mark.parametrize("bits", [32, 8])
def test_first_step_of_small_gradients(thc, bits):
    """Gradients from 1e-15 to 1e-21 and no eps: every parameter moves by the rate, as far as the root's own few bits allow."""
    rng = np.random.default_rng(2)
    g = (rng.choice([-1, 1], 4099) * 10.0 ** rng.uniform(-21, -15, 4099)).astype(np.float32)
    p = rng.standard_normal(4099).astype(np.float32)
    d = _put(thc, [p])
    thc.AdamW(d, _put(thc, [g]), bits=bits, **NOTHING).step()
    want, _, v = _numpy_step(p, g, np.zeros_like(p), np.zeros_like(p), 1, 1.0, NOTHING)
    assert (v > 0).all() and (v < 2.0 ** -126).any() and (v > 2.0 ** -110).any()
    assert_bit_equal(d[0].numpy(), want)
