"""SiLU of 32-bit values: products over no columns are the activation of the bias."""
import numpy as np
import pytest

from glow_amd import capi
from tests import mx4_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device():
    capi.init(0)


def silu_of(v, M):
    """As a product of M rows gives it: M chooses the kernel."""
    got = capi.mx4_fc(np.zeros((M, 0), np.float32), ref.F32, np.zeros((v.size, 0), np.uint8), v, 0, ref.F32, capi.ACT_SILU)
    assert (got.view(np.uint32) == got[:1].view(np.uint32)).all()
    return got[0]


@pytest.mark.parametrize("M", [1, 40, 700])
def test_silu_is_within_what_the_header_says(M):
    rng = np.random.default_rng(M)
    v = np.concatenate([np.linspace(-87, 87, 4001), rng.normal(0, 1, 2000), 10.0 ** rng.uniform(-30, 38, 500),
                        -10.0 ** rng.uniform(-30, 1.9, 500)]).astype(np.float32)
    x = v.astype(np.float64)
    want = x / (1 + np.exp(-x))
    assert np.all(np.abs(silu_of(v, M) - want) <= (1.3 * np.abs(x) + 6) * 2.0 ** -24 * np.abs(want))


@pytest.mark.parametrize("M", [1, 40, 700])
def test_silu_of_far_and_special_values(M):
    far = np.concatenate([np.linspace(-700, -87, 3000), [-1e4, -1e30, -3e38]]).astype(np.float32)
    got = silu_of(far, M).astype(np.float64)
    x = far.astype(np.float64)
    with np.errstate(over="ignore"):
        want = x / (1 + np.exp(-x))
    assert np.all(np.abs(got - want) <= 2.0 ** -119) and np.all(got <= 0)
    special = silu_of(np.array([np.nan, np.inf, -np.inf, 0.0, -0.0], np.float32), M)
    assert np.isnan(special[0]) and special[1] == np.inf and np.isnan(special[2])        # (-inf / inf)
    assert (special[3:] == 0).all()
