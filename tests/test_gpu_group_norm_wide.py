"""Group norm of slices of more than 8192 channels over many pixels, whose sums are long."""
import numpy as np
import pytest

from glow_amd import capi
from tests import group_norm_ref, mx4_ref as ref

pytestmark = pytest.mark.gpu
#: Sums are held in 64 bits there: what is left is the rounding of mean and variance to two and one
#: numbers of 32 bits.
STEPS = 4


@pytest.fixture(scope="module", autouse=True)
def _device():
    capi.init(0)


@pytest.mark.parametrize("type_, value", [(ref.F16, 1.1), (ref.F32, 1.1), (ref.BF16, -1.1), (ref.F32, 1000.3)])
@pytest.mark.parametrize("pixels, C, groups", [(784, 16384, 1), (1000, 18001, 1), (301, 33 * 600, 2)])
def test_constant_groups_are_beta(pixels, C, groups, type_, value):
    x = np.broadcast_to(ref.to_type(np.array([value]), type_), (1, pixels, C))
    beta = np.linspace(-1, 1, C).astype(np.float32)
    got = capi.group_norm(x, groups, None, beta, type_=type_)
    np.testing.assert_array_equal(got, np.broadcast_to(ref.to_type(beta, type_), x.shape))
    rows = capi.group_norm(x, groups, None, beta, type_=type_, out_type=capi.TYPE_MX4)
    np.testing.assert_array_equal(rows[0], np.broadcast_to(ref.rows_of(beta[None]), rows[0].shape))


@pytest.mark.parametrize("type_", [ref.F32, ref.F16, ref.BF16])
@pytest.mark.parametrize("offset", [0.3, 1000.3])
@pytest.mark.parametrize("n, pixels, C, groups", [(1, 1568, 9000, 1), (2, 500, 8300 * 2, 2)])
def test_long_sums(n, pixels, C, groups, offset, type_):
    rng = np.random.default_rng(pixels + type_)
    x = ref.to_type(rng.normal(0, 1, (n, pixels, C)).astype(np.float32) + np.float32(offset), type_)
    gamma, beta = (1 + 0.3 * rng.normal(0, 1, C)).astype(np.float32), rng.normal(0, 1, C).astype(np.float32)
    want, err = group_norm_ref.norm(ref.to_f64(x, type_), groups, gamma, beta, 1e-5, 1, STEPS)
    ref.check_float(capi.group_norm(x, groups, gamma, beta, 1e-5, 1, type_), want, err, type_)


def test_a_drift_over_the_pixels():
    # a sum that is joined block by block must not lose the blocks that come late
    pixels, C = 3000, 8200
    x = np.broadcast_to(np.linspace(-50, 950, pixels, dtype=np.float32)[None, :, None], (1, pixels, C))
    want, err = group_norm_ref.norm(x.astype(np.float64), 1, None, None, 1e-5, 0, STEPS)
    ref.check_float(capi.group_norm(x, 1), want, err, ref.F32)


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("where", [0, 1, -1])
def test_nan_and_infinity_stay_in_their_group(where, value):
    rng = np.random.default_rng(1)
    x = rng.normal(0, 1, (2, 40, 2 * 8400)).astype(np.float32)
    pixel, channel = (0, 8400 + where) if where >= 0 else (39, 2 * 8400 - 1)
    x[1, pixel, channel] = value
    with np.errstate(invalid="ignore"):
        want, err = group_norm_ref.norm(x.astype(np.float64), 2, None, None, 1e-5, 1, STEPS)
    assert np.isnan(want[1, :, 8400:]).all() and np.isfinite(want[0]).all() and np.isfinite(want[1, :, :8400]).all()
    ref.check_float(capi.group_norm(x, 2, activation=1), want, np.where(np.isfinite(err), err, 0), ref.F32)
