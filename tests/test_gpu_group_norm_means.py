"""Group norm of values that lie far from zero, or next to each other: the error goes by what they
are apart, in every type and on every way through the kernels."""
import numpy as np
import pytest

from glow_amd import capi
from tests import group_norm_ref, mx4_ref as ref

pytestmark = pytest.mark.gpu
TYPES = [ref.F32, ref.F16, ref.BF16]
#: groups of whole vectors, of 25 and of 3 channels; in registers and in parts
SHAPES = [(2, 49, 64, 8), (3, 50, 100, 4), (2, 61, 30, 10), (40, 150, 96, 6), (1, 20011, 64, 8), (2, 9001, 100, 4),
          (1, 12007, 24, 8)]
#: A thread sums up to 128 values one by one; lanes, waves and the parts of a slice are joined in
#: less than as many steps again, where a slice has as few pixels as here.
STEPS = 256


@pytest.fixture(scope="module", autouse=True)
def _device():
    capi.init(0)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("n, pixels, C, groups", SHAPES)
def test_constant_groups_are_beta(n, pixels, C, groups, type_):
    beta = np.linspace(-1, 1, C).astype(np.float32)
    for value in (3.25, -1.1, 1000.3, 60000.0) + ((1.5e36, -3e38) if type_ != ref.F16 else ()):
        x = np.broadcast_to(ref.to_type(np.array([value]), type_), (n, pixels, C))
        got = capi.group_norm(x, groups, None, beta, type_=type_)
        np.testing.assert_array_equal(got, np.broadcast_to(ref.to_type(beta, type_), x.shape), str(value))
        rows = capi.group_norm(x, groups, None, beta, type_=type_, out_type=capi.TYPE_MX4)
        np.testing.assert_array_equal(rows, np.broadcast_to(ref.rows_of(beta[None]), rows.shape), str(value))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("n, pixels, C, groups", SHAPES)
def test_means_far_from_zero(n, pixels, C, groups, type_):
    """A million deviations away in 32 bits, a few thousand in fp16, a few hundred in bf16."""
    far, spread = {ref.F32: (1e6, 1.0), ref.F16: (30000.0, 12.0), ref.BF16: (-20000.0, 60.0)}[type_]
    rng = np.random.default_rng(pixels + type_)
    x = ref.to_type(far * rng.uniform(0.6, 1, (n, 1, groups)).repeat(C // groups, 2)
                    + spread * rng.normal(0, 1, (n, pixels, C)), type_)
    gamma, beta = (1 + 0.3 * rng.normal(0, 1, C)).astype(np.float32), rng.normal(0, 1, C).astype(np.float32)
    for act in (0, 6):
        want, err = group_norm_ref.norm(ref.to_f64(x, type_), groups, gamma, beta, 1e-5, act, STEPS)
        ref.check_float(capi.group_norm(x, groups, gamma, beta, 1e-5, act, type_), want, err, type_)
        rows = capi.group_norm(x, groups, gamma, beta, 1e-5, act, type_, capi.TYPE_MX4)
        ref.check_mx4(rows.reshape(n * pixels, -1), C, want.reshape(-1, C), err.reshape(-1, C))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("n, pixels, C, groups", SHAPES)
def test_one_value_beside_equal_ones(n, pixels, C, groups, type_):
    """The group's first value, its last, or one in between is a step away from all others."""
    per = C // groups
    for at in ((0, 0), (pixels - 1, per - 1), (pixels // 2, per // 3)):
        x = ref.to_type(np.full((n, pixels, C), 1000.0), type_)
        x.reshape(n, pixels, groups, per)[:, at[0], :, at[1]] = ref.to_type(np.array([1008.0]), type_)
        want, err = group_norm_ref.norm(ref.to_f64(x, type_), groups, None, None, 1e-5, 0, STEPS)
        ref.check_float(capi.group_norm(x, groups, type_=type_), want, err, type_)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("n, pixels, C, groups", SHAPES)
def test_a_first_value_that_is_no_number(n, pixels, C, groups, value, type_):
    rng = np.random.default_rng(3)
    per = C // groups
    x = rng.normal(0, 1, (n, pixels, C))
    x[-1, 0, per] = value
    x = ref.to_type(x, type_)
    with np.errstate(invalid="ignore"):
        want, err = group_norm_ref.norm(ref.to_f64(x, type_), groups, None, None, 1e-5, 1, STEPS)
    assert np.isnan(want[-1, :, per:2 * per]).all() and np.isfinite(want[-1, :, :per]).all()
    err = np.where(np.isfinite(err), err, 0)
    ref.check_float(capi.group_norm(x, groups, activation=1, type_=type_), want, err, type_)
    rows = capi.group_norm(x, groups, activation=1, type_=type_, out_type=capi.TYPE_MX4)
    ref.check_mx4(rows.reshape(n * pixels, -1), C, want.reshape(-1, C), err.reshape(-1, C))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("n, pixels, C, groups", SHAPES)
def test_far_means_in_place(n, pixels, C, groups, type_):
    rng = np.random.default_rng(5)
    x = ref.to_type(5000 + 40 * rng.normal(0, 1, (n, pixels, C)), type_)
    apart = capi.group_norm(x, groups, activation=1, type_=type_)
    dx, ws_bytes = capi.to_device(x), capi.group_norm_workspace_bytes(n, pixels, C, groups)
    ws = capi.DeviceBuffer(ws_bytes)
    capi.launch_group_norm(dx, type_, C * x.itemsize, dx, type_, C * x.itemsize, None, None, n, pixels, C, groups, 1e-5, 1,
                           ws, ws_bytes)
    np.testing.assert_array_equal(dx.numpy(), apart)


@pytest.mark.parametrize("n, pixels, C, groups", SHAPES)
def test_values_below_the_normal_ones_of_fp16(n, pixels, C, groups):
    rng = np.random.default_rng(6)
    x = ref.to_type(2e-5 + 1e-5 * rng.normal(0, 1, (n, pixels, C)), ref.F16)
    want, err = group_norm_ref.norm(ref.to_f64(x, ref.F16), groups, None, None, 1e-10, 0, STEPS)
    ref.check_float(capi.group_norm(x, groups, epsilon=1e-10, type_=ref.F16), want, err, ref.F16)
