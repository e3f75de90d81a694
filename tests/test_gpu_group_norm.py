"""Group norm with an activation against 64 bits, and the way from it through microscaled
rows into products."""
import numpy as np
import pytest

from glow_amd import capi
from tests import mx4_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device():
    capi.init(0)


def image(rng, n, pixels, C, type_, offset=1.0):
    x = rng.normal(0, 1, (n, pixels, C)) * np.exp(0.5 * rng.normal(0, 1, C)) + offset * rng.normal(0, 1, C)
    return ref.to_type(x, type_)


SHAPES = [(1, 1, 1, 1), (1, 1, 64, 64), (2, 1, 96, 8), (3, 2, 10, 5), (1, 49, 512, 32), (2, 49, 64, 1), (2, 35, 100, 4),
          (3, 1225, 100, 4), (4, 784, 128, 32), (1, 5000, 24, 3), (2, 3136, 256, 32), (1, 7, 2048, 16), (5, 64, 130, 2),
          (1, 40000, 16, 1), (33, 17, 40, 40), (1, 3, 5000, 8), (1, 20000, 128, 32)]


@pytest.mark.parametrize("type_", [ref.F32, ref.F16, ref.BF16])
@pytest.mark.parametrize("n, pixels, C, groups", SHAPES)
def test_group_norm(n, pixels, C, groups, type_):
    rng = np.random.default_rng(n + pixels + C)
    x = image(rng, n, pixels, C, type_)
    gamma, beta = (1 + 0.3 * rng.normal(0, 1, C)).astype(np.float32), rng.normal(0, 1, C).astype(np.float32)
    act = (0, 1, 6)[(n + pixels + type_) % 3]
    for g, b in ((gamma, beta), (None, None)) if C < 200 else ((gamma, beta),):
        want, err = ref.group_norm(ref.to_f64(x, type_), groups, g, b, 1e-5, act)
        ref.check_float(capi.group_norm(x, groups, g, b, 1e-5, act, type_), want, err, type_)
        rows = capi.group_norm(x, groups, g, b, 1e-5, act, type_, capi.TYPE_MX4)
        ref.check_mx4(rows.reshape(n * pixels, -1), C, want.reshape(n * pixels, C), err.reshape(n * pixels, C))


@pytest.mark.parametrize("seed", range(48))
def test_group_norm_of_random_shapes(seed):
    """Groups of 1 to 60 channels, samples enough for slices on one die, rows apart by any number of
    elements and from any element on, each result type, in place."""
    rng = np.random.default_rng(1000 + seed)
    type_ = int(rng.integers(0, 3))
    size = 4 if type_ == ref.F32 else 2
    per, groups = int(rng.integers(1, 61)), int(rng.integers(1, 40))
    C = per * groups
    n = int(np.exp(rng.uniform(0, np.log(40))))
    pixels = int(np.exp(rng.uniform(0, np.log(max(2, 1_500_000 // (C * n))))))
    act, gap, start = int(rng.choice([0, 1, 6])), int(rng.integers(0, 4)), int(rng.integers(0, 5))
    x = image(rng, n, pixels, C, type_)
    gamma, beta = (1 + 0.3 * rng.normal(0, 1, C)).astype(np.float32), rng.normal(0, 1, C).astype(np.float32)
    want, err = ref.group_norm(ref.to_f64(x, type_), groups, gamma, beta, 1e-5, act)
    wide = np.zeros((n * pixels, C + gap), x.dtype)
    wide[:, :C] = x.reshape(-1, C)
    flat = np.concatenate([np.zeros(start, x.dtype), wide.reshape(-1)])
    dx, dg, db = capi.to_device(flat), capi.to_device(gamma), capi.to_device(beta)
    ws_bytes = capi.group_norm_workspace_bytes(n, pixels, C, groups)
    ws = capi.DeviceBuffer(ws_bytes)
    pitch = (C + gap) * size
    row = capi.mx4_row_bytes(C)
    rows = capi.to_device(np.full((n * pixels, row + 16), 0xA5, np.uint8))
    args = (dg, db, n, pixels, C, groups, 1e-5, act, ws, ws_bytes)
    capi.launch_group_norm(rows, capi.TYPE_MX4, row + 16, dx.ptr + start * size, type_, pitch, *args)
    got = rows.numpy()
    assert (got[:, row:] == 0xA5).all()
    ref.check_mx4(got[:, :row], C, want.reshape(-1, C), err.reshape(-1, C))
    out = capi.to_device(np.zeros(flat.size, x.dtype))
    capi.launch_group_norm(out.ptr + start * size, type_, pitch, dx.ptr + start * size, type_, pitch, *args)
    apart = out.numpy()
    capi.launch_group_norm(dx.ptr + start * size, type_, pitch, dx.ptr + start * size, type_, pitch, *args)
    np.testing.assert_array_equal(dx.numpy(), apart)        # (the gaps are zero on both sides)
    vals = apart[start:].reshape(n * pixels, C + gap)
    assert not vals[:, C:].any()
    ref.check_float(np.ascontiguousarray(vals[:, :C]).reshape(x.shape), want, err, type_)


@pytest.mark.parametrize("type_", [ref.F32, ref.F16, ref.BF16])
@pytest.mark.parametrize("per", [1, 2, 3, 4, 5, 6, 7, 8, 9, 12, 16, 20, 31])
def test_large_slices_of_every_kind_of_group(per, type_):
    """Slices that fill a workgroup to the last pixel it can hold, one more, and far more."""
    rng = np.random.default_rng(per)
    for n, pixels, groups in ((16, 1024, 8), (16, 1025, 8), (16, 2047, 8), (9, 4097, 3), (130, 1500, 1)):
        x = image(rng, n, pixels, per * groups, type_)
        want, err = ref.group_norm(ref.to_f64(x, type_), groups, None, None, 1e-5, 1)
        ref.check_float(capi.group_norm(x, groups, activation=1, type_=type_), want, err, type_)


@pytest.mark.parametrize("type_", [ref.F32, ref.F16])
@pytest.mark.parametrize("n, pixels, C, groups", [(2, 3, 20000, 2), (1, 5, 9000, 1), (3, 2, 8200, 8), (2, 2, 31 * 300, 300)])
def test_slices_wider_than_a_workgroup(type_, n, pixels, C, groups):
    rng = np.random.default_rng(C)
    x = image(rng, n, pixels, C, type_)
    beta = rng.normal(0, 1, C).astype(np.float32)
    want, err = ref.group_norm(ref.to_f64(x, type_), groups, None, beta, 1e-5, 6)
    ref.check_float(capi.group_norm(x, groups, None, beta, 1e-5, 6, type_), want, err, type_)
    rows = capi.group_norm(x, groups, None, beta, 1e-5, 6, type_, capi.TYPE_MX4)
    ref.check_mx4(rows.reshape(n * pixels, -1), C, want.reshape(-1, C), err.reshape(-1, C))


@pytest.mark.parametrize("n, pixels, C, groups", [(2, 3136, 64, 8), (1, 49, 512, 32), (1, 30000, 32, 4)])
def test_errors_are_of_32_bits(n, pixels, C, groups):
    # the norm of the error of sums whose roundings go either way: well under a hundred of the
    # 2^-24 that each is off by, a mean of a few deviations included
    x = image(np.random.default_rng(9), n, pixels, C, ref.F32, offset=3.0)
    want, _ = ref.group_norm(ref.to_f64(x, ref.F32), groups, None, None, 1e-5, 0)
    got = capi.group_norm(x, groups).astype(np.float64)
    assert np.linalg.norm(got - want) <= 100 * 2.0 ** -24 * np.linalg.norm(want)


def test_a_mean_far_from_zero():
    # 1000 deviations: the values themselves have the rounding of 2^-24 * 1000, the norm no more
    # than the sums' bound
    x = (np.random.default_rng(4).normal(0, 1, (2, 900, 32)) + 1000).astype(np.float32)
    want, err = ref.group_norm(x.astype(np.float64), 4, None, None, 1e-5, 0)
    got = capi.group_norm(x, 4)
    ref.check_float(got, want, err, ref.F32)
    assert np.abs(got.astype(np.float64) - want).max() < 1e-3


def test_constant_groups_are_beta():
    x = np.full((2, 300, 24), 3.25, np.float32)
    beta = np.linspace(-1, 1, 24).astype(np.float32)
    np.testing.assert_array_equal(capi.group_norm(x, 3, None, beta), np.broadcast_to(beta, x.shape))


@pytest.mark.parametrize("type_", [ref.F32, ref.F16, ref.BF16])
@pytest.mark.parametrize("n, pixels, C, groups", [(3, 50, 48, 6), (2, 3000, 40, 4)])
def test_nan_and_infinity_stay_in_their_group(n, pixels, C, groups, type_):
    rng = np.random.default_rng(8)
    x = ref.to_f64(image(rng, n, pixels, C, type_), type_)
    x[0, 3, 0] = np.nan
    x[1, pixels - 1, C - 1] = np.inf
    x[1, 5, 1] = -np.inf
    x = ref.to_type(x, type_)
    with np.errstate(invalid="ignore"):
        want, err = ref.group_norm(ref.to_f64(x, type_), groups, None, None, 1e-5, 1)
    assert np.isnan(want).any() and np.isfinite(want).any()
    err = np.where(np.isfinite(err), err, 0)
    ref.check_float(capi.group_norm(x, groups, activation=1, type_=type_), want, err, type_)


@pytest.mark.parametrize("type_", [ref.F32, ref.F16])
@pytest.mark.parametrize("pixels", [30, 4000])
def test_strided_pixels_leave_the_rest_alone(type_, pixels):
    rng = np.random.default_rng(2)
    n, C, groups, size = 2, 72, 9, 4 if type_ == ref.F32 else 2
    x = image(rng, n, pixels, C, type_)
    gap = 3                                             # elements: rows at any address
    wide = np.full((n * pixels, (C + gap) * size), 0xFF, np.uint8)      # NaN between the pixels
    wide[:, :C * size] = x.reshape(n * pixels, C).view(np.uint8)
    dx = capi.to_device(wide)
    ws_bytes = capi.group_norm_workspace_bytes(n, pixels, C, groups)
    ws = capi.DeviceBuffer(max(ws_bytes, 1))
    want, err = ref.group_norm(ref.to_f64(x, type_), groups, None, None, 1e-5, 0)
    pitch = (C + 5) * size
    out = capi.to_device(np.full((n * pixels + 1, pitch), 0xA5, np.uint8))
    capi.launch_group_norm(out, type_, pitch, dx, type_, (C + gap) * size, None, None, n, pixels, C, groups, 1e-5, 0,
                           ws, ws_bytes)
    got = out.numpy()
    assert (got[:, C * size:] == 0xA5).all() and (got[-1] == 0xA5).all()
    vals = np.ascontiguousarray(got[:-1, :C * size]).view(x.dtype).reshape(x.shape)
    ref.check_float(vals, want, err, type_)
    rows = capi.to_device(np.full((n * pixels, capi.mx4_row_bytes(C) + 16), 0xA5, np.uint8))
    capi.launch_group_norm(rows, capi.TYPE_MX4, rows.shape[1], dx, type_, (C + gap) * size, None, None, n, pixels, C,
                           groups, 1e-5, 0, ws, ws_bytes)
    got = rows.numpy()
    assert (got[:, -16:] == 0xA5).all()
    ref.check_mx4(got[:, :-16], C, want.reshape(-1, C), err.reshape(-1, C))
    # in place
    capi.launch_group_norm(dx, type_, (C + gap) * size, dx, type_, (C + gap) * size, None, None, n, pixels, C, groups,
                           1e-5, 0, ws, ws_bytes)
    got = dx.numpy()
    assert (got[:, C * size:] == 0xFF).all()
    np.testing.assert_array_equal(np.ascontiguousarray(got[:, :C * size]).view(x.dtype).reshape(x.shape), vals)


@pytest.mark.parametrize("n, pixels, C, groups", [(2, 60, 130, 13), (3, 784, 256, 32), (1, 9000, 96, 8)])
def test_microscaled_results_are_the_quantised_float_ones(n, pixels, C, groups):
    x = image(np.random.default_rng(6), n, pixels, C, ref.F32)
    for act in (capi.ACT_NONE, capi.ACT_RELU):
        y = capi.group_norm(x, groups, activation=act)
        rows = capi.group_norm(x, groups, activation=act, out_type=capi.TYPE_MX4)
        np.testing.assert_array_equal(rows.reshape(n * pixels, -1), ref.rows_of(y.reshape(n * pixels, C)))


def test_block_of_norm_and_products_replays():
    """Group norm with SiLU to microscaled rows, a pointwise product with Relu to microscaled
    rows, another back to the image's type: eager on a stream, then from two graphs that
    were captured over the same buffers and are replayed in turn."""
    rng = np.random.default_rng(1)
    n, C, groups, mid = 2, 96, 8, 40
    stream = capi.Stream()
    w1, w2 = ref.rows_of(rng.normal(0, C ** -0.5, (mid, C))), ref.rows_of(rng.normal(0, mid ** -0.5, (C, mid)))
    b1, b2 = rng.normal(0, 0.1, mid).astype(np.float32), rng.normal(0, 0.1, C).astype(np.float32)
    dw1, dw2, db1, db2 = (capi.to_device(v) for v in (w1, w2, b1, b2))
    most = n * 3000
    x = capi.DeviceBuffer.empty((most, C), np.float16)
    normed = capi.DeviceBuffer.empty((most, capi.mx4_row_bytes(C)), np.uint8)
    hidden = capi.DeviceBuffer.empty((most, capi.mx4_row_bytes(mid)), np.uint8)
    out = capi.DeviceBuffer.empty((most, C), np.float16)

    def launch(pixels, ws, ws_bytes):
        rows = n * pixels
        capi.launch_group_norm(normed, capi.TYPE_MX4, normed.shape[1], x, capi.TYPE_F16, 2 * C, None, None, n, pixels,
                               C, groups, 1e-5, capi.ACT_SILU, ws, ws_bytes, stream)
        capi.launch_mx4_fc(hidden, capi.TYPE_MX4, hidden.shape[1], normed, capi.TYPE_MX4, normed.shape[1], dw1,
                           w1.shape[1], db1, rows, C, mid, capi.ACT_RELU, None, 0, stream)
        capi.launch_mx4_fc(out, capi.TYPE_F16, 2 * C, hidden, capi.TYPE_MX4, hidden.shape[1], dw2, w2.shape[1], db2,
                           rows, mid, C, capi.ACT_NONE, None, 0, stream)

    def inputs(i, pixels):
        return image(np.random.default_rng(i), n, pixels, C, ref.F16).reshape(-1, C)

    scratch = {}
    for pixels in (30, 3000):
        nbytes = capi.group_norm_workspace_bytes(n, pixels, C, groups)
        scratch[pixels] = (capi.DeviceBuffer(max(nbytes, 1)), nbytes)
    eager = {}
    for pixels in (30, 3000):
        rows = n * pixels
        for i in range(2):
            x.upload(inputs(i, pixels), stream)
            launch(pixels, *scratch[pixels])
            eager[pixels, i] = [b.numpy(stream)[:rows] for b in (normed, hidden, out)]
        got = eager[pixels, 0]
        want, err = ref.group_norm(ref.to_f64(inputs(0, pixels), ref.F16).reshape(n, pixels, C), groups, None, None,
                                   1e-5, 6)
        ref.check_mx4(got[0], C, want.reshape(-1, C), err.reshape(-1, C))
        want, err = ref.fc(ref.values(got[0], C), ref.values(w1, C), b1.astype(np.float64), 1)
        ref.check_mx4(got[1], mid, want, err)
        want, err = ref.fc(ref.values(got[1], mid), ref.values(w2, mid), b2.astype(np.float64), 0)
        ref.check_float(got[2], want, err, ref.F16)
    graphs = {}
    for pixels in (30, 3000):
        with capi.Graph(stream) as graphs[pixels]:
            launch(pixels, *scratch[pixels])
    for pixels, i in ((3000, 1), (30, 0), (3000, 0), (30, 1), (3000, 1)):
        x.upload(inputs(i, pixels), stream)
        graphs[pixels].launch(stream)
        for got, want in zip((normed, hidden, out), eager[pixels, i]):
            np.testing.assert_array_equal(got.numpy(stream)[:n * pixels], want)
        capi.sync()
