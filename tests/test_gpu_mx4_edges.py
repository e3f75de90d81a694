"""Group norm and the quantisation where launches take turns, slices are wider than a wave, and calls
run at once or again."""
import numpy as np
import pytest

from glow_amd import capi
from tests import group_norm_ref, mx4_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device():
    capi.init(0)


def image(rng, n, pixels, C, type_):
    return ref.to_type(rng.normal(0, 1, (n, pixels, C)) * np.exp(0.5 * rng.normal(0, 1, C)) + rng.normal(0, 1, C), type_)


class Norm:
    """A group norm's buffers, and its launch."""

    def __init__(self, x, type_, groups, act=0, out_type=None, in_place=False, stream=None):
        self.args = (x.shape, type_, groups, act, type_ if out_type is None else out_type)
        n, pixels, C = x.shape
        self.row = capi.mx4_row_bytes(C) if out_type == ref.MX4 else C * x.itemsize
        self.x = capi.to_device(x)
        self.out = self.x if in_place else capi.DeviceBuffer.empty((n * pixels, self.row), np.uint8)
        self.ws_bytes = capi.group_norm_workspace_bytes(n, pixels, C, groups)
        self.ws, self.stream = capi.DeviceBuffer(self.ws_bytes), stream

    def launch(self):
        (n, pixels, C), type_, groups, act, out_type = self.args
        capi.launch_group_norm(self.out, out_type, self.row, self.x, type_, C * self.x.dtype.itemsize, None, None, n, pixels,
                               C, groups, 1e-5, act, self.ws, self.ws_bytes, self.stream)


@pytest.mark.parametrize("type_", [ref.F32, ref.F16, ref.BF16])
@pytest.mark.parametrize("n, pixels, per, groups", [(1, 4000, 625, 2), (1, 4000, 515, 3), (130, 30, 625, 1), (130, 7, 1301, 1),
                                                    (2, 900, 1301, 1), (9, 40, 515, 2)])
def test_in_place_where_waves_share_a_vector(n, pixels, per, groups, type_):
    """Slices of more than 64 vectors of eight, the last of which overlaps the one in front."""
    x = image(np.random.default_rng(per), n, pixels, per * groups, type_)
    want, err = group_norm_ref.norm(ref.to_f64(x, type_), groups, None, None, 1e-5, 1, 256)
    job = Norm(x, type_, groups, act=1, in_place=True)
    job.launch()
    got = job.out.numpy()
    ref.check_float(got, want, err, type_)
    apart = Norm(x, type_, groups, act=1)
    apart.launch()
    np.testing.assert_array_equal(apart.out.numpy().reshape(-1), got.reshape(-1).view(np.uint8))


def test_samples_past_a_launch():
    # 64 threads a sample: a launch has room for 62.9 million
    n = 65_000_000
    rng = np.random.default_rng(1)
    x = rng.integers(-1000, 1000, (n, 1, 2)).astype(np.float16)
    job = Norm(x, ref.F16, 1, act=0)
    job.launch()
    got = job.out.numpy().view(np.float16).reshape(n, 2)
    for i in range(0, n, 5_000_000):
        part = x[i:i + 5_000_000, 0].astype(np.float32)
        half = (part[:, 0] - part[:, 1]) / 2                 # (exact)
        y = half / np.sqrt(half.astype(np.float64) ** 2 + 1e-5)
        # a result's own rounding, and a few of 32 bits on its way, |y| <= 1
        bound = 2.0 ** -11 * np.abs(y) + 16 * 2.0 ** -24
        assert np.all(np.abs(got[i:i + 5_000_000, 0] - y) <= bound) and np.all(np.abs(got[i:i + 5_000_000, 1] + y) <= bound)


def test_rows_past_a_launch():
    # 2^23 workgroups of sixteen rows, and some more that the first of them take in a second turn
    rows, cols, period = (1 << 27) + 1000, 2, 4099
    table = ref.to_type(np.random.default_rng(2).normal(0, 3, (period, cols)), ref.F16)
    packed = ref.rows_of(ref.to_f64(table, ref.F16))
    back = ref.to_type(ref.values(packed, cols), ref.F16)
    times = -(-rows // period)
    x = capi.to_device(np.tile(table, (times, 1))[:rows])
    row = capi.mx4_row_bytes(cols)
    q = capi.DeviceBuffer(rows * row)
    capi.launch_mx4_quantize(q, row, x, ref.F16, 2 * cols, rows, cols)
    capi.sync()
    for start in (0, (1 << 27) - 2000, rows - 3000):
        got = np.empty((3000, row), np.uint8)
        capi.check(capi.lib().mi355x_memcpy_d2h(capi._vp(got), capi._vp(q.ptr + start * row), capi._sz(got.nbytes), None))
        capi.sync()
        np.testing.assert_array_equal(got, packed[(start + np.arange(3000)) % period])
    x.fill(0xEE)
    capi.launch_mx4_dequantize(x, ref.F16, 2 * cols, q, row, rows, cols)
    got = x.numpy()
    whole = rows // period * period
    assert (got[:whole].reshape(-1, period, cols) == back).all() and (got[whole:] == back[:rows - whole]).all()


def test_two_group_norms_at_once():
    rng = np.random.default_rng(3)
    jobs = []
    for n, pixels, C, groups, type_, out_type in ((2, 9000, 128, 8, ref.F16, None), (40, 300, 100, 4, ref.F32, ref.MX4)):
        x = image(rng, n, pixels, C, type_)
        jobs.append((Norm(x, type_, groups, act=6, out_type=out_type, stream=capi.Stream()), x, groups, type_, out_type))
    for _ in range(6):
        for job, *_ in jobs:
            job.launch()
    for job, x, groups, type_, out_type in jobs:
        want, err = group_norm_ref.norm(ref.to_f64(x, type_), groups, None, None, 1e-5, 6, 256)
        got = job.out.numpy(job.stream)
        if out_type == ref.MX4:
            C = x.shape[2]
            ref.check_mx4(got, C, want.reshape(-1, C), err.reshape(-1, C))
        else:
            ref.check_float(got.view(x.dtype).reshape(x.shape), want, err, type_)


def test_equal_calls_give_equal_bits():
    """A norm with SiLU to microscaled rows and the product over them, with other calls between and
    other bits in every buffer that they write."""
    rng = np.random.default_rng(4)
    n, pixels, C, groups, wide = 32, 784, 512, 32, 128
    norm = Norm(image(rng, n, pixels, C, ref.BF16), ref.BF16, groups, act=6, out_type=ref.MX4)
    other = Norm(image(rng, 3, 700, C, ref.BF16), ref.BF16, groups, act=6, out_type=ref.MX4)
    w = ref.rows_of(rng.normal(0, C ** -0.5, (wide, C)))
    dw, db = capi.to_device(w), capi.to_device(rng.normal(0, 0.1, wide).astype(np.float32))
    out = capi.DeviceBuffer.empty((n * pixels, wide), np.uint16)
    first = None
    for i in range(12):
        for b in (norm.out, norm.ws, out):
            b.fill(i * 37 % 256)
        if i % 3 == 2:
            other.launch()
        norm.launch()
        capi.launch_mx4_fc(out, ref.BF16, 2 * wide, norm.out, ref.MX4, norm.row, dw, w.shape[1], db, n * pixels, C, wide)
        got = (norm.out.numpy(), out.numpy())
        first = first or got
        for a, b in zip(got, first):
            np.testing.assert_array_equal(a, b)
