"""Products of microscaled rows with low-rank adapters of each row's own, against 64 bits."""
import numpy as np
import pytest

from glow_amd import capi
from tests import mx4_ref as ref

pytestmark = pytest.mark.gpu
TYPES = [ref.F32, ref.F16, ref.BF16]


@pytest.fixture(scope="module", autouse=True)
def _device():
    capi.init(0)


class Case:
    def __init__(self, rng, M, K, N, rank, count, in_type, type_, bias=True, scales=True, none=0.2, runs=1):
        x = rng.normal(0, 1, (M, K)) * 10.0 ** rng.uniform(-1, 1, (M, 1))
        if in_type == ref.MX4:
            self.x = ref.rows_of(x)
            self.shared = self.own = ref.values(self.x, K)
        else:
            self.x = ref.to_type(x, in_type)
            self.own = ref.to_f64(self.x, in_type)
            self.shared = ref.values(ref.rows_of(self.own), K)
        self.w = ref.rows_of(rng.normal(0, max(K, 1) ** -0.5, (N, K)))
        self.b = rng.normal(0, 1, N).astype(np.float32) if bias else None
        self.down = ref.to_type(rng.normal(0, max(K, 1) ** -0.5, (count, rank, K)), type_)
        self.up = ref.to_type(rng.normal(0, 1, (count, N, rank)), type_)
        self.scales = np.exp(rng.normal(0, 1, count)).astype(np.float32) if scales else None
        ids = rng.integers(0, max(count, 1), -(-M // runs))
        ids = np.where(rng.random(ids.size) < none, rng.choice([-1, count, 2 ** 31 - 1, -2 ** 31], ids.size), ids)
        self.ids = np.repeat(ids, runs)[:M].astype(np.int32)
        self.K, self.N, self.in_type, self.type_, self.count = K, N, in_type, type_, count

    def run(self, out_type, act=0):
        return capi.mx4_fc_adapters(self.x, self.in_type, self.w, self.b, self.K, self.down, self.up, self.ids, self.scales,
                                    self.type_, out_type, act)

    def want(self, act=0):
        """(results, bound of the error before the result's own rounding): the sums of the shared product, of down and of
        up in any order, each rounded or cut to 24 bits, what goes on from down in 24 bits, and the last sums."""
        w = ref.values(self.w, self.K)
        v, mag = self.shared @ w.T, np.abs(self.shared) @ np.abs(w).T
        err = (self.K + 2) * 2.0 ** -23 * mag
        for a in range(self.count):
            rows = self.ids == a
            down, up = ref.to_f64(self.down[a], self.type_), ref.to_f64(self.up[a], self.type_)
            s = 1.0 if self.scales is None else float(self.scales[a])
            low = self.own[rows] @ down.T * s
            low_err = (self.K + 10) * 2.0 ** -23 * (np.abs(self.own[rows]) @ np.abs(down).T) * s
            part = np.abs(low) @ np.abs(up).T
            v[rows] += low @ up.T
            err[rows] += low_err @ np.abs(up).T + (up.shape[1] + 10) * 2.0 ** -23 * part
            mag[rows] += part
        if self.b is not None:
            v, mag = v + self.b, mag + np.abs(self.b)
        err += 4 * 2.0 ** -23 * mag
        return ref.activate(v, act), ref.act_error(v, err, act)

    def check(self, out_type, act=0):
        want, err = self.want(act)
        got = self.run(out_type, act)
        if out_type == ref.MX4:
            ref.check_mx4(got, self.N, want, err)
        else:
            ref.check_float(got, want, err, out_type)
        return got


# every kind of tile of the product, odd sizes, ranks up to several steps of 32 and of 64
SHAPES = [(1, 1, 1, 1), (1, 4096, 64, 16), (3, 129, 33, 5), (17, 512, 48, 33), (61, 415, 509, 5), (33, 300, 129, 64),
          (64, 1024, 256, 16), (130, 640, 130, 70), (300, 96, 64, 8), (257, 130, 1000, 3), (600, 700, 520, 32),
          (1100, 257, 640, 9), (2048, 1024, 1100, 17)]


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("in_type", TYPES + [ref.MX4])
@pytest.mark.parametrize("M, K, N, rank", SHAPES)
def test_adapters(M, K, N, rank, in_type, type_):
    rng = np.random.default_rng(M + K + N + rank)
    out_type = type_ if (M + K) % 3 else ref.MX4
    Case(rng, M, K, N, rank, 7, in_type, type_, runs=1 + M % 5).check(out_type, act=(0, 1, 6)[M % 3])


@pytest.mark.parametrize("out_type", TYPES + [ref.MX4])
@pytest.mark.parametrize("M, K, N", [(16, 4096, 512), (40, 256, 512), (96, 1024, 1024), (2000, 300, 512), (4096, 512, 2304),
                                     (1500, 1500, 1500), (4096, 640, 4096)])
def test_results_of_every_type(M, K, N, out_type):
    rng = np.random.default_rng(M + K)
    Case(rng, M, K, N, 16, 5, ref.BF16, ref.BF16, bias=False, scales=False, runs=37).check(out_type)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("M", [1, 16, 40, 700])
def test_one_adapter_many_and_none(M, type_):
    rng = np.random.default_rng(M)
    for none, count, runs in ((0, 1, 1), (0, 300, 1), (1, 3, 1), (0.5, 2, 16)):
        c = Case(rng, M, 512, 200, 12, count, ref.BF16, type_, none=none, runs=runs)
        got = c.check(ref.F32)
        if none == 1:
            np.testing.assert_array_equal(got, capi.mx4_fc(c.x, c.in_type, c.w, c.b, c.K))


@pytest.mark.parametrize("M, K, N", [(20, 300, 100), (300, 200, 400), (1200, 1024, 600)])
def test_what_is_in_an_adapter_stays_with_its_rows(M, K, N):
    rng = np.random.default_rng(M)
    for type_ in TYPES:
        c = Case(rng, M, K, N, 6, 4, ref.F16, type_)
        good = c.run(ref.F32)
        for a in (c.down, c.up):
            bits = a[2].reshape(-1)
            bits[::7] = 0x7fc0 if type_ == ref.BF16 else np.nan
            bits[3::7] = 0x7f80 if type_ == ref.BF16 else np.inf
        got = c.run(ref.F32)
        np.testing.assert_array_equal(got[c.ids != 2], good[c.ids != 2])
        assert np.isnan(got[c.ids == 2]).any()


def test_nothing_beside_the_product():
    rng = np.random.default_rng(1)
    for M, K, N, rank, count in ((5, 100, 30, 0, 3), (5, 100, 30, 4, 0), (5, 0, 30, 4, 2)):
        c = Case(rng, M, K, N, rank, count, ref.F32, ref.F32, none=0)
        np.testing.assert_array_equal(c.run(ref.F32), capi.mx4_fc(c.x, ref.F32, c.w, c.b, K))
    c = Case(rng, 5, 100, 30, 4, 2, ref.F32, ref.F32)
    assert capi.mx4_fc_adapters(c.x[:0], ref.F32, c.w, c.b, 100, c.down, c.up, c.ids[:0], c.scales).shape == (0, 30)
