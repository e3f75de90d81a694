"""Microscaled 4-bit rows on the device: quantisation bit for bit, and products against 64
bits within the rounding of 32-bit sums."""
import numpy as np
import pytest

from glow_amd import capi
from tests import mx4_ref as ref
from tests.test_host_mx4 import special_rows

pytestmark = pytest.mark.gpu
TYPES = [ref.F32, ref.F16, ref.BF16]


@pytest.fixture(scope="module", autouse=True)
def _device():
    capi.init(0)


def spread(rng, rows, cols):
    return rng.normal(0, 1, (rows, cols)) * 10.0 ** rng.uniform(-2, 2, (rows, 1))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 32), (3, 33), (5, 127), (2, 128), (7, 129), (61, 415), (33, 1000),
                                        (1, 5000), (4, 2049), (300, 13), (1, 65537), (8197, 2049), (270000, 65)])
def test_quantize_is_the_definition(type_, rows, cols):
    x = ref.to_type(spread(np.random.default_rng(rows * cols), rows, cols), type_)
    np.testing.assert_array_equal(capi.mx4_quantize(x, type_), ref.rows_of(ref.to_f64(x, type_)))


def test_quantize_of_special_values():
    x = special_rows()
    with np.errstate(invalid="ignore"):
        for cols in (31, 127, 415):
            np.testing.assert_array_equal(capi.mx4_quantize(x[:, :cols].copy()), ref.rows_of(x[:, :cols]))


@pytest.mark.parametrize("type_", [ref.F16, ref.BF16])
def test_quantize_of_every_16_bit_value(type_):
    # each value beside a larger one of a few binades, so that all its bits meet every scale
    bits = np.arange(65536, dtype=np.uint16)
    x = np.zeros((65536, 33), np.uint16)
    x[:, 0] = bits
    x[:, 32] = bits
    sign_and_exponent = bits & (0xfc00 if type_ == ref.F16 else 0xff80)
    step = 0x400 if type_ == ref.F16 else 0x80
    x[:, 5] = np.where((sign_and_exponent & 0x7fff) < (0x7000 if type_ == ref.F16 else 0x7c00),
                       sign_and_exponent + step * (bits % 4), 0)
    x = x.view(np.float16) if type_ == ref.F16 else x
    with np.errstate(invalid="ignore"):
        want = ref.rows_of(ref.to_f64(x, type_))
    np.testing.assert_array_equal(capi.mx4_quantize(x, type_), want)


@pytest.mark.parametrize("type_", TYPES)
def test_strided_rows_leave_the_rest_alone(type_):
    rng = np.random.default_rng(5)
    rows, cols, size = 37, 205, 4 if type_ == ref.F32 else 2
    x = ref.to_type(spread(rng, rows, cols + 11), type_)
    flat = capi.to_device(np.concatenate([x.reshape(-1), x.reshape(-1)[:8]]))
    pitch = capi.mx4_row_bytes(cols) + 48
    out = capi.to_device(np.full((rows, pitch), 0xA5, np.uint8))
    # rows that start one element into the buffer, eleven elements apart
    capi.launch_mx4_quantize(out.ptr, pitch, flat.ptr + size, type_, (cols + 11) * size, rows, cols)
    got = out.numpy()
    seen = np.concatenate([x.reshape(-1), x.reshape(-1)[:8]])[1:1 + rows * (cols + 11)].reshape(rows, -1)[:, :cols]
    n = capi.mx4_row_bytes(cols)
    np.testing.assert_array_equal(got[:, :n], ref.rows_of(ref.to_f64(seen, type_)))
    assert (got[:, n:] == 0xA5).all()
    back = capi.to_device(np.full((rows, (cols + 3) * size), 0xA5, np.uint8))
    capi.launch_mx4_dequantize(back.ptr + size, type_, (cols + 3) * size, out.ptr, pitch, rows - 1, cols)
    b = back.numpy().reshape(-1)
    view = b[size:size + (rows - 1) * (cols + 3) * size].reshape(rows - 1, -1)
    vals = np.ascontiguousarray(view[:, :cols * size]).view(x.dtype)
    np.testing.assert_array_equal(vals, ref.to_type(ref.values(got[:rows - 1, :n], cols), type_))
    assert (view[:, cols * size:] == 0xA5).all() and (b[:size] == 0xA5).all()
    assert (b[size + (rows - 1) * (cols + 3) * size:] == 0xA5).all()


@pytest.mark.parametrize("type_", TYPES)
def test_dequantize_of_every_scale_and_code(type_):
    codes = np.tile(np.arange(16, dtype=np.uint8), (256, 8))
    byte = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 4, 1)
    rows = ref.pack(codes, byte)
    with np.errstate(over="ignore"):
        want = ref.values(rows, 128).astype(np.float32)     # 6 * 2^127 is an infinity in 32 bits
    got = capi.mx4_dequantize(rows, 128, type_)
    want = ref.to_type(want, type_)
    if type_ == ref.BF16:
        nan = byte[:, :1] == 255
        np.testing.assert_array_equal(np.where(nan, 0, got), np.where(nan, 0, want))
        assert np.isnan(ref.to_f64(got[255:], type_)).all()
    else:
        np.testing.assert_array_equal(got, want)


# ---- products --------------------------------------------------------------------------

def product(rng, M, K, N, in_type):
    x = spread(rng, M, K)
    w = ref.rows_of(rng.normal(0, K ** -0.5 if K else 1, (N, K)))
    if in_type == ref.MX4:
        rows = ref.rows_of(x)
        return rows, ref.values(rows, K), w
    x = ref.to_type(x, in_type)
    return x, ref.values(ref.rows_of(ref.to_f64(x, in_type)), K), w


def check(got, want, err, out_type, N):
    if out_type == ref.MX4:
        ref.check_mx4(got, N, want, err)
    else:
        ref.check_float(got, want, err, out_type)


SHAPES = [(1, 1, 1), (1, 32, 5), (2, 33, 31), (3, 129, 33), (7, 128, 64), (16, 257, 100), (17, 512, 48), (33, 300, 129),
          (61, 415, 509), (64, 1024, 256), (65, 130, 257), (130, 640, 130), (257, 96, 300), (1, 4096, 1000), (300, 64, 1),
          (5, 8200, 70), (512, 512, 512)]


@pytest.mark.parametrize("M, K, N", SHAPES)
@pytest.mark.parametrize("in_type", [ref.F32, ref.F16, ref.BF16, ref.MX4])
def test_fc(M, K, N, in_type):
    rng = np.random.default_rng(M * 7 + K * 3 + N)
    x, a, w = product(rng, M, K, N, in_type)
    bias = rng.normal(0, 1, N).astype(np.float32)
    # every result type and activation over the shapes
    out_type, act = (M + K + in_type) % 4, (0, 1, 6)[(M + N + in_type) % 3]
    want, err = ref.fc(a, ref.values(w, K), bias.astype(np.float64), act)
    check(capi.mx4_fc(x, in_type, w, bias, K, out_type, act), want, err, out_type, N)


@pytest.mark.parametrize("out_type", [ref.F32, ref.F16, ref.BF16, ref.MX4])
@pytest.mark.parametrize("M, K, N", [(4, 200, 70), (150, 300, 290), (600, 256, 516)])
def test_fc_results_of_every_type(M, K, N, out_type):
    rng = np.random.default_rng(out_type)
    x, a, w = product(rng, M, K, N, ref.MX4)
    for act in (0, 1, 6):
        want, err = ref.fc(a, ref.values(w, K), None, act)
        check(capi.mx4_fc(x, ref.MX4, w, None, K, out_type, act), want, err, out_type, N)


@pytest.mark.parametrize("out_type", [ref.F32, ref.F16, ref.BF16, ref.MX4])
@pytest.mark.parametrize("M, K, N", [(1801, 150, 2003), (1793, 1040, 1798), (3201, 160, 4098), (3090, 1300, 3851), (3000, 512, 3001),
                                     (1990, 650, 150), (10000, 385, 65)])
def test_fc_of_large_results(M, K, N, out_type):
    # the tiles of 128 and 256: one step of K and two, an odd count past a group of scales
    rng = np.random.default_rng(M + out_type)
    x, a, w = product(rng, M, K, N, ref.MX4)
    bias = rng.normal(0, 1, N).astype(np.float32)
    act = (0, 1, 6)[(K + out_type) % 3]
    want, err = ref.fc(a, ref.values(w, K), bias.astype(np.float64), act)
    check(capi.mx4_fc(x, ref.MX4, w, bias, K, out_type, act), want, err, out_type, N)


@pytest.mark.parametrize("in_type", [ref.F32, ref.F16, ref.BF16])
@pytest.mark.parametrize("M, K, N", [(1, 4096, 70), (4, 515, 3000), (186, 895, 792), (186, 894, 792), (40, 895, 400), (3, 5000, 40), (2, 130, 33), (1, 49152, 20), (4, 6100, 18), (1, 24576, 50), (31, 96, 700), (90, 1050, 290), (1990, 13, 300),
                                     (2000, 511, 190), (700, 300, 2000)])
def test_float_inputs_give_what_their_rows_give(M, K, N, in_type):
    """Quantised by the product or in front of it: the same bits."""
    rng = np.random.default_rng(K)
    x, _, w = product(rng, M, K, N, in_type)
    rows = capi.mx4_quantize(x, in_type)
    for out_type in (ref.F32, ref.MX4):
        np.testing.assert_array_equal(capi.mx4_fc(x, in_type, w, None, K, out_type),
                                      capi.mx4_fc(rows, ref.MX4, w, None, K, out_type))


@pytest.mark.parametrize("M, N", [(1, 40), (20, 200), (300, 300)])
def test_fc_of_no_columns_is_the_bias(M, N):
    bias = np.linspace(-2, 2, N).astype(np.float32)
    got = capi.mx4_fc(np.zeros((M, 0), np.float32), ref.F32, np.zeros((N, 0), np.uint8), bias, 0, ref.F32, 1)
    np.testing.assert_array_equal(got, np.tile(np.maximum(bias, 0), (M, 1)))
    assert not capi.mx4_fc(np.zeros((M, 0), np.float32), ref.F32, np.zeros((N, 0), np.uint8), None, 0, ref.F16).any()


@pytest.mark.parametrize("M", [1, 9, 40, 200])
def test_nan_blocks_and_far_scales(M):
    rng = np.random.default_rng(M)
    K, N = 300, 150
    x, _, w = product(rng, M, K, N, ref.MX4)
    x, w = x.copy(), w.copy()
    p = ref.groups(K)
    x[M // 2, 64 * p + 3] = 255                 # a NaN block of one input row
    w[7, 64 * p + 9] = 255                      # and of one weight row, in its last, short block
    x[0, 64 * p:64 * p + 10] = 20               # 2^-107
    w[11, 64 * p:64 * p + 10] = 0               # with this: below every number of 32 bits
    w[12, 64 * p:64 * p + 10] = 250             # 2^123
    for out_type in (ref.F32, ref.MX4):
        with np.errstate(invalid="ignore"):
            want, err = ref.fc(ref.values(x, K), ref.values(w, K), None, 1)
        got = capi.mx4_fc(x, ref.MX4, w, None, K, out_type, 1)
        if out_type == ref.F32:
            # (a single row's NaN byte has been overwritten by the far scales)
            assert np.isnan(got[:, 7]).all() and (M == 1 or np.isnan(got[M // 2]).all())
        check(got, want, err, out_type, N)


@pytest.mark.parametrize("out_type", [ref.F32, ref.BF16, ref.MX4])
@pytest.mark.parametrize("in_type", [ref.F16, ref.MX4])
@pytest.mark.parametrize("M, K, N", [(3, 130, 45), (70, 260, 140), (290, 200, 270)])
def test_fc_of_strided_rows_leaves_the_rest_alone(M, K, N, in_type, out_type):
    rng = np.random.default_rng(M)
    x, a, w = product(rng, M, K, N, in_type)
    bias = rng.normal(0, 1, N).astype(np.float32)
    x8 = np.ascontiguousarray(x).view(np.uint8).reshape(M, -1)
    gap = 32 if in_type == ref.MX4 else 6
    wide = np.full((M, x8.shape[1] + gap), 0xFF, np.uint8)
    wide[:, :x8.shape[1]] = x8
    wide_w = np.full((N, w.shape[1] + 16), 0xFF, np.uint8)
    wide_w[:, :w.shape[1]] = w
    size = {ref.F32: 4, ref.BF16: 2, ref.MX4: 0}[out_type]
    row = capi.mx4_row_bytes(N) if out_type == ref.MX4 else N * size
    pitch = row + (16 if out_type == ref.MX4 else 3 * size)
    out = capi.to_device(np.full((M + 1, pitch), 0xA5, np.uint8))
    dx, dw, db = capi.to_device(wide), capi.to_device(wide_w), capi.to_device(bias)
    n = capi.mx4_fc_workspace_bytes(M, K, N, in_type)
    ws = capi.DeviceBuffer(max(n, 1))
    capi.launch_mx4_fc(out, out_type, pitch, dx, in_type, wide.shape[1], dw, wide_w.shape[1], db, M, K, N, 0,
                       ws if n else None, n)
    got = out.numpy()
    want, err = ref.fc(a, ref.values(w, K), bias.astype(np.float64), 0)
    assert (got[M] == 0xA5).all() and (got[:, row:] == 0xA5).all()
    body = np.ascontiguousarray(got[:M, :row])
    if out_type != ref.MX4:
        body = body.view(np.float32 if out_type == ref.F32 else np.uint16)
    check(body, want, err, out_type, N)


@pytest.mark.parametrize("seed", range(60))
def test_fc_of_random_shapes(seed):
    rng = np.random.default_rng(2000 + seed)
    M, K, N = (int(np.exp(rng.uniform(0, np.log(top)))) for top in (3000, 3000, 3000))
    while M * K * N > 2_000_000_000:
        K = max(1, K // 2)
    in_type, out_type, act = int(rng.integers(0, 4)), int(rng.integers(0, 4)), int(rng.choice([0, 1, 6]))
    x, a, w = product(rng, M, K, N, in_type)
    bias = rng.normal(0, 1, N).astype(np.float32) if rng.random() < 0.7 else None
    want, err = ref.fc(a, ref.values(w, K), None if bias is None else bias.astype(np.float64), act)
    got = capi.mx4_fc(x, in_type, w, bias, K, out_type, act)
    check(got, want, err, out_type, N)
    np.testing.assert_array_equal(capi.mx4_fc(x, in_type, w, bias, K, out_type, act), got)   # equal calls, equal bits


class FarRows:
    """Rows of device memory `pitch` bytes apart, over 4 GiB in all."""

    def __init__(self, rows, pitch):
        self.rows, self.pitch = rows, pitch
        self.memory = capi.DeviceBuffer((rows - 1) * pitch + (1 << 20))

    def put(self, a):
        a = np.ascontiguousarray(a)
        for r in range(self.rows):
            capi.check(capi.lib().mi355x_memcpy_h2d(capi._vp(self.memory.ptr + r * self.pitch), capi._vp(a[r]),
                                                    capi._sz(a[r].nbytes), None))
        capi.sync()
        return self

    def get(self, cols, dtype):
        out = np.empty((self.rows, cols), dtype)
        capi.sync()
        for r in range(self.rows):
            capi.check(capi.lib().mi355x_memcpy_d2h(capi._vp(out[r]), capi._vp(self.memory.ptr + r * self.pitch),
                                                    capi._sz(out[r].nbytes), None))
        capi.sync()
        return out


@pytest.mark.parametrize("M, K, N", [(3, 200, 3), (290, 256, 290), (290, 700, 290)])
def test_rows_past_4_gib(M, K, N):
    rng = np.random.default_rng(K)
    pitch = (5 << 30) // (min(M, N) - 1) // 16 * 16
    x, a, w = product(rng, M, K, N, ref.F16)
    want, err = ref.fc(a, ref.values(w, K), None, 0)
    far_x, far_w = FarRows(M, pitch).put(x), FarRows(N, pitch).put(w)
    far_q, far_out = FarRows(M, pitch), FarRows(M, pitch)
    capi.launch_mx4_quantize(far_q.memory, pitch, far_x.memory, ref.F16, pitch, M, K)
    rows = ref.rows_of(ref.to_f64(x, ref.F16))
    np.testing.assert_array_equal(far_q.get(rows.shape[1], np.uint8), rows)
    capi.launch_mx4_fc(far_out.memory, ref.F32, pitch, far_q.memory, ref.MX4, pitch, far_w.memory, pitch, None, M, K, N)
    ref.check_float(far_out.get(N, np.float32), want, err, ref.F32)
    n = capi.mx4_fc_workspace_bytes(M, K, N, ref.F16)
    ws = capi.DeviceBuffer(max(n, 1))
    capi.launch_mx4_fc(far_out.memory, ref.MX4, pitch, far_x.memory, ref.F16, pitch, far_w.memory, pitch, None, M, K, N, 0,
                       ws if n else None, n)
    ref.check_mx4(far_out.get(capi.mx4_row_bytes(N), np.uint8), N, want, err)
    capi.launch_mx4_dequantize(far_x.memory, ref.F16, pitch, far_q.memory, pitch, M, K)
    np.testing.assert_array_equal(far_x.get(K, np.float16), ref.to_type(ref.values(rows, K), ref.F16))
    # and the pixels of a group norm
    C, groups = min(K, 64), 4
    y, yerr = ref.group_norm(a[None, :, :C], groups, None, None, 1e-5, 1)
    wsn = capi.group_norm_workspace_bytes(1, M, C, groups)
    ws = capi.DeviceBuffer(wsn)
    capi.launch_group_norm(far_out.memory, ref.F16, pitch, far_x.memory, ref.F16, pitch, None, None, 1, M, C, groups, 1e-5,
                           1, ws, wsn)
    ref.check_float(far_out.get(C, np.float16)[None], y, yerr, ref.F16)


@pytest.mark.parametrize("M, N", [(2, 100), (40, 2000), (2100, 2100)])
def test_first_call_inside_a_capture(M, N):
    """Nothing has to have run before: attributes of a kernel are no stream's work."""
    rng = np.random.default_rng(N)
    K = 640
    x, a, w = product(rng, M, K, N, ref.MX4)
    dx, dw, stream = capi.to_device(x), capi.to_device(w), capi.Stream()
    out = capi.DeviceBuffer.empty((M, N), np.float16)
    with capi.Graph(stream) as graph:
        capi.launch_mx4_fc(out, ref.F16, 2 * N, dx, ref.MX4, x.shape[1], dw, w.shape[1], None, M, K, N, 0, None, 0, stream)
    want, err = ref.fc(a, ref.values(w, K), None, 0)
    for _ in range(3):
        out.fill(0xEE, stream)
        graph.launch(stream)
        check(out.numpy(stream), want, err, ref.F16, N)
        capi.sync()


def test_two_streams_at_once():
    rng = np.random.default_rng(77)
    shapes = [(700, 600, 900), (5, 900, 3000)]
    jobs = []
    for M, K, N in shapes:
        x, a, w = product(rng, M, K, N, ref.F16)
        n = capi.mx4_fc_workspace_bytes(M, K, N, ref.F16)
        jobs.append((M, K, N, capi.to_device(x), capi.to_device(w), w.shape[1], capi.DeviceBuffer(max(n, 1)), n,
                     capi.DeviceBuffer.empty((M, N), np.float32), capi.Stream(), ref.fc(a, ref.values(w, K), None, 0)))
    for _ in range(4):
        for M, K, N, dx, dw, pitch, ws, n, out, stream, _ in jobs:
            capi.launch_mx4_fc(out, ref.F32, 4 * N, dx, ref.F16, 2 * K, dw, pitch, None, M, K, N, 0, ws if n else None, n,
                               stream)
    for M, K, N, *_, out, stream, (want, err) in jobs:
        check(out.numpy(stream), want, err, ref.F32, N)


def test_tower_hands_rows_on_and_replays():
    """Three layers as a ranking net runs them, on a stream of their own and from a graph that
    is replayed with other inputs, the library's own work between the replays."""
    rng = np.random.default_rng(3)
    M, sizes = 130, (13, 512, 256, 64)
    stream = capi.Stream()
    weights = [ref.rows_of(rng.normal(0, k ** -0.5, (n, k))) for k, n in zip(sizes, sizes[1:])]
    biases = [rng.normal(0, 0.1, n).astype(np.float32) for n in sizes[1:]]
    dw, db = [capi.to_device(w) for w in weights], [capi.to_device(b) for b in biases]
    dx = capi.DeviceBuffer.empty((M, sizes[0]), np.float32)
    hidden = [capi.DeviceBuffer.empty((M, capi.mx4_row_bytes(n)), np.uint8) for n in sizes[1:3]]
    out = capi.DeviceBuffer.empty((M, sizes[3]), np.float32)
    n = max(capi.mx4_fc_workspace_bytes(M, sizes[0], sizes[1], capi.TYPE_F32), 1)
    ws = capi.DeviceBuffer(n)

    def launch():
        src, kind, pitch = dx, capi.TYPE_F32, sizes[0] * 4
        for i, (k, cols) in enumerate(zip(sizes, sizes[1:])):
            dst = hidden[i] if i < 2 else out
            capi.launch_mx4_fc(dst, capi.TYPE_MX4 if i < 2 else capi.TYPE_F32, dst.shape[1] * dst.dtype.itemsize, src,
                               kind, pitch, dw[i], weights[i].shape[1], db[i], M, k, cols, capi.ACT_RELU, ws, n, stream)
            src, kind, pitch = dst, capi.TYPE_MX4, dst.shape[1]

    def inputs(i):
        return np.random.default_rng(i).normal(0, 1, (M, sizes[0])).astype(np.float32)

    eager = []
    for i in range(3):
        dx.upload(inputs(i), stream)
        launch()
        eager.append((hidden[0].numpy(stream), hidden[1].numpy(stream), out.numpy(stream)))
    a = ref.values(ref.rows_of(inputs(0)), sizes[0])
    for got, w, b, k, cols in zip(eager[0], weights, biases, sizes, sizes[1:]):
        want, err = ref.fc(a, ref.values(w, k), b.astype(np.float64), 1)
        if cols == sizes[3]:
            ref.check_float(got, want, err, ref.F32)
        else:
            ref.check_mx4(got, cols, want, err)
            a = ref.values(got, cols)
    with capi.Graph(stream) as graph:
        launch()
    for i in (2, 0, 1, 1, 2):
        dx.upload(inputs(i), stream)
        for h in (*hidden, out):
            h.fill(0xEE, stream)
        graph.launch(stream)
        for got, want in zip((hidden[0].numpy(stream), hidden[1].numpy(stream), out.numpy(stream)), eager[i]):
            np.testing.assert_array_equal(got, want)
        capi.sync()
