"""Microscaled 4-bit rows, their product and group norm from their definitions, in numpy and
64 bits."""
import numpy as np

VALUES = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
BORDERS = (VALUES[1:] + VALUES[:-1]) / 2
F32, F16, BF16, MX4 = range(4)
#: Half a step of each type relative to the value: what a rounding is off by at most.
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def to_type(x, type_):
    """float array -> the type's array (bfloat16: uint16 bits, rounded to nearest even)."""
    if type_ == F32:
        return np.asarray(x, np.float32)
    if type_ == F16:
        with np.errstate(over="ignore"):
            return np.asarray(x, np.float32).astype(np.float16)
    bits = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    nan = np.isnan(np.asarray(x, np.float32))
    up = (bits + 0x7fff + ((bits >> 16) & 1)) >> 16
    return np.where(nan, 0x7fc0, up).astype(np.uint16)


def to_f64(x, type_):
    if type_ == BF16:
        return (x.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return x.astype(np.float64)


def groups(cols):
    return -(-cols // 128)


def row_bytes(cols):
    return -(-groups(cols) * 68 // 16) * 16


def scale_bytes(most):
    """E8M0 bytes of blocks whose largest magnitudes are `most` (64 bits)."""
    most = np.asarray(most, np.float64)
    fine = np.isfinite(most)
    _, e = np.frexp(np.where(fine & (most > 0), most, 1.0))
    byte = np.maximum(e - 1 - 2, -127) + 127
    return np.where(fine, np.where(most > 0, byte, 0), 255).astype(np.int64)


def codes_of(v):
    """E2M1 codes of finite values that are scaled to their block."""
    a = np.abs(v)
    low = np.searchsorted(BORDERS, a, side="left")     # on a border: the lower code
    high = np.searchsorted(BORDERS, a, side="right")
    code = np.where(low % 2 == 0, low, high)
    return (code + 8 * np.signbit(v)).astype(np.uint8)


def quantize(x):
    """x [rows, cols] (64 bits) -> codes [rows, 128 * groups], bytes [rows, 4 * groups]."""
    rows, cols = x.shape
    p = groups(cols)
    padded = np.zeros((rows, 128 * p))
    padded[:, :cols] = x
    blocks = padded.reshape(rows, 4 * p, 32)
    byte = scale_bytes(np.abs(blocks).max(-1) if cols else np.zeros((rows, 0)))
    with np.errstate(invalid="ignore"):
        v = np.where(byte[..., None] == 255, 0.0, blocks / 2.0 ** np.minimum(byte - 127.0, 127)[..., None])
    return codes_of(v).reshape(rows, -1), byte.astype(np.uint8)


def pack(codes, byte):
    rows, p = codes.shape[0], byte.shape[1] // 4
    out = np.zeros((rows, -(-p * 68 // 16) * 16), np.uint8)
    out[:, :64 * p] = codes[:, 0::2] | (codes[:, 1::2] << 4)
    out[:, 64 * p:68 * p] = byte
    return out


def rows_of(x):
    return pack(*quantize(np.asarray(x, np.float64)))


def unpack(rows, cols):
    """codes [rows, cols], bytes [rows, blocks of cols]."""
    p = groups(cols)
    c = np.stack((rows[:, :64 * p] & 15, rows[:, :64 * p] >> 4), -1).reshape(rows.shape[0], -1)
    return c[:, :cols], rows[:, 64 * p:64 * p + -(-cols // 32)]


def values(rows, cols):
    """What rows stand for, 64 bits."""
    c, byte = unpack(rows, cols)
    v = np.where(c >= 8, -1.0, 1.0) * VALUES[c & 7]
    scale = np.where(byte == 255, np.nan, 2.0 ** (byte.astype(np.float64) - 127))
    return v * np.repeat(scale, 32, axis=1)[:, :cols]


def activate(v, act):
    if act == 1:
        return np.where(v < 0, 0.0, v)
    if act == 6:
        with np.errstate(over="ignore"):
            return v / (1 + np.exp(-v))
    return v


def act_error(v, err, act):
    """How far act(v') may be from act(v) for |v' - v| <= err, computed in 32 bits: SiLU's slope
    is below 1.1, and exp(-v) in 32 bits is off by its argument's rounding, |v| steps, and a few
    of its own, the sum and the division."""
    if act == 1:
        return err
    if act == 6:
        return 1.1 * err + np.abs(activate(v, 6)) * (8 + np.abs(v)) * 2.0 ** -23
    return err


def fc(a, w, bias, act):
    """(results, bound of the error before the result's own rounding) for 64-bit a, w."""
    v, mag = a @ w.T, np.abs(a) @ np.abs(w).T
    if bias is not None:
        v, mag = v + bias, mag + np.abs(bias)
    # any order of K sums, each rounded or cut to 24 bits, and the bias; nothing below 2^-126
    err = (a.shape[1] + 2) * 2.0 ** -23 * mag + a.shape[1] * 2.0 ** -126
    # partial sums may be up to `mag`: where that is past the range of 32 bits, a sum may be an
    # infinity, and the difference of two of them NaN, whatever the whole is
    err = np.where(mag < 3.4e38, err, np.inf)
    return activate(v, act), act_error(v, err, act)


def group_norm(x, n_groups, gamma, beta, eps, act):
    """(results, bound of the error before the result's own rounding), x [N, pixels, C]."""
    n, pixels, C = x.shape
    g = x.reshape(n, pixels, n_groups, C // n_groups)
    mean = g.mean((1, 3), keepdims=True)
    d = g - mean
    var = (d * d).mean((1, 3), keepdims=True)
    rstd = 1 / np.sqrt(var + eps)
    gamma = np.ones(C) if gamma is None else gamma.astype(np.float64)
    beta = np.zeros(C) if beta is None else beta.astype(np.float64)
    y = (d * rstd).reshape(x.shape) * gamma + beta
    # sums over a group in 32 bits: at least 64 lanes share one, so that no value passes through
    # more than count / 64 + 64 roundings
    count = pixels * (C // n_groups)
    steps = (count / 64 + 64) * 2.0 ** -24
    off = steps * np.abs(g).mean((1, 3), keepdims=True)
    rel = steps + (off * rstd) ** 2 + 8 * 2.0 ** -24
    err = ((off + np.abs(d) * (rel + 4 * 2.0 ** -24) + 2 * 2.0 ** -24 * np.abs(mean)) * rstd).reshape(x.shape)
    err = err * np.abs(gamma) + 4 * 2.0 ** -24 * (np.abs(y) + np.abs(beta))
    return activate(y, act), act_error(y, err, act)


def check_float(got, want, err, type_):
    """`got` (of the type) within `err` and its own rounding of `want`."""
    got = to_f64(got, type_)
    known = ~np.isinf(err)
    got, want, err = got[known], want[known], err[known]
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    least = 2.0 ** -25 if type_ == F16 else 0.0        # half a step of fp16's smallest numbers
    bound = np.where(fine, err, 0) + HALF_STEP[type_] * (np.abs(want) + np.where(fine, err, 0)) + least
    off = np.abs(np.where(fine, got - np.where(fine, want, 0), 0))
    assert np.all(off <= np.where(fine, bound, 0)), float(np.max(off / np.maximum(np.where(fine, bound, 1), 1e-300)))


def check_mx4(rows, cols, want, err):
    """Rows whose blocks are the quantised form of values within `err` of `want`: the scale is
    that of a largest magnitude in reach, each code that of a value in reach."""
    p = groups(cols)
    assert rows.shape[1] == row_bytes(cols)
    c, byte = unpack(rows, 128 * p)
    padded, e = np.zeros((rows.shape[0], 128 * p)), np.zeros((rows.shape[0], 128 * p))
    padded[:, :cols], e[:, :cols] = want, err
    assert not c[:, cols:].any() and not byte[:, -(-cols // 32):].any() and not rows[:, 68 * p:].any()
    blocks, e = padded.reshape(-1, 4 * p, 32), e.reshape(-1, 4 * p, 32)
    nan, known = ~np.isfinite(blocks).all(-1), ~np.isinf(e).any(-1)
    assert np.array_equal((byte == 255)[known], nan[known])
    nan = nan | ~known
    blocks, e = np.where(nan[..., None], 0, blocks), np.where(nan[..., None], 0, e)
    size = np.abs(blocks)
    low = scale_bytes(np.maximum(size - e, 0).max(-1))
    high = scale_bytes((size + e).max(-1))
    assert np.all(nan | ((low <= byte) & (byte <= high)))
    unit = 2.0 ** (np.where(nan, 0, byte.astype(np.float64)) - 127)[..., None]
    got = (np.where(c >= 8, -1.0, 1.0) * VALUES[c & 7]).reshape(blocks.shape)

    def nearest(v):
        v = v / unit
        return np.where(np.signbit(v), -1.0, 1.0) * VALUES[codes_of(v) & 7]
    assert np.all((nearest(blocks - e) <= got) & (got <= nearest(blocks + e)))
