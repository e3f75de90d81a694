"""The cache of microscaled rows on the device, and attention over it, against 64 bits."""
import numpy as np
import pytest

from glow_amd import capi
from tests import mx4_attention_ref as aref, mx4_ref as ref

pytestmark = pytest.mark.gpu
TYPES = [ref.F32, ref.F16, ref.BF16]


@pytest.fixture(scope="module", autouse=True)
def _device():
    capi.init(0)


def run(b, q, heads, type_, out_type=None, pages=..., **kw):
    return capi.mx4_attention(q, heads, b.keys, b.values, b.starts, b.lengths, b.kv_heads, b.head_dim, b.page_tokens,
                              b.pages if pages is ... else pages, type_=type_, out_type=out_type, **kw)


def queries(rng, b, heads, type_):
    x = rng.normal(0, 1.5, (b.rows, heads * b.head_dim)) * np.exp(0.5 * rng.normal(0, 1, heads * b.head_dim))
    return ref.to_type(x, type_)


def check(b, q, heads, type_, out_type=None, **kw):
    rows = capi.mx4_row_bytes(heads * b.head_dim) if out_type == ref.MX4 else heads * b.head_dim
    before = np.full((b.rows, rows), 0x5a, np.uint8 if out_type == ref.MX4 else q.dtype)
    got = run(b, q, heads, type_, out_type, out=before, **kw)
    want, err, used = aref.attention(b, ref.to_f64(q, type_), heads, type_, **kw)
    np.testing.assert_array_equal(got[~used], before[~used])
    if out_type == ref.MX4:
        ref.check_mx4(got[used], heads * b.head_dim, want[used], err[used])
    else:
        ref.check_float(got[used], want[used], err[used], type_)
    return got


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 33, 100, 257, 530]


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dim, kv_heads, group, page", [(64, 2, 4, 16), (64, 1, 1, 48), (64, 3, 3, 0), (128, 1, 8, 32),
                                                        (128, 8, 1, 16), (128, 3, 2, 0), (256, 1, 5, 64), (256, 2, 2, 0)])
def test_single_tokens(dim, kv_heads, group, page, type_):
    rng = np.random.default_rng(dim + kv_heads + group)
    b = aref.Batch(rng, LENGTHS, [min(1, t) for t in LENGTHS], kv_heads, dim, page or 32, bool(page), pad=2)
    heads = kv_heads * group
    q = queries(rng, b, heads, type_)
    check(b, q, heads, type_)
    check(b, q, heads, type_, ref.MX4)
    check(b, q, heads, type_, window=40, sinks=3)
    check(b, q, heads, type_, window=1)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dim, kv_heads, group, page", [(64, 3, 3, 16), (64, 1, 2, 0), (128, 2, 4, 48), (128, 1, 1, 0), (256, 1, 3, 16)])
def test_prompts(dim, kv_heads, group, page, type_):
    rng = np.random.default_rng(dim + kv_heads + group)
    lengths = [1, 5, 0, 64, 97, 130, 200]
    new = [1, 5, 0, 64, 33, 1, 130]
    b = aref.Batch(rng, lengths, new, kv_heads, dim, page or 64, bool(page), pad=3)
    heads = kv_heads * group
    q = queries(rng, b, heads, type_)
    check(b, q, heads, type_)
    check(b, q, heads, type_, ref.MX4)
    check(b, q, heads, type_, window=19, sinks=5)
    check(b, q, heads, type_, window=70, sinks=20)


@pytest.mark.parametrize("type_", TYPES)
def test_more_rows_than_tokens(type_):
    """Rows in front of the first token see nothing."""
    rng = np.random.default_rng(1)
    b = aref.Batch(rng, [3, 0, 20, 40], [7, 4, 21, 40], 2, 64, 16, pad=1)
    q = queries(rng, b, 4, type_)
    check(b, q, 4, type_)
    check(b, q, 4, type_, ref.MX4)
    check(b, q, 4, type_, max_length=25)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("length, window, sinks", [(5000, 0, 0), (9001, 0, 0), (9001, 3001, 17), (9001, 4, 300), (9001, 1, 0),
                                                   (9001, 8995, 4), (9001, 9001, 4), (9001, 2 ** 40, 2 ** 40)])
def test_long_sequences_in_shares(length, window, sinks, type_):
    rng = np.random.default_rng(length)
    b = aref.Batch(rng, [length, 700], [2, 1], 1, 128, 80)
    q = queries(rng, b, 6, type_)
    check(b, q, 6, type_, window=window, sinks=sinks)
    if window == 0:
        check(b, q, 6, type_, ref.MX4)


@pytest.mark.parametrize("type_", TYPES)
def test_scales(type_):
    rng = np.random.default_rng(3)
    b = aref.Batch(rng, [300, 40], [3, 1], 2, 64, 16)
    q = queries(rng, b, 4, type_)
    for scale in (0.0, -0.125, 1.0, 3.0):
        check(b, q, 4, type_, scale=scale, window=50, sinks=2)
        check(b, q, 4, type_, scale=scale)


@pytest.mark.parametrize("type_", TYPES)
def test_queries_of_all_sizes(type_):
    """Blocks whose columns lie binades apart, zeros, and the smallest numbers."""
    rng = np.random.default_rng(4)
    b = aref.Batch(rng, [120, 33], [40, 3], 1, 128, 32)
    span = 6 if type_ == ref.F16 else 25
    q = rng.normal(0, 1, (b.rows, 256)) * 2.0 ** rng.uniform(-span, 1, (b.rows, 256))
    q[0] = 0
    q[1] *= 2.0 ** -10
    q[2, :128] = 0
    q[3] = 2.0 ** -24 if type_ == ref.F16 else 2.0 ** -126
    q = ref.to_type(q, type_)
    check(b, q, 2, type_)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_nan_stays_where_it_is_seen(dim, type_):
    """One NaN block of a key or a value: rows in front of it, sequences and heads beside it, and columns of other blocks
    do not change."""
    rng = np.random.default_rng(5)
    lengths, new = [150, 150], [120, 1]
    b = aref.Batch(rng, lengths, new, 2, dim, 16)
    q = queries(rng, b, 4, type_)
    clean, _, _ = aref.attention(b, ref.to_f64(q, type_), 4, type_)
    groups = ref.groups(2 * dim)
    for rows, token, head, block in ((b.values, 61, 1, 0), (b.values, 90, 0, dim // 32 - 1), (b.keys, 100, 1, 1)):
        rows[b.places(0, 150)[token], 64 * groups + head * (dim // 32) + block] = 255
    got = check(b, q, 4, type_)
    at = ref.to_f64(got, type_).reshape(b.rows, 4, dim)
    positions = np.arange(30, 150)
    assert np.isnan(at[:120, 2:, :32][positions >= 61]).all() and not np.isnan(at[:120, 2:, :32][positions < 61]).any()
    assert np.isnan(at[:120, :2, -32:][positions >= 90]).all() and not np.isnan(at[:120, :2, :32]).any()
    assert np.isnan(at[:120, 2:][positions >= 100]).all() and not np.isnan(at[120]).any()
    check(b, q, 4, type_, ref.MX4)
    check(b, q, 4, type_, window=7, sinks=62)


def test_values_past_fp16_count_as_nan():
    rng = np.random.default_rng(6)
    b = aref.Batch(rng, [40], [1], 1, 128, 16)
    row = b.places(0, 40)[7]
    for byte, nan in ((140, False), (141, True), (254, True)):
        b.values[row, 64 + 2] = byte
        q = queries(rng, b, 2, ref.F16)
        got = run(b, q, 2, ref.F16).reshape(2, 128)
        assert np.isnan(got[:, 64:96]).all() == nan and not np.isnan(got[:, :64]).any() and not np.isnan(got[:, 96:]).any()
        if not nan:
            check(b, q, 2, ref.F16)
        got = ref.to_f64(run(b, ref.to_type(ref.to_f64(q, ref.F16), ref.BF16), 2, ref.BF16), ref.BF16)
        assert not np.isnan(got).any()


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("type_", TYPES)
def test_queries_that_are_no_numbers(type_, bad):
    rng = np.random.default_rng(7)
    b = aref.Batch(rng, [30, 20], [20, 1], 2, 64, 16)
    q = queries(rng, b, 4, type_)
    good = run(b, q, 4, type_).copy()
    x = ref.to_f64(q, type_)
    x[3, 64 + 40] = bad
    with np.errstate(invalid="ignore"):
        got = run(b, ref.to_type(x, type_), 4, type_)
    assert np.isnan(ref.to_f64(got[3], type_)[64:128]).all()
    keep = np.ones(got.shape, bool)
    keep[3, 64:128] = False
    np.testing.assert_array_equal(got[keep], good[keep])


@pytest.mark.parametrize("type_", TYPES + [ref.MX4])
@pytest.mark.parametrize("kv_heads, dim, page", [(1, 64, 16), (3, 64, 32), (2, 128, 0), (8, 128, 16), (3, 256, 48)])
def test_cache_write(kv_heads, dim, page, type_):
    rng = np.random.default_rng(kv_heads)
    lengths, new = [0, 5, 70, 33, 16, 3], [0, 5, 9, 33, 1, 5]
    b = aref.Batch(rng, lengths, new, kv_heads, dim, page or 80, bool(page), pad=4)
    cols = kv_heads * dim
    x = [ref.to_type(rng.normal(0, 2, (b.rows, cols)), type_ if type_ != ref.MX4 else ref.F32) for _ in range(2)]
    packed = [ref.rows_of(ref.to_f64(v, type_ if type_ != ref.MX4 else ref.F32)) for v in x]
    if type_ == ref.MX4:
        x = packed
    want = [b.keys.copy(), b.values.copy()]
    for i, (length, n) in enumerate(zip(lengths, new)):
        k = min(length, n)                     # (the newest: one sequence has more rows than tokens)
        for w, rows in zip(want, packed):
            w[b.places(i, length)[length - k:]] = rows[b.starts[i + 1] - k:b.starts[i + 1]]
    got = capi.mx4_cache_write(b.keys, b.values, x[0], x[1], b.starts, b.lengths, kv_heads, dim, b.page_tokens, b.pages,
                               type_)
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g, w)
