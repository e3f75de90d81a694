"""Attention over a cache of microscaled rows whose memory holds anything where no token is seen: no bit of a result comes
from there. Scale bytes of which some codes are past the range of a type (253 and 254 of 32 bits and bfloat16, 141 on of
fp16) count as what they stand for where they are seen, fp16's as NaN."""
import numpy as np
import pytest

from glow_amd import capi
from tests import mx4_attention_ref as aref, mx4_ref as ref
from tests.test_gpu_mx4_attention import check, queries, run

pytestmark = pytest.mark.gpu
TYPES = [ref.F32, ref.F16, ref.BF16]
BYTES = [0, 1, 140, 141, 252, 253, 254, 255]
# heads one by one, heads in sets, prompts; the last two with shares of a long sequence
SHAPES = [(64, 2, 4, 1, 700), (128, 1, 2, 1, 700), (128, 2, 2, 3, 700), (128, 8, 1, 1, 700), (256, 1, 2, 2, 700),
          (64, 2, 4, 70, 300), (128, 2, 4, 70, 300), (256, 1, 4, 70, 300), (128, 1, 4, 1, 6001), (128, 2, 4, 2, 6001)]


@pytest.fixture(scope="module", autouse=True)
def _device():
    capi.init(0)


def anything(rng, count, cols):
    """Rows of any bytes, their scales of those that matter."""
    rows = rng.integers(0, 256, (count, ref.row_bytes(cols))).astype(np.uint8)
    groups = ref.groups(cols)
    rows[:, 64 * groups:68 * groups] = rng.choice(BYTES, (count, 4 * groups))
    return rows


def batch(rng, dim, kv_heads, new, longest):
    """Three sequences, one with a page that is none; the cache's first page belongs to nobody."""
    b = aref.Batch(rng, [longest, 5, 161], [new, min(5, new), new], kv_heads, dim, 32)
    b.pages = np.where((b.pages >= 0) & (b.pages <= b.n_pages), b.pages + 1, b.pages).astype(np.int32)
    b.n_pages += 1
    b.keys, b.values = (np.concatenate((np.zeros_like(v[:32]), v)) for v in (b.keys, b.values))
    b.pages[0, 2] = -1
    held = np.zeros(b.keys.shape[0], bool)
    for i, length in enumerate(b.lengths):
        t = np.arange(length)
        held[b.places(i, int(length))[b.pages[i, t // 32] >= 0]] = True
    return b, ~held


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dim, kv_heads, group, new, longest", SHAPES)
def test_memory_of_no_token(dim, kv_heads, group, new, longest, type_):
    """The rest of a sequence's last page, pages of nobody, the cache's first rows beside pages that are none."""
    rng = np.random.default_rng(dim + kv_heads + new)
    b, free = batch(rng, dim, kv_heads, new, longest)
    heads, cols = kv_heads * group, kv_heads * dim
    q = queries(rng, b, heads, type_)
    for kw in (dict(), dict(window=45, sinks=3)):
        b.keys[free] = b.values[free] = 0
        clean = [run(b, q, heads, type_, t, **kw) for t in (None, ref.MX4)]
        for k in range(3):
            b.keys[free], b.values[free] = anything(rng, free.sum(), cols), anything(rng, free.sum(), cols)
            for t, want in zip((None, ref.MX4), clean):
                np.testing.assert_array_equal(run(b, q, heads, type_, t, **kw).view(np.uint8), want.view(np.uint8))
        check(b, q, heads, type_, **kw)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dim, kv_heads, group, new, longest", [s for s in SHAPES if s[3] > 1])
def test_tokens_behind_a_row(dim, kv_heads, group, new, longest, type_):
    rng = np.random.default_rng(dim + new)
    b, _ = batch(rng, dim, kv_heads, new, longest)
    heads = kv_heads * group
    q = queries(rng, b, heads, type_)
    clean = run(b, q, heads, type_)
    hidden = new // 2                                # the newest tokens of the first sequence
    at = b.places(0, longest)[longest - hidden:]
    for byte in (141, 253, 254, 255):
        for rows in (b.keys, b.values):
            rows[at] = anything(rng, hidden, kv_heads * dim)
            rows[at, 64 * ref.groups(kv_heads * dim):68 * ref.groups(kv_heads * dim)] = byte
        got = run(b, q, heads, type_)
        for rows in (slice(0, new - hidden), slice(new, None)):
            np.testing.assert_array_equal(got[rows].view(np.uint8), clean[rows].view(np.uint8))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dim, kv_heads, group, new, longest", SHAPES)
def test_tokens_outside_of_a_window(dim, kv_heads, group, new, longest, type_):
    rng = np.random.default_rng(dim + new)
    b, _ = batch(rng, dim, kv_heads, new, longest)
    heads, window, sinks = kv_heads * group, 61, 5
    q = queries(rng, b, heads, type_)
    clean = run(b, q, heads, type_, window=window, sinks=sinks)
    for i, length in enumerate(b.lengths):
        first = max(sinks, int(length - b.new[i]) - window + 1)       # tokens that no row of the sequence sees
        there = b.pages[i, np.arange(sinks, first) // 32] >= 0
        at = b.places(i, first)[sinks:][there]
        b.keys[at], b.values[at] = (anything(rng, at.size, kv_heads * dim) for _ in range(2))
    np.testing.assert_array_equal(run(b, q, heads, type_, window=window, sinks=sinks).view(np.uint8), clean.view(np.uint8))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("byte", [141, 252, 253, 254])
@pytest.mark.parametrize("dim, kv_heads, group, new", [(64, 2, 4, 3), (128, 1, 2, 3), (128, 2, 2, 3), (256, 1, 2, 3),
                                                       (64, 2, 4, 70), (128, 2, 4, 70), (256, 1, 4, 70)])
def test_large_values_that_are_seen(dim, kv_heads, group, new, byte, type_):
    """One block whose codes are past a type's range: its mean with the others' is within that of 32 bits."""
    rng = np.random.default_rng(byte + dim)
    b = aref.Batch(rng, [200], [new], kv_heads, dim, 32)
    heads = kv_heads * group
    at = b.places(0, 200)[198]
    b.values[at] = rng.integers(0, 256, b.values.shape[1]).astype(np.uint8)
    groups = ref.groups(kv_heads * dim)
    b.values[at, 64 * groups:] = 0
    b.values[at, 64 * groups:64 * groups + kv_heads * dim // 32] = 127
    b.values[at, 64 * groups + 1] = byte
    q = queries(rng, b, heads, type_)
    if type_ != ref.F16:
        check(b, q, heads, type_, scale=0.001)
        check(b, q, heads, type_, ref.MX4, scale=0.001)
        return
    got = run(b, q, heads, type_, scale=0.001).reshape(new, heads, dim)
    sees = np.arange(200 - new, 200) >= 198
    assert np.isnan(got[sees, :group, 32:64]).all()
    got[sees, :group, 32:64] = 0
    assert not np.isnan(got).any()


@pytest.mark.parametrize("type_", [ref.F32, ref.BF16])
@pytest.mark.parametrize("size", [250, 252, 70])
@pytest.mark.parametrize("dim, kv_heads, group, new, longest", SHAPES)
def test_values_at_the_ends_of_the_range(dim, kv_heads, group, new, longest, size, type_):
    """Sums over many tokens of values up to 2^127, whose mean is within the range, and of values down to 2^-60. Scores rise
    from token to token, so that weights are as large as they get before the running maximum moves."""
    rng = np.random.default_rng(size + dim)
    b = aref.Batch(rng, [longest], [new], kv_heads, dim, 32)
    heads, cols = kv_heads * group, kv_heads * dim
    groups = ref.groups(cols)
    at = b.places(0, longest)
    b.values[np.ix_(at, 64 * groups + np.arange(cols // 32))] = size
    b.values[at, :64 * groups] |= 0x44                   # (magnitudes 2 to 6: sums without much cancelling)
    b.values[at, :64 * groups] &= 0x77
    rising = rng.normal(0, 0.2, (longest, cols))
    rising[:, ::32] = np.linspace(-4, 4, longest)[:, None]
    b.keys[at] = ref.rows_of(rising)
    q = rng.normal(0, 0.3, (b.rows, heads * dim))
    q[:, ::32] = 1.5
    q = ref.to_type(q, type_)
    scale = 8 / dim
    check(b, q, heads, type_, scale=scale)
    check(b, q, heads, type_, ref.MX4, scale=scale, window=90, sinks=7)


@pytest.mark.parametrize("sizes", [(75, 78), (85, 110), (120, 150), (140, 142), (240, 252)])
@pytest.mark.parametrize("dim, kv_heads, group, new, longest", SHAPES)
def test_values_that_fp16_does_not_hold_in_a_microscaled_result(dim, kv_heads, group, new, longest, sizes):
    """Blocks with scales from 2^-52 to 2^125 under fp16 queries: a microscaled result is quantised from what they stand for."""
    rng = np.random.default_rng(sizes[0] + dim)
    b = aref.Batch(rng, [longest, 40], [new, min(new, 40)], kv_heads, dim, 32)
    heads, cols = kv_heads * group, kv_heads * dim
    groups = ref.groups(cols)
    for i, length in enumerate(b.lengths):
        at = b.places(i, int(length))
        b.values[np.ix_(at, 64 * groups + np.arange(cols // 32))] = rng.integers(*sizes, (at.size, cols // 32))
    q = queries(rng, b, heads, ref.F16)
    check(b, q, heads, ref.F16, ref.MX4)
    check(b, q, heads, ref.F16, ref.MX4, window=50, sinks=4)


@pytest.mark.parametrize("dim, kv_heads, group, new, longest", SHAPES)
def test_small_values_under_fp16(dim, kv_heads, group, new, longest):
    """An fp16 result of values with scales from 2^-40 on: each is rounded to a multiple of 2^-24, by half of one at most."""
    rng = np.random.default_rng(dim)
    b = aref.Batch(rng, [longest], [new], kv_heads, dim, 32)
    heads, cols = kv_heads * group, kv_heads * dim
    groups, at = ref.groups(cols), b.places(0, longest)
    b.values[np.ix_(at, 64 * groups + np.arange(cols // 32))] = rng.integers(87, 112, (at.size, cols // 32))
    q = queries(rng, b, heads, ref.F16)
    want, err, used = aref.attention(b, ref.to_f64(q, ref.F16), heads, ref.F16)
    ref.check_float(run(b, q, heads, ref.F16)[used], want[used], err[used] + 2.0 ** -25, ref.F16)


def test_a_vector_is_no_cache():
    rows, one = np.zeros(160, np.uint8), np.zeros((1, 128), np.float32)
    with pytest.raises(capi.MI355XError, match="keys of shape"):
        capi.mx4_attention(one, 1, rows, rows, [0, 1], [1], 1, 128, 16, [[0]])
    with pytest.raises(capi.MI355XError, match="keys of shape"):
        capi.mx4_cache_write(rows, rows, one, one, [0, 1], [1], 1, 128, 16, [[0]])
