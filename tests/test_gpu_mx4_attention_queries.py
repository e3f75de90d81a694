"""Attention over a cache of microscaled rows with queries of which one column of each block of 32 stands out: how many bits of
the others take part in a score."""
import numpy as np
import pytest

from glow_amd import capi
from tests import mx4_attention_ref as aref, mx4_ref as ref
from tests.test_gpu_mx4_attention import run

pytestmark = pytest.mark.gpu
TYPES = [ref.F32, ref.F16, ref.BF16]
# heads one by one, heads in sets, prompts, shares
SHAPES = [(64, 2, 4, 1, 300), (128, 1, 4, 1, 300), (128, 2, 4, 3, 300), (128, 8, 2, 1, 300), (256, 1, 4, 1, 300),
          (64, 2, 4, 70, 200), (128, 2, 4, 70, 200), (256, 1, 4, 70, 200), (128, 2, 4, 1, 5000)]


@pytest.fixture(scope="module", autouse=True)
def _device():
    capi.init(0)


def attention(b, q, heads, type_, scale):
    """(results, bound of the error before the result's own rounding) of a batch of one sequence, 64 bits.

    A query is a sum of three terms, each of which leaves a thirty-second of what it takes, and one that leaves an eighth: 2^-17 of
    its block's largest; of six of the former in fp32, 2^-29. Sums of D products a term, of the terms and of weights are of
    32 bits in any order; a weight's exponent is rounded at the size of its score and of the largest, 2^x is within 2^-22, and a
    weight is rounded to the type (24 bits in fp32)."""
    d, group, length, n = b.head_dim, heads // b.kv_heads, int(b.lengths[0]), b.rows
    cut = 2.0 ** (-29 if type_ == ref.F32 else -17)
    at = b.places(0, length)
    K, V = (ref.values(t[at], b.kv_heads * d).reshape(length, b.kv_heads, d) for t in (b.keys, b.values))
    out, err = np.zeros((n, heads, d)), np.zeros((n, heads, d))
    q = q.reshape(n, heads, d)
    for r in range(n):
        k, v = K[:length - n + r + 1], V[:length - n + r + 1]
        for h in range(heads):
            x, kh, vh = q[r, h], k[:, h // group], v[:, h // group]
            s = kh @ x * scale
            p = np.exp(s - s.max())
            out[r, h] = p @ vh / p.sum()
            most = np.repeat(np.abs(x).reshape(-1, 32).max(-1), 32)
            ds = scale * (np.abs(kh) @ (most * cut) + (d + 10) * 2.0 ** -23 * (np.abs(kh) @ np.abs(x)))
            ds += 2.0 ** -22 * (np.abs(s) + np.abs(s).max() + 1)
            rel, steps = np.expm1(ds), (len(s) + 40) * 2.0 ** -23
            top = (p * (rel + ref.HALF_STEP[type_] * (1 + rel) + steps)) @ np.abs(vh) + 2.0 ** -32 * np.abs(vh).sum(0)
            err[r, h] = (top / p.sum() + np.abs(out[r, h]) * ((p @ rel) / p.sum() + steps)) * 1.01
    return out.reshape(n, -1), err.reshape(n, -1)


def check(b, q, heads, type_, scale):
    want, err = attention(b, ref.to_f64(q, type_), heads, type_, scale)
    ref.check_float(run(b, q, heads, type_, scale=scale), want, err, type_)
    ref.check_mx4(run(b, q, heads, type_, ref.MX4, scale=scale), heads * b.head_dim, want, err)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("loud", [1, 16, 64, 1024])
@pytest.mark.parametrize("dim, kv_heads, group, new, length", SHAPES)
def test_loud_columns(dim, kv_heads, group, new, length, loud, type_):
    rng = np.random.default_rng(dim + loud)
    b = aref.Batch(rng, [length], [new], kv_heads, dim, 32)
    q = rng.normal(0, 1.5, (b.rows, kv_heads * group * dim))
    q[:, 7::32] *= loud
    q = ref.to_type(q, type_)
    check(b, q, kv_heads * group, type_, dim ** -0.5 * 4 / (3 + loud))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("below", [10, 12, 13, 15])
@pytest.mark.parametrize("dim, kv_heads, group, new, length", SHAPES)
def test_what_small_columns_add_up_to(dim, kv_heads, group, new, length, below, type_):
    """Columns 2^below smaller than their block's largest, each just under a power of two and all of the sign of the
    key's: cut off, they would be missing from a score together, and the signs of values are those of the scores."""
    rng = np.random.default_rng(dim + below)
    b = aref.Batch(rng, [length], [new], kv_heads, dim, 32)
    heads, cols = kv_heads * group, kv_heads * dim
    sign = rng.choice([-1.0, 1.0], cols)
    size = rng.choice([-4, -3, -1.5, 1.5, 3, 4], (length, 1))
    keys = sign * size
    keys[:, 7::32] = 0
    at = b.places(0, length)
    b.keys[at] = ref.rows_of(keys)
    b.values[at] = ref.rows_of(np.sign(size) * rng.choice([0.5, 1, 1.5], (length, cols)))
    q = np.repeat(sign.reshape(1, kv_heads, 1, dim) * 0.97 * 2.0 ** -below, group, 2).reshape(1, -1).repeat(b.rows, 0)
    q *= rng.choice([1.0, 1.01, 0.98], (b.rows, 1))
    q[:, 7::32] = rng.choice([1.0, -1.03, 1.5, -1.97], q[:, 7::32].shape)
    q = ref.to_type(q * 16, type_)
    check(b, q, heads, type_, 2.0 ** below / dim / 64)
