"""A cache of microscaled rows and attention over it from their definitions, in numpy and 64 bits."""
import numpy as np

from tests import mx4_ref as ref


class Batch:
    """Sequences of `lengths` tokens of which the last `new` are rows of a batch, and a cache for them. Rows of the
    cache that hold no token, and pages that belong to nobody, are NaN."""

    def __init__(self, rng, lengths, new, kv_heads, head_dim, page_tokens, paged=True, pad=0, spare=1):
        self.lengths, self.new = np.array(lengths, np.int32), np.array(new, np.int32)
        self.kv_heads, self.head_dim, self.page_tokens = kv_heads, head_dim, page_tokens
        n, cols = len(lengths), kv_heads * head_dim
        per = max(1, -(-int(max(lengths, default=1)) // page_tokens)) + spare
        self.starts = np.concatenate(([0], np.cumsum(self.new))).astype(np.int32)
        self.rows = int(self.starts[-1]) + pad
        if paged:
            used = [-(-int(t) // page_tokens) for t in lengths]
            self.n_pages = sum(used) + 2
            order = rng.permutation(self.n_pages)
            self.pages, done = np.full((n, per), -1, np.int32), 0
            for i, k in enumerate(used):
                self.pages[i, :k] = order[done:done + k]
                self.pages[i, k:] = rng.choice([-1, self.n_pages, 2 ** 31 - 1, -2 ** 31, order[-1]])
                done += k
        else:
            self.pages, self.n_pages = None, n * per
        self.per = per
        total = self.n_pages * page_tokens
        loud = np.exp(0.5 * rng.normal(0, 1, cols))
        self.keys = ref.rows_of(rng.normal(0, 1, (total, cols)) * loud)
        self.values = ref.rows_of(rng.normal(0, 1, (total, cols)) * 10.0 ** rng.uniform(-1, 1, (total, 1)))
        there = np.zeros(total, bool)
        for i in range(n):
            there[self.places(i, int(lengths[i]))] = True
        for rows in (self.keys, self.values):
            rows[~there] = 0xff

    def places(self, i, count):
        t = np.arange(count)
        page = self.pages[i, t // self.page_tokens] if self.pages is not None else i * self.per + t // self.page_tokens
        return page.astype(np.int64) * self.page_tokens + t % self.page_tokens


def sees(position, tokens, window, sinks):
    t = np.arange(tokens)
    seen = t <= position
    if window:
        seen &= (t > position - window) | (t < sinks)
    return seen


def attention(b, q, heads, type_, scale=None, window=0, sinks=0, max_length=None):
    """(results [rows, heads * dim], bound of the error before the result's own rounding, rows that belong to a
    sequence) for q in 64 bits.

    A query is a sum of 3 (16-bit types) or 6 (fp32) terms of four bits, each of which leaves a sixteenth of the block's
    largest at most. Scores are D products a term in any order and the sums of the terms, in 32 bits; a weight's exponent is
    rounded at the size of its score and of the largest, twice, and 2^x within 2^-22. Weights are rounded to the type, in fp16
    shifted so that the smallest step is 2^-32 of the largest weight; in fp32 to 24 bits."""
    d, group = b.head_dim, heads // b.kv_heads
    scale = d ** -0.5 if scale is None else scale
    half = {ref.F32: 2.0 ** -24, ref.F16: 2.0 ** -11, ref.BF16: 2.0 ** -8}[type_]
    cut = 2.0 ** -24 if type_ == ref.F32 else 2.0 ** -12
    out, err = np.zeros((b.rows, heads, d)), np.zeros((b.rows, heads, d))
    used = np.zeros(b.rows, bool)
    q = q.reshape(b.rows, heads, d)
    for i in range(len(b.lengths)):
        length = int(b.lengths[i]) if max_length is None else min(int(b.lengths[i]), max_length)
        n, begin = int(b.starts[i + 1] - b.starts[i]), int(b.starts[i])
        used[begin:begin + n] = True
        if not length or not n:
            continue
        # tokens on no page are not seen
        at = b.places(i, length)
        there = np.ones(length, bool)
        if b.pages is not None:
            page = b.pages[i, np.arange(length) // b.page_tokens]
            there = (page >= 0) & (page < b.n_pages)
        at = np.where(there, at, 0)
        K = ref.values(b.keys[at], b.kv_heads * d).reshape(length, b.kv_heads, d)
        V = ref.values(b.values[at], b.kv_heads * d).reshape(length, b.kv_heads, d)
        for r in range(n):
            seen = sees(length - n + r, length, window, sinks) & there
            if not seen.any():
                continue
            for h in range(heads):
                x, k, v = q[begin + r, h], K[seen, h // group], V[seen, h // group]
                with np.errstate(invalid="ignore"):
                    s = (k @ x) * scale
                    p = np.exp(s - s.max())
                    out[begin + r, h] = p @ v / p.sum()
                    if not np.isfinite(s).all():
                        out[begin + r, h] = np.nan
                if not np.isfinite(out[begin + r, h]).any():
                    continue
                most = np.repeat(np.abs(x).reshape(-1, 32).max(-1), 32)
                ds = abs(scale) * (np.abs(k) @ (most * cut) + (d + 10) * 2.0 ** -23 * (np.abs(k) @ np.abs(x)))
                ds += 2.0 ** -22 * (np.abs(s) + np.abs(s).max() + 1)
                rel = np.expm1(ds)
                count, av = seen.sum(), np.abs(v)
                steps = (count + 40) * 2.0 ** -23
                top = (p * (rel + half * (1 + rel) + steps)) @ av + 2.0 ** -32 * av.sum(0)
                below = (p @ rel) / p.sum() + steps
                err[begin + r, h] = (top + np.abs(out[begin + r, h]) * p.sum() * below) / p.sum() * 1.01
    return out.reshape(b.rows, -1), err.reshape(b.rows, -1), used
