"""The cache of microscaled rows, attention and adapters as a program that serves a transformer calls them: long prompts,
many sequences, far pages, strided rows, streams, captured launches, and a layer from its norm to its last product."""
import numpy as np
import pytest

from glow_amd import capi
from tests import mx4_attention_ref as aref, mx4_ref as ref
from tests.test_gpu_mx4_adapters import Case
from tests.test_gpu_mx4_attention import check, queries, run

pytestmark = pytest.mark.gpu
TYPES = [ref.F32, ref.F16, ref.BF16]


@pytest.fixture(scope="module", autouse=True)
def _device():
    capi.init(0)


class Call:
    """A batch on the device, its attention's buffers and launch."""

    def __init__(self, b, q, heads, type_, stream=None, most=None, window=0, sinks=0, out=None):
        self.held = [capi.to_device(v) for v in (b.keys, b.values, b.starts, b.lengths)]
        self.pages = capi.to_device(b.pages) if b.pages is not None else None
        self.cache = capi.Mx4Cache(self.held[0].ptr, self.held[1].ptr, b.keys.shape[1], self.pages.ptr if self.pages else None,
                                   b.n_pages, b.page_tokens, b.per, b.kv_heads, b.head_dim)
        self.q, self.out = capi.to_device(q), capi.to_device(np.zeros_like(q) if out is None else out)
        self.most = b.per * b.page_tokens if most is None else most
        self.n = capi.mx4_attention_workspace_bytes(self.cache, heads, len(b.lengths), b.rows, self.most)
        self.ws = capi.DeviceBuffer(self.n)
        self.args, self.stream, self.size = (b, heads, type_, window, sinks), stream, q.itemsize

    def launch(self, stream=None, in_place=False):
        b, heads, type_, window, sinks = self.args
        pitch = heads * b.head_dim * self.size
        capi.launch_mx4_attention(self.q if in_place else self.out, type_, pitch, self.q, type_, pitch, heads, self.cache,
                                  self.held[2], self.held[3], len(b.lengths), b.rows, self.most, b.head_dim ** -0.5, window,
                                  sinks, self.ws, self.n, stream or self.stream)

    def check(self, got):
        b, heads, type_, window, sinks = self.args
        q = self.q_host
        want, err, used = aref.attention(b, ref.to_f64(q, type_), heads, type_, window=window, sinks=sinks)
        ref.check_float(got[used], want[used], err[used], type_)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dim, kv_heads, group", [(64, 1, 8), (128, 2, 4), (256, 1, 2)])
def test_few_rows_of_a_long_prompt_in_shares(dim, kv_heads, group, type_):
    """Enough rows for the kernel of prompts, too few workgroups: tokens in shares."""
    rng = np.random.default_rng(dim)
    b = aref.Batch(rng, [3000, 40], [70, 17], kv_heads, dim, 48)
    heads = kv_heads * group
    assert b.rows * group > 64 * 2 and Call(b, queries(rng, b, heads, type_), heads, type_).n > 0
    q = queries(rng, b, heads, type_)
    check(b, q, heads, type_)
    check(b, q, heads, type_, ref.MX4)
    check(b, q, heads, type_, window=1500, sinks=70)


@pytest.mark.parametrize("count, longest", [(63, 40), (64, 40), (65, 300), (1100, 20), (5000, 3)])
def test_many_sequences(count, longest):
    rng = np.random.default_rng(count)
    lengths = rng.integers(0, longest + 1, count)
    new = np.minimum(lengths, rng.integers(0, 3, count))
    b = aref.Batch(rng, lengths, new, 2, 128, 16, pad=5)
    q = queries(rng, b, 4, ref.BF16)
    check(b, q, 4, ref.BF16)
    x = [ref.to_type(rng.normal(0, 1, (b.rows, 256)), ref.BF16) for _ in range(2)]
    want = [b.keys.copy(), b.values.copy()]
    for w, v in zip(want, x):
        rows = ref.rows_of(ref.to_f64(v, ref.BF16))
        for i in range(count):
            w[b.places(i, lengths[i])[lengths[i] - new[i]:]] = rows[b.starts[i]:b.starts[i + 1]]
    for g, w in zip(capi.mx4_cache_write(b.keys, b.values, x[0], x[1], b.starts, b.lengths, 2, 128, 16, b.pages, ref.BF16), want):
        np.testing.assert_array_equal(g, w)


@pytest.mark.parametrize("kv_heads", [2, 3, 4, 6, 8, 12, 16])
def test_sets_of_heads(kv_heads):
    """Eight, four, two heads of 128 columns a workgroup, or one; sequences of one share and of several."""
    rng = np.random.default_rng(kv_heads)
    b = aref.Batch(rng, [2500, 1, 31, 300], [1, 1, 2, 3], kv_heads, 128, 32)
    for type_ in TYPES:
        q = queries(rng, b, kv_heads * 2, type_)
        check(b, q, kv_heads * 2, type_)
        check(b, q, kv_heads * 2, type_, ref.MX4, window=700, sinks=9)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("dim, kv_heads, new", [(64, 1, 1), (128, 2, 1), (256, 1, 2), (64, 2, 70), (128, 2, 70), (256, 1, 70)])
def test_shared_pages_and_pages_that_are_none(dim, kv_heads, new, type_):
    """Sequences with the same first pages, and sequences with holes: what is on no page is not seen."""
    rng = np.random.default_rng(15)
    b = aref.Batch(rng, [200, 150, 700], [new] * 3, kv_heads, dim, 32)
    b.pages[1, :2] = b.pages[0, :2]
    b.pages[2, [0, 5, 6, 21]] = -1, b.n_pages, 2 ** 31 - 1, -2 ** 31
    q = queries(rng, b, kv_heads * 4, type_)
    check(b, q, kv_heads * 4, type_)
    check(b, q, kv_heads * 4, type_, ref.MX4, window=90, sinks=40)
    b.pages[:] = -1
    assert not run(b, q, kv_heads * 4, type_).view(np.uint8).any()
    x = ref.to_type(rng.normal(0, 1, (b.rows, kv_heads * dim)), type_)
    for g, w in zip(capi.mx4_cache_write(b.keys, b.values, x, x, b.starts, b.lengths, kv_heads, dim, 32, b.pages, type_),
                    (b.keys, b.values)):
        np.testing.assert_array_equal(g, w)


def test_starts_and_lengths_out_of_range():
    """Entries outside of the batch, and lengths past the pages, count as the nearest."""
    rng = np.random.default_rng(8)
    b = aref.Batch(rng, [48, 20], [3, 2], 1, 64, 16, spare=0)
    q = queries(rng, b, 2, ref.F16)
    want = run(b, q, 2, ref.F16)
    b.starts[0], b.starts[2], b.lengths[0] = -7, 2 ** 31 - 1, 2 ** 31 - 1
    np.testing.assert_array_equal(run(b, q, 2, ref.F16), want)
    b.lengths[:] = -5, 0
    assert not run(b, q, 2, ref.F16).view(np.uint16).any()


@pytest.mark.parametrize("type_", TYPES)
def test_strided_rows(type_):
    """Queries, keys and values as columns of one projection's rows, and a cache of rows further apart."""
    rng = np.random.default_rng(9)
    lengths, new = [70, 5, 200], [1, 5, 2]
    b = aref.Batch(rng, lengths, new, 2, 128, 16, pad=1)
    heads, size = 6, 4 if type_ == ref.F32 else 2
    width = heads * 128 + 2 * 256 + 3
    x = ref.to_type(rng.normal(0, 1, (b.rows + 1, width)), type_)
    at = [1, 1 + heads * 128, 1 + heads * 128 + 256]
    row = b.keys.shape[1] + 48
    wide = [np.full((b.keys.shape[0], row), 0x77, np.uint8) for _ in range(2)]
    for w, rows in zip(wide, (b.keys, b.values)):
        w[:, :rows.shape[1]] = rows
    dx, dk, dv = capi.to_device(x), capi.to_device(wide[0]), capi.to_device(wide[1])
    dp, ds, dl = capi.to_device(b.pages), capi.to_device(b.starts), capi.to_device(b.lengths)
    cache = capi.Mx4Cache(dk.ptr, dv.ptr, row, dp.ptr, b.n_pages, 16, b.per, 2, 128)
    capi.launch_mx4_cache_write(cache, dx.ptr + at[1] * size, dx.ptr + at[2] * size, type_, width * size, ds, dl, 3, b.rows)
    got = [dk.numpy(), dv.numpy()]
    for g, rows, col in zip(got, (b.keys, b.values), at[1:]):
        packed = ref.rows_of(ref.to_f64(np.ascontiguousarray(x[:, col:col + 256]), type_))
        for i in range(3):
            rows[b.places(i, lengths[i])[lengths[i] - new[i]:]] = packed[b.starts[i]:b.starts[i + 1]]
        np.testing.assert_array_equal(g[:, :rows.shape[1]], rows)
        assert (g[:, rows.shape[1]:] == 0x77).all()
    out_row = (heads * 128 + 5) * size
    out = capi.to_device(np.full(b.rows * out_row + size, 0x5a, np.uint8))
    n = capi.mx4_attention_workspace_bytes(cache, heads, 3, b.rows, b.per * 16)
    ws = capi.DeviceBuffer(n)
    capi.launch_mx4_attention(out.ptr + size, type_, out_row, dx.ptr + at[0] * size, type_, width * size, heads, cache, ds, dl, 3,
                              b.rows, b.per * 16, 128 ** -0.5, 0, 0, ws, n)
    bytes_ = out.numpy()[size:].reshape(b.rows, out_row)
    q = np.ascontiguousarray(x[:b.rows, 1:1 + heads * 128])
    want, err, used = aref.attention(b, ref.to_f64(q, type_), heads, type_)
    ref.check_float(np.ascontiguousarray(bytes_[used, :heads * 128 * size]).view(q.dtype), want[used], err[used], type_)
    assert (bytes_[:, heads * 128 * size:] == 0x5a).all() and (bytes_[~used] == 0x5a).all()


def test_pages_past_4_gib():
    """A sequence's tokens in the last pages of 6 GiB of keys and as many of values, by a table and in a row."""
    rng = np.random.default_rng(10)
    kv_heads, dim, page = 8, 128, 64
    row = capi.mx4_row_bytes(kv_heads * dim)
    n_pages = (6 << 30) // (page * row)
    lengths = [100, 700]
    b = aref.Batch(rng, lengths, [1, 1], kv_heads, dim, page, False, spare=0)
    q = queries(rng, b, 16, ref.BF16)
    want = run(b, q, 16, ref.BF16)
    held = [capi.DeviceBuffer(n_pages * page * row) for _ in range(2)]
    per = b.per
    first = n_pages - 2 * per
    for buffer, rows in zip(held, (b.keys, b.values)):
        part = capi.to_device(rows)
        capi.check(capi.lib().mi355x_memcpy_d2d(capi._vp(buffer.ptr + first * page * row), capi._vp(part), capi._sz(rows.nbytes),
                                                capi._vp(None)))
    table = capi.to_device((first + np.arange(2 * per, dtype=np.int32)).reshape(2, per))
    dq, out = capi.to_device(q), capi.to_device(np.zeros_like(q))
    ds, dl = capi.to_device(b.starts), capi.to_device(b.lengths)
    cache = capi.Mx4Cache(held[0].ptr, held[1].ptr, row, table.ptr, n_pages, page, per, kv_heads, dim)
    n = capi.mx4_attention_workspace_bytes(cache, 16, 2, 2, per * page)
    ws = capi.DeviceBuffer(n)
    capi.launch_mx4_attention(out, ref.BF16, 4096, dq, ref.BF16, 4096, 16, cache, ds, dl, 2, 2, per * page, dim ** -0.5, 0, 0, ws, n)
    np.testing.assert_array_equal(out.numpy(), want)
    # the newest token of each again, through the writer
    x = ref.to_type(rng.normal(0, 1, (2, 2048)), ref.BF16)
    dx = capi.to_device(x)
    capi.launch_mx4_cache_write(cache, dx, dx.ptr + 2048, ref.BF16, 4096, ds, dl, 2, 2)
    for k, (buffer, rows) in enumerate(zip(held, (b.keys, b.values))):
        packed = ref.rows_of(ref.to_f64(np.ascontiguousarray(x[:, k * 1024:(k + 1) * 1024]), ref.BF16))
        for i in range(2):
            rows[b.places(i, lengths[i])[-1]] = packed[i]
        got = np.empty_like(rows)
        capi.check(capi.lib().mi355x_memcpy_d2h(capi._vp(got), capi._vp(buffer.ptr + first * page * row), capi._sz(got.nbytes), None))
        capi.sync()
        np.testing.assert_array_equal(got, rows)


@pytest.mark.parametrize("lengths, new", [([400, 3, 60], [1, 1, 2]), ([9000], [1]), ([300, 80], [200, 80])])
def test_in_place_at_once_and_again(lengths, new):
    """The result in the queries' place; two calls at once on streams of their own; equal calls with other bits in
    every buffer that they write."""
    rng = np.random.default_rng(11)
    b = aref.Batch(rng, lengths, new, 8, 128, 16)
    q = queries(rng, b, 16, ref.F16)
    first = run(b, q, 16, ref.F16)
    streams = [capi.Stream(), capi.Stream()]
    calls = [Call(b, q, 16, ref.F16, s) for s in streams]
    for i in range(5):
        for c in calls:
            c.out.fill(i * 37, c.stream)
            if c.n:
                c.ws.fill(255 - i, c.stream)
            c.launch()
        for c in calls:
            np.testing.assert_array_equal(c.out.numpy(c.stream).view(np.uint16), first.view(np.uint16))
    calls[0].launch(in_place=True)
    np.testing.assert_array_equal(calls[0].q.numpy(streams[0]).view(np.uint16), first.view(np.uint16))


def test_captured_steps_of_a_growing_sequence():
    """One captured write and attention, replayed token by token: starts, lengths and rows change, the graph does not."""
    rng = np.random.default_rng(12)
    kv_heads, dim, heads, page, steps = 2, 128, 8, 16, 6
    final = aref.Batch(rng, [40 + steps, 500 + steps, steps], [1, 1, 1], kv_heads, dim, page)
    x = ref.to_type(rng.normal(0, 1, (steps, 3, (heads + 2 * kv_heads) * dim)), ref.BF16)
    lengths = final.lengths - steps
    stream = capi.Stream()
    call = Call(final, np.zeros((3, heads * dim), np.uint16), heads, ref.BF16, stream)
    row = x.shape[2] * 2
    dx = capi.to_device(x[0])
    def go():
        capi.launch_mx4_cache_write(call.cache, dx.ptr + heads * dim * 2, dx.ptr + (heads + kv_heads) * dim * 2, ref.BF16, row,
                                    call.held[2], call.held[3], 3, 3, stream)
        capi.launch_mx4_attention(call.out, ref.BF16, heads * dim * 2, dx, ref.BF16, row, heads, call.cache, call.held[2],
                                  call.held[3], 3, 3, call.most, dim ** -0.5, 0, 0, call.ws, call.n, stream)
    assert call.n > 0
    go()                                   # (the first launch sets what capture may not)
    stream.sync()
    with capi.Graph(stream) as graph:
        go()
    keys, values = final.keys.copy(), final.values.copy()
    call.held[0].upload(keys, stream)
    call.held[1].upload(values, stream)
    for i in range(steps):
        final.lengths = (lengths + i + 1).astype(np.int32)
        dx.upload(x[i], stream)
        call.held[3].upload(final.lengths, stream)
        graph.launch()
        got = call.out.numpy(stream)
        for rows, at in ((final.keys, heads), (final.values, heads + kv_heads)):
            packed = ref.rows_of(ref.to_f64(np.ascontiguousarray(x[i][:, at * dim:(at + kv_heads) * dim]), ref.BF16))
            for s in range(3):
                rows[final.places(s, final.lengths[s])[-1]] = packed[s]
        q = np.ascontiguousarray(x[i][:, :heads * dim])
        want, err, _ = aref.attention(final, ref.to_f64(q, ref.BF16), heads, ref.BF16)
        ref.check_float(got, want, err, ref.BF16)
        np.testing.assert_array_equal(run(final, q, heads, ref.BF16), got)
    np.testing.assert_array_equal(call.held[0].numpy(stream), final.keys)


def test_adapters_at_once_captured_and_again():
    rng = np.random.default_rng(13)
    cases = [Case(rng, 40, 1024, 600, 16, 5, ref.BF16, ref.BF16), Case(rng, 700, 700, 300, 40, 3, ref.F32, ref.F16, runs=100)]
    want = [c.run(ref.F32) for c in cases]
    jobs = []
    for c in cases:
        M = c.x.shape[0]
        held = [capi.to_device(v) for v in (c.x, c.w, c.b, c.down, c.up, c.scales, c.ids)]
        n = capi.mx4_fc_adapters_workspace_bytes(M, c.K, c.N, c.in_type, c.down.shape[1])
        jobs.append((c, M, held, capi.DeviceBuffer(n), n, capi.DeviceBuffer.empty((M, c.N), np.float32), capi.Stream()))

    def go(job):
        c, M, (x, w, b, down, up, scales, ids), ws, n, out, stream = job
        a = capi.Mx4Adapters(down.ptr, up.ptr, scales.ptr, c.count, c.down.shape[1], c.type_)
        capi.launch_mx4_fc_adapters(out, ref.F32, 4 * c.N, x, c.in_type, c.x.shape[1] * c.x.itemsize, w, c.w.shape[1], b, a, ids, M,
                                    c.K, c.N, 0, ws, n, stream)
    for i in range(4):
        for job in jobs:
            job[3].fill(i * 77 % 256, job[6])
            job[5].fill(i * 50, job[6])
            go(job)
        for job, w in zip(jobs, want):
            np.testing.assert_array_equal(job[5].numpy(job[6]), w)
    for job, w in zip(jobs, want):
        with capi.Graph(job[6]) as graph:
            go(job)
        for i in range(3):
            job[5].fill(i, job[6])
            job[3].fill(255 - i, job[6])
            graph.launch()
            np.testing.assert_array_equal(job[5].numpy(job[6]), w)


@pytest.mark.parametrize("lengths, new", [([30, 1, 300, 17], [1, 1, 1, 1]), ([90, 40], [90, 7])])
def test_a_layer(lengths, new):
    """Norm, projection with adapters, cache, attention, projection with adapters: microscaled rows from one to the next, each
    checked in 64 bits from what it was handed."""
    rng = np.random.default_rng(14)
    heads, kv_heads, dim, width, type_ = 4, 2, 64, 320, ref.BF16
    b = aref.Batch(rng, lengths, new, kv_heads, dim, 16)
    M, cols = b.rows, kv_heads * dim
    x = ref.to_type(rng.normal(0, 2, (M, 1, width)), type_)
    gamma = (1 + 0.1 * rng.normal(0, 1, width)).astype(np.float32)
    h = capi.group_norm(x, 1, gamma, None, type_=type_, out_type=ref.MX4).reshape(M, -1)
    want, err = ref.group_norm(ref.to_f64(x, type_), 1, gamma, None, 1e-5, 0)
    ref.check_mx4(h, width, want.reshape(M, -1), err.reshape(M, -1))

    def project(rows, K, N, out_type):
        c = Case(rng, M, K, N, 8, 3, ref.MX4, type_, bias=False, runs=3)
        c.x, c.shared = rows, ref.values(rows, K)
        c.own = c.shared
        return c.check(out_type)
    q = project(h, width, heads * dim, type_)
    k, v = (project(h, width, cols, ref.MX4) for _ in range(2))
    b.keys, b.values = capi.mx4_cache_write(b.keys, b.values, k, v, b.starts, b.lengths, kv_heads, dim, 16, b.pages, ref.MX4)
    for i in range(len(lengths)):
        np.testing.assert_array_equal(b.keys[b.places(i, lengths[i])[lengths[i] - new[i]:]], k[b.starts[i]:b.starts[i + 1]])
    o = check(b, q, heads, type_, ref.MX4, window=100, sinks=2)
    project(o, heads * dim, width, type_)
