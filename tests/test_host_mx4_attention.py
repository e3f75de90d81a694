"""A cache of microscaled rows, attention over it and adapters beside a product, as far as no GPU is involved: workspaces, and
what the calls refuse."""
import ctypes as C

import numpy as np
import pytest

from glow_amd import capi
from tests import mx4_attention_ref as aref, mx4_ref as ref
from tests.test_host_mx4 import refused, sz, vp

P = 1 << 40          # addresses that no refused call touches, 2^36 apart
KEYS, VALUES, PAGES, STARTS, LENGTHS, Q, OUT, WS, X, W = (P + (i << 36) for i in range(10))


def cache(**change):
    a = dict(keys=KEYS, values=VALUES, row_bytes=272, pages=PAGES, n_pages=10, page_tokens=16, pages_per_sequence=5,
             kv_heads=4, head_dim=128)
    a.update(change)
    return capi.Mx4Cache(**a)


CACHE_REFUSALS = [
    (dict(page_tokens=0), "multiple of 16", -1),
    (dict(page_tokens=24), "multiple of 16", -1),
    (dict(head_dim=96), "64, 128 and 256", -1),
    (dict(head_dim=0), "64, 128 and 256", -1),
    (dict(kv_heads=0), "0 heads", -1),
    (dict(kv_heads=1 << 25), "heads", -1),
    (dict(pages_per_sequence=1 << 28), "2^31 - 1 tokens", -1),
    (dict(row_bytes=256), "take 272", -1),
    (dict(row_bytes=280), "multiples of 16", -1),
    (dict(row_bytes=(1 << 26) + 16), "2^26", -1),
    (dict(keys=KEYS + 8), "multiples of 16", -1),
    (dict(values=VALUES + 4), "multiples of 16", -1),
    (dict(pages=PAGES + 2), "multiple of 4", -1),
    (dict(keys=0), "NULL", -1),
    (dict(values=0), "NULL", -1),
    (dict(n_pages=1 << 31, page_tokens=32, pages_per_sequence=1), "2^35", -4),
]


def write_args(c=None, keys=Q, values=X, type_=1, row=1024, vrow=1024, starts=STARTS, lengths=LENGTHS, sequences=3, rows=7):
    return (C.byref(c or cache()), *vp(keys, values), type_, *sz(row, vrow), *vp(starts, lengths), *sz(sequences, rows), None)


def attention_args(c=None, out=OUT, out_type=1, out_row=2048, q=Q, type_=1, q_row=2048, heads=8, starts=STARTS, lengths=LENGTHS,
                   sequences=3, rows=7, most=80, scale=0.1, window=0, sinks=0, ws=WS, ws_bytes=1 << 30):
    return (*vp(out), out_type, *sz(out_row), *vp(q), type_, *sz(q_row, heads), C.byref(c or cache()), *vp(starts, lengths),
            *sz(sequences, rows, most), C.c_float(scale), *sz(window, sinks), *vp(ws), *sz(ws_bytes), None)


@pytest.mark.parametrize("change, word, code", CACHE_REFUSALS)
def test_caches_that_are_refused(change, word, code):
    c = cache(**change)
    refused("mi355x_mx4_cache_write", write_args(c), word, code)
    refused("mi355x_mx4_attention", attention_args(c), word, code)
    n = C.c_size_t(0)
    refused("mi355x_mx4_attention_workspace_bytes", (C.byref(c), *sz(8, 3, 7, 80), C.byref(n)), word, code)


@pytest.mark.parametrize("change, word", [
    (dict(type_=4), "unknown element type"),
    (dict(row=1022), "take 1024"),
    (dict(vrow=1000), "take 1024"),
    (dict(row=1025), "multiples of 2"),
    (dict(keys=Q + 1), "multiples of 2"),
    (dict(type_=3, row=264), "take 272"),
    (dict(type_=3, row=280, vrow=280), "multiples of 16"),
    (dict(keys=0), "NULL"),
    (dict(values=0), "NULL"),
    (dict(starts=0), "NULL"),
    (dict(lengths=0), "NULL"),
    (dict(starts=STARTS + 2), "multiples of 4"),
    (dict(rows=1 << 30), "2^30"),
    (dict(sequences=1 << 30), "2^30"),
    (dict(keys=KEYS + 16), "overlaps"),
    (dict(values=KEYS - 2048), "overlaps"),
    (dict(lengths=VALUES + 64), "overlaps"),
    (dict(c=cache(values=KEYS + 16 * 10 * 272 - 272)), "overlap"),
    (dict(c=cache(pages=KEYS + 100)), "overlaps"),
])
def test_cache_write_refuses(change, word):
    refused("mi355x_mx4_cache_write", write_args(**change), word)


def test_no_cache_is_refused():
    refused("mi355x_mx4_cache_write", (None, *write_args()[1:]), "no cache")
    args = attention_args()
    refused("mi355x_mx4_attention", (*args[:7], None, *args[8:]), "no cache")


@pytest.mark.parametrize("change, word", [
    (dict(type_=3), "none of the float types"),
    (dict(out_type=2), "the queries'"),
    (dict(out_type=0), "the queries'"),
    (dict(heads=0), "over the cache's 4"),
    (dict(heads=6), "over the cache's 4"),
    (dict(heads=1 << 30), "over the cache's 4"),
    (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"),
    (dict(q_row=2046), "take 2048"),
    (dict(out_row=2047), "take 2048"),
    (dict(out_row=2049), "multiples of 2"),
    (dict(q=0), "NULL"),
    (dict(out=0), "NULL"),
    (dict(out_type=3, out_row=540), "take 544"),
    (dict(out=OUT + 1), "multiples of 2"),
    (dict(out=Q + 2048), "without being their place"),
    (dict(out=Q, out_row=4096), "without being their place"),
    (dict(out=KEYS), "overlaps the cache"),
    (dict(out=PAGES), "overlaps the cache"),
    (dict(out=LENGTHS), "overlaps the cache"),
    (dict(rows=1 << 30), "2^30"),
])
def test_attention_refuses(change, word):
    refused("mi355x_mx4_attention", attention_args(**change), word)


def test_attention_refuses_workspaces():
    c = cache(n_pages=5000, pages_per_sequence=1000)
    n = capi.mx4_attention_workspace_bytes(c, 8, 3, 7, 16000)
    assert n > 0 and capi.mx4_attention_workspace_bytes(c, 8, 3, 7, 100) == 0
    long = dict(c=c, most=16000)
    for change in (dict(ws=0), dict(ws_bytes=n - 1), dict(ws=WS + 8)):
        refused("mi355x_mx4_attention", attention_args(**long, **change), "workspace")
    for at in (Q, OUT, KEYS, STARTS):
        refused("mi355x_mx4_attention", attention_args(**long, ws=at - 16), "overlaps")


def test_attention_is_limited():
    refused("mi355x_mx4_attention", attention_args(rows=(1 << 30) - 1, heads=16, q_row=4096, out_row=4096), "rows", -4)
    n = C.c_size_t(0)
    refused("mi355x_mx4_attention_workspace_bytes", (C.byref(cache()), *sz(8, 1 << 29, 7, 80), C.byref(n)), "sequences", -4)


def test_workspaces_hold_for_windows_and_types():
    """What is asked for with no window is enough with one (the call does not ask again)."""
    for kv, dim in ((1, 64), (8, 128), (3, 256)):
        c = cache(kv_heads=kv, head_dim=dim, row_bytes=ref.row_bytes(kv * dim), n_pages=10 ** 6, pages_per_sequence=10 ** 5)
        sizes = [capi.mx4_attention_workspace_bytes(c, kv * 2, 3, rows, most) for rows in (1, 3, 500) for most in (10, 5000, 10 ** 6)]
        assert all(s % 16 == 0 for s in sizes)


@pytest.mark.parametrize("call", ["mi355x_mx4_cache_write", "mi355x_mx4_attention"])
def test_nothing_to_do(call):
    args = write_args if call.endswith("write") else attention_args
    for change in (dict(rows=0), dict(sequences=0)):
        assert getattr(capi.lib(), call)(*args(**change)) == 0


def adapters(**change):
    a = dict(down=KEYS, up=VALUES, scales=PAGES, count=3, rank=4, type=2)
    a.update(change)
    return capi.Mx4Adapters(**a)


def fc_args(a=None, out=OUT, out_type=1, out_row=200, x=X, in_type=1, in_row=200, w=W, w_row=80, bias=0, of_row=LENGTHS, M=5, K=100,
            N=100, act=0, ws=WS, ws_bytes=1 << 30):
    return (*vp(out), out_type, *sz(out_row), *vp(x), in_type, *sz(in_row), *vp(w), *sz(w_row), *vp(bias),
            C.byref(a) if a is not None else C.byref(adapters()), *vp(of_row), *sz(M, K, N), act, *vp(ws), *sz(ws_bytes), None)


@pytest.mark.parametrize("change, word", [
    (dict(a=adapters(type=3)), "none of the float types"),
    (dict(a=adapters(rank=1025)), "up to 1024"),
    (dict(a=adapters(count=1 << 31)), "adapters"),
    (dict(a=adapters(down=0)), "NULL"),
    (dict(a=adapters(up=0)), "NULL"),
    (dict(of_row=0), "NULL"),
    (dict(a=adapters(down=KEYS + 1)), "multiples of 2"),
    (dict(a=adapters(type=0, up=VALUES + 2)), "multiples of 4"),
    (dict(a=adapters(scales=PAGES + 2)), "multiples of 4"),
    (dict(of_row=LENGTHS + 1), "multiples of 4"),
    (dict(a=adapters(count=0x7fffffff, rank=1024), N=0x7fffffff, out_row=1 << 33), "adapters"),
    (dict(act=2), "activation"),
    (dict(bias=STARTS + 2), "multiple of 4"),
    (dict(out_row=198), "take 200"),
    (dict(w_row=64), "take 80"),
    (dict(out=X + 100), "overlaps"),
    (dict(out=KEYS + 2), "overlaps"),
    (dict(out=VALUES - 100), "overlaps"),
    (dict(out=PAGES), "overlaps"),
    (dict(out=LENGTHS), "overlaps"),
    (dict(ws=0), "workspace"),
    (dict(ws=WS + 8), "workspace"),
    (dict(ws_bytes=100), "workspace"),
    (dict(ws=KEYS - 16), "overlaps"),
    (dict(ws=X - 16), "overlaps"),
])
def test_adapters_refuse(change, word):
    refused("mi355x_mx4_fc_adapters", fc_args(**change), word)


def test_no_adapters_are_refused():
    args = fc_args()
    refused("mi355x_mx4_fc_adapters", (*args[:9], None, *args[10:]), "no adapters")


def test_conveniences_refuse_shapes():
    rng = np.random.default_rng(0)
    b = aref.Batch(rng, [20, 3], [1, 1], 2, 64, 16)
    q = np.zeros((2, 256), np.float32)
    for change in (dict(q=q[:, :200]), dict(starts=b.starts[:2]), dict(pages=b.pages[:1]), dict(page_tokens=24),
                   dict(out=np.zeros((2, 255), np.float32))):
        a = dict(q=q, starts=b.starts, page_tokens=16, pages=b.pages, out=None)
        a.update(change)
        with pytest.raises(capi.MI355XError):
            capi.mx4_attention(a["q"], 4, b.keys, b.values, a["starts"], b.lengths, 2, 64, a["page_tokens"], a["pages"], out=a["out"])
    with pytest.raises(capi.MI355XError):
        capi.mx4_cache_write(b.keys, b.values, q[:, :100], q[:, :100], b.starts, b.lengths, 2, 64, 16, b.pages)
    w = np.zeros((5, 80), np.uint8)
    with pytest.raises(capi.MI355XError):
        capi.mx4_fc_adapters(np.zeros((2, 100), np.float32), 0, w, None, 100, np.zeros((1, 4, 99), np.float32),
                             np.zeros((1, 5, 4), np.float32), np.zeros(2, np.int32))


def test_reference_attention_by_hand():
    """The oracle of the GPU tests on two tokens that can be worked out on paper."""
    b = aref.Batch(np.random.default_rng(1), [2], [2], 1, 64, 16)
    at = b.places(0, 2)
    k, v = np.zeros((2, 64)), np.zeros((2, 64))
    k[0, 0], k[1, 0], v[0, 0], v[1, 0] = 1, 2, 4, -1
    b.keys[at], b.values[at] = ref.rows_of(k), ref.rows_of(v)
    q = np.zeros((2, 64))
    q[:, 0] = np.log(3)
    got, err, used = aref.attention(b, q, 1, ref.F32, scale=1.0)
    assert used.all() and got[0, 0] == 4 and abs(got[1, 0] - (3 * 4 - 9) / 12) < 1e-12 and (err < 1e-3).all()
    got, _, _ = aref.attention(b, q, 1, ref.F32, scale=1.0, window=1)
    assert got[1, 0] == -1
