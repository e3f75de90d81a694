"""Microscaled 4-bit rows and the entry points around them, as far as no GPU is involved: the
host quantiser, sizes, and what the launches refuse."""
import ctypes as C

import numpy as np
import pytest

from glow_amd import capi
from tests import mx4_ref as ref

P = 1 << 20          # addresses that no refused call touches
Q, R, S = P + (1 << 32), P + (2 << 32), P + (3 << 32)


def special_rows():
    rng = np.random.default_rng(0)
    x = (rng.normal(0, 1, (40, 415)) * 10.0 ** rng.integers(-3, 4, (40, 1))).astype(np.float32)
    x[0] = 0
    x[1] = -0.0
    x[2, 7] = np.inf
    x[3, 300] = np.nan
    x[4, 40] = -np.inf
    x[5, ::2] *= np.float32(1e-38)
    x[6] = np.float32(1e-45)
    x[7] = np.finfo(np.float32).max
    x[8] = np.float32(2.0 ** -126)
    x[9, :32] = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 7] * 4, np.float32) * np.tile([1, -1], 16)
    x[9, 32:64] = np.nextafter(x[9, :32], np.float32(100))
    x[9, 64:96] = np.nextafter(x[9, :32], np.float32(-100))
    x[9, [0, 32, 64]] = 4
    return x


@pytest.mark.parametrize("cols", [1, 31, 32, 33, 127, 128, 129, 415])
def test_host_quantiser_is_the_definition(cols):
    x = special_rows()[:, :cols]
    assert capi.mx4_row_bytes(cols) == ref.row_bytes(cols)
    with np.errstate(invalid="ignore"):
        want = ref.rows_of(x)
    np.testing.assert_array_equal(capi.mx4_quantize_host(x), want)


def test_reference_rows_round_trip():
    x = special_rows()
    rows = ref.rows_of(np.where(np.isfinite(x), x, 1))
    back = ref.values(rows, 415)
    np.testing.assert_array_equal(ref.values(ref.rows_of(back), 415), back)
    assert ref.row_bytes(0) == capi.mx4_row_bytes(0) == 0


def refused(fn, args, word, code=-1):
    rc = getattr(capi.lib(), fn)(*args)
    said = capi.lib().mi355x_last_error().decode()
    assert rc == code and word in said, (rc, said)


def sz(*v):
    return tuple(C.c_size_t(x) for x in v)


def vp(*v):
    return tuple(C.c_void_p(x) for x in v)


def quantize_args(dst=P, dst_row=80, src=Q, type_=0, src_row=400, rows=3, cols=100):
    return (*vp(dst), *sz(dst_row), *vp(src), type_, *sz(src_row, rows, cols), None)


@pytest.mark.parametrize("change, word, code", [
    (dict(type_=3), "none of the float types", -1),
    (dict(type_=7), "none of the float types", -1),
    (dict(dst=P + 8), "multiples of 16", -1),
    (dict(dst_row=88), "multiples of 16", -1),
    (dict(dst_row=64), "take 80", -1),
    (dict(src_row=396), "take 400", -1),
    (dict(src=Q + 2), "multiples of 4", -1),
    (dict(src_row=402), "multiples of 4", -1),
    (dict(dst=0), "NULL", -1),
    (dict(src=0), "NULL", -1),
    (dict(dst=Q + 800), "overlaps", -1),
    (dict(rows=1 << 32), "2^31", -1),
    (dict(cols=1 << 31, dst_row=1 << 40, src_row=1 << 40), "2^31", -1),
    (dict(rows=0x7fffffff, dst_row=1 << 60), "rows", -1),
])
def test_quantize_refuses(change, word, code):
    refused("mi355x_mx4_quantize", quantize_args(**change), word, code)
    if "type_" not in change:
        a = dict(dst=P, dst_row=80, src=Q, type_=0, src_row=400, rows=3, cols=100)
        a.update(change)
        refused("mi355x_mx4_dequantize", (*vp(a["src"]), 0, *sz(a["src_row"]), *vp(a["dst"]),
                                          *sz(a["dst_row"], a["rows"], a["cols"]), None), word, code)


def fc_args(out=P, out_type=0, out_row=400, x=Q, in_type=3, in_row=80, w=R, w_row=80, bias=0, M=5, K=100, N=100,
            act=0, ws=0, ws_bytes=0):
    return (*vp(out), out_type, *sz(out_row), *vp(x), in_type, *sz(in_row), *vp(w), *sz(w_row), *vp(bias),
            *sz(M, K, N), act, *vp(ws), *sz(ws_bytes), None)


@pytest.mark.parametrize("change, word", [
    (dict(out_type=4), "unknown element type"),
    (dict(in_type=-1), "unknown element type"),
    (dict(act=2), "activation"),
    (dict(act=5), "activation"),
    (dict(act=7), "activation"),
    (dict(w_row=64), "take 80"),
    (dict(w=R + 4), "multiples of 16"),
    (dict(in_row=72), "take 80"),
    (dict(x=Q + 8), "multiples of 16"),
    (dict(out_row=396), "take 400"),
    (dict(out_type=1, out=P + 1), "multiples of 2"),
    (dict(out_type=3, out_row=72), "take 80"),
    (dict(bias=S + 2), "multiple of 4"),
    (dict(out=0), "NULL"),
    (dict(x=0), "NULL"),
    (dict(w=0), "NULL"),
    (dict(out=Q + 100), "overlaps"),
    (dict(out=R + 4000), "overlaps"),
    (dict(out=S, bias=S + 800), "overlaps"),
    (dict(M=1 << 31), "2^31"),
])
def test_fc_refuses(change, word):
    refused("mi355x_mx4_fc", fc_args(**change), word)


def test_fc_refuses_a_workspace_that_does_not_fit():
    M, K, N = 3000, 1000, 1000
    need = capi.mx4_fc_workspace_bytes(M, K, N, capi.TYPE_F32)
    assert capi.mx4_fc_workspace_bytes(M, K, N, capi.TYPE_MX4) == 0
    assert capi.mx4_fc_workspace_bytes(1, K, N, capi.TYPE_F32) == 0       # a single row needs none
    assert need >= M * capi.mx4_row_bytes(K)
    a = dict(in_type=0, in_row=4000, M=M, K=K, N=N, w_row=capi.mx4_row_bytes(K), out_row=4000)
    for change in (dict(), dict(ws=S, ws_bytes=need - 1), dict(ws=S + 4, ws_bytes=need)):
        refused("mi355x_mx4_fc", fc_args(**a, **change), "workspace")
    refused("mi355x_mx4_fc", fc_args(**a, ws=R + 160, ws_bytes=need), "overlaps")
    refused("mi355x_mx4_fc", fc_args(**a, ws=P + 160, ws_bytes=need), "overlaps")
    with pytest.raises(capi.MI355XError):
        capi.mx4_fc_workspace_bytes(M, K, N, 9)


def norm_args(out=P, out_type=0, out_row=400, x=Q, in_type=0, in_row=400, gamma=0, beta=0, N=2, pixels=9, C_=100,
              groups=4, eps=1e-5, act=0, ws=S, ws_bytes=1 << 20):
    return (*vp(out), out_type, *sz(out_row), *vp(x), in_type, *sz(in_row), *vp(gamma, beta),
            *sz(N, pixels, C_, groups), C.c_float(eps), act, *vp(ws), *sz(ws_bytes), None)


@pytest.mark.parametrize("change, word", [
    (dict(groups=3), "groups"),
    (dict(groups=0), "groups"),
    (dict(in_type=3), "none of the float types"),
    (dict(out_type=1), "result type"),
    (dict(out_type=3, out_row=64), "take 80"),
    (dict(out_type=3, out_row=88), "multiples of 16"),
    (dict(in_row=396), "take 400"),
    (dict(x=Q + 2), "multiples of 4"),
    (dict(eps=-1.0), "epsilon"),
    (dict(eps=float("nan")), "epsilon"),
    (dict(act=3), "activation"),
    (dict(gamma=R + 1), "multiples of 4"),
    (dict(beta=R + 2), "multiples of 4"),
    (dict(out=0), "NULL"),
    (dict(x=0), "NULL"),
    (dict(out=Q + 400), "overlaps"),
    (dict(out=Q, out_row=800), "overlaps"),
    (dict(out=P, gamma=P + 80), "overlaps"),
    (dict(N=1 << 20, pixels=1 << 20), "2^31"),
])
def test_group_norm_refuses(change, word):
    refused("mi355x_group_norm", norm_args(**change), word)


def test_group_norm_refuses_a_workspace_that_does_not_fit():
    N, pixels, C_, groups = 2, 5000, 100, 4
    need = capi.group_norm_workspace_bytes(N, pixels, C_, groups)
    a = dict(N=N, pixels=pixels, C_=C_, groups=groups)
    if need:
        for change in (dict(ws=0), dict(ws_bytes=need - 1), dict(ws=S + 4)):
            refused("mi355x_group_norm", norm_args(**a, **change), "workspace")
        refused("mi355x_group_norm", norm_args(**a, ws=Q + 160), "overlaps")
    with pytest.raises(capi.MI355XError):
        capi.group_norm_workspace_bytes(2, 9, 100, 7)


def test_empty_tensors_are_a_no_op():
    lib = capi.lib()
    for rows, cols in ((0, 100), (3, 0)):
        assert lib.mi355x_mx4_quantize(*quantize_args(dst=0, src=0, rows=rows, cols=cols) if not cols else
                                       quantize_args(rows=rows, cols=cols)) == 0
    assert lib.mi355x_mx4_fc(*fc_args(M=0)) == 0
    assert lib.mi355x_mx4_fc(*fc_args(N=0, w=0)) == 0
    assert lib.mi355x_group_norm(*norm_args(N=0)) == 0
    assert lib.mi355x_group_norm(*norm_args(pixels=0)) == 0
    assert lib.mi355x_group_norm(*norm_args(C_=0, groups=1)) == 0


def test_group_norm_workspace_of_more_groups_than_memory_is_refused():
    most = 0x7fffffff
    for N, pixels, groups in ((most, 1, most), (most, 1, 1 << 30), (1 << 30, most, 1 << 30)):
        with pytest.raises(capi.MI355XError, match="groups"):
            capi.group_norm_workspace_bytes(N, pixels, groups, groups)
    assert capi.group_norm_workspace_bytes(1 << 20, 1, 1 << 20, 1 << 20) >= 1 << 40
    # a slot is the more for every part that a slice may be cut into: never less for more pixels
    sizes = [capi.group_norm_workspace_bytes(3, pixels, 64, 8) for pixels in (1, 7, 100, 10 ** 6)]
    assert sizes == sorted(sizes) and sizes[0] > 0


def test_group_norm_refuses_workspaces_of_any_size_that_do_not_fit():
    for N, pixels, C_, groups in ((2, 5000, 100, 4), (2, 9, 100, 4), (1, 1, 9000, 1)):
        need = capi.group_norm_workspace_bytes(N, pixels, C_, groups)
        assert need > 0
        a = dict(N=N, pixels=pixels, C_=C_, groups=groups, in_row=4 * C_, out_row=4 * C_)
        for change in (dict(ws=0), dict(ws_bytes=need - 1), dict(ws_bytes=0), dict(ws=S + 4)):
            refused("mi355x_group_norm", norm_args(**a, **change), "workspace")
        refused("mi355x_group_norm", norm_args(**a, ws=Q + 160), "overlaps")
        refused("mi355x_group_norm", norm_args(**a, ws=P + 160), "overlaps")


def test_sizes_past_a_launch_are_not_supported():
    # 2^31 - 8 channels, each a group: 2^26 slices and more, of 64 threads; refused before any launch
    C_ = (1 << 31) - 8
    for pixels, channels in ((1, C_), (2000, 1 << 25)):
        need = capi.group_norm_workspace_bytes(8, pixels, channels, channels)
        far = dict(out=1 << 45, x=1 << 50, ws=1 << 55, ws_bytes=need, in_type=1, out_type=1, in_row=2 * channels, out_row=2 * channels)
        refused("mi355x_group_norm", norm_args(N=8, pixels=pixels, C_=channels, groups=channels, **far), "channels", -4)
    # 2^34 tiles of 128 x 128 results; 2^23 of 16 x 16
    refused("mi355x_mx4_fc", fc_args(out=1 << 55, x=1 << 45, w=1 << 50, M=1 << 24, N=1 << 24, out_row=1 << 26), "results", -4)
    refused("mi355x_mx4_fc", fc_args(out=1 << 55, x=1 << 45, w=1 << 50, M=3, N=1 << 27, out_row=1 << 29), "results", -4)
    refused("mi355x_mx4_quantize", quantize_args(dst=1 << 61, src=1 << 62, rows=1 << 22, cols=(1 << 31) - 8, src_row=1 << 33,
                                                 dst_row=1 << 31), "values", -4)
