"""The numpy conveniences of microscaled rows, their products and group norm: what they refuse before
anything is on the device, and what they pass on."""
import numpy as np
import pytest

from glow_amd import capi
from tests import mx4_ref as ref


class Reached(Exception):
    """The call went on to the device."""


@pytest.fixture(autouse=True)
def _no_device(monkeypatch):
    def reached(*_):
        raise Reached()
    monkeypatch.setattr(capi, "to_device", reached)
    monkeypatch.setattr(capi.DeviceBuffer, "__init__", reached)


ROWS = ref.rows_of(np.ones((5, 100)))
IMAGE = np.ones((2, 9, 12), np.float32)


@pytest.mark.parametrize("length", [0, 1, 4, 6])
def test_a_bias_of_another_length_is_refused(length):
    with pytest.raises(capi.MI355XError, match="bias"):
        capi.mx4_fc(np.ones((3, 100), np.float32), capi.TYPE_F32, ROWS, np.ones(length, np.float32), 100)
    with pytest.raises(capi.MI355XError, match="bias"):
        capi.mx4_fc(ROWS[:3], capi.TYPE_MX4, ROWS, np.ones(length, np.float32), 100)


@pytest.mark.parametrize("length", [0, 1, 11, 13])
def test_gamma_and_beta_of_another_length_are_refused(length):
    for out_type in (None, capi.TYPE_MX4):
        with pytest.raises(capi.MI355XError, match="gamma"):
            capi.group_norm(IMAGE, 3, np.ones(length, np.float32), np.ones(12, np.float32), out_type=out_type)
        with pytest.raises(capi.MI355XError, match="beta"):
            capi.group_norm(IMAGE, 3, None, np.ones(length, np.float32), out_type=out_type)


def test_values_in_the_place_of_microscaled_rows_are_refused():
    # (a conversion to bytes would pass them off as codes)
    x = np.ones((5, 80), np.float32)
    for call in (lambda: capi.mx4_dequantize(x, 100), lambda: capi.mx4_fc(x, capi.TYPE_MX4, ROWS, None, 100),
                 lambda: capi.mx4_fc(ROWS, capi.TYPE_MX4, x, None, 100)):
        with pytest.raises(AssertionError):
            call()


def test_what_fits_goes_on():
    for call in (lambda: capi.mx4_fc(ROWS, capi.TYPE_MX4, ROWS, np.ones(5), 100),
                 lambda: capi.mx4_fc(ROWS, capi.TYPE_MX4, ROWS, None, 100),
                 lambda: capi.group_norm(IMAGE, 3, np.ones(12), None), lambda: capi.mx4_dequantize(ROWS, 100)):
        with pytest.raises(Reached):
            call()


class Device:
    def __init__(self, shape, dtype=np.uint8):
        self.shape, self.dtype = shape, np.dtype(dtype)

    def numpy(self):
        return None


@pytest.mark.parametrize("rows", [lambda x: x[::3][:1], lambda x: x[::-1][:1], lambda x: x[:1], lambda x: x[:0], lambda x: x])
def test_rows_are_as_far_apart_as_they_are_long(monkeypatch, rows):
    """numpy leaves the stride of an axis of one or no rows as it was, whatever it calls contiguous."""
    seen = []
    monkeypatch.setattr(capi, "to_device", lambda a: Device(a.shape, a.dtype))
    monkeypatch.setattr(capi.DeviceBuffer, "empty", classmethod(lambda cls, shape, dtype: Device(shape, dtype)))
    monkeypatch.setattr(capi, "launch_mx4_quantize", lambda *a: seen.append(a))
    x = rows(np.ones((9, 40), np.float32))
    capi.mx4_quantize(x)
    (_, _, _, type_, src_row_bytes, n, cols), = seen
    assert (type_, src_row_bytes, n, cols) == (capi.TYPE_F32, 160, x.shape[0], 40)
