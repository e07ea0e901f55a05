"""Frequencies of rotary positions and the calls that are refused without a pool (no GPU)."""
import ctypes
import math

import numpy as np
import pytest

import airkv
from airkv import _lib, rotary

HALF_STEP = 2.0 ** -24


def _plain(rot, base):
    return [base ** (-2.0 * i / rot) for i in range(rot // 2)]


def _close(got, want):
    want = np.array(want)
    assert got.dtype == np.float32
    # one rounding to f32; the powers' own errors in 64 bits are 2^-50 and less
    assert (np.abs(got - want) <= (HALF_STEP + 2.0 ** -50) * want).all()


@pytest.mark.parametrize("rot,base", [(2, 10000.0), (8, 10000.0), (64, 500000.0), (128, 1e6), (256, 10000.0)])
def test_frequencies(rot, base):
    f, m = rotary.frequencies(rot, base)
    _close(f, _plain(rot, base))
    assert m == 1.0
    f, m = rotary.frequencies(rot, base, "linear", factor=4.0)
    _close(f, [x / 4 for x in _plain(rot, base)])
    assert m == 1.0
    if rot > 2:
        f, m = rotary.frequencies(rot, base, "base", factor=8.0)
        _close(f, _plain(rot, base * 8.0 ** (rot / (rot - 2))))
        assert f[0] == 1.0 and abs(f[-1] * 8 / rotary.frequencies(rot, base)[0][-1] - 1) < 1e-6 and m == 1.0


def test_bands():
    """Short wavelengths keep their frequency, long ones are divided, between them a blend."""
    length, low, high, factor = 8192.0, 1.0, 4.0, 8.0
    want = []
    for f in _plain(128, 500000.0):
        w = 2 * math.pi / f
        if w < length / high:
            want.append(f)
        elif w > length / low:
            want.append(f / factor)
        else:
            t = (length / w - low) / (high - low)
            want.append((1 - t) * f / factor + t * f)
    got, m = rotary.frequencies(128, 500000.0, "bands", factor, length, low, high)
    _close(got, want)
    assert m == 1.0 and 0 < sum(x != y and x != y / factor for x, y in zip(want, _plain(128, 500000.0)))


@pytest.mark.parametrize("rot,length", [(128, 4096.0), (64, 32768.0), (32, 20.0)])
def test_ramp(rot, length):
    base, low, high, factor = 10000.0, 1.0, 32.0, 16.0

    def turns(n):
        return rot * math.log(length / (2 * math.pi * n)) / (2 * math.log(base))
    a, b = max(0.0, math.floor(turns(high))), min(rot - 1.0, math.ceil(turns(low)))
    b = b if b > a else a + 0.001
    want = []
    for i, f in enumerate(_plain(rot, base)):
        t = min(1.0, max(0.0, (i - a) / (b - a)))
        want.append((1 - t) * f + t * f / factor)
    got, m = rotary.frequencies(rot, base, "ramp", factor, length, low, high)
    _close(got, want)
    assert m == np.float32(0.1 * math.log(factor) + 1)
    assert rotary.frequencies(rot, base, "ramp", 1.0, length, low, high)[1] == 1.0


@pytest.mark.parametrize("bad", [
    dict(rot_dim=0), dict(rot_dim=7), dict(rot_dim=-2), dict(base=1.0), dict(base=math.inf), dict(base=math.nan),
    dict(scaling="linear", factor=0.5), dict(scaling="base", factor=math.nan), dict(scaling="base", rot_dim=2, factor=2.0),
    dict(scaling="bands", factor=2.0), dict(scaling="ramp", factor=2.0, trained_len=4096.0, low=4.0, high=4.0),
    dict(scaling="ramp", factor=2.0, trained_len=math.inf, low=1.0, high=4.0), dict(scaling="bands", factor=2.0, trained_len=1.0, low=0.0)])
def test_frequencies_refused(bad):
    with pytest.raises(airkv.AirKvError) as e:
        rotary.frequencies(**{"rot_dim": 64, **bad})
    assert e.value.code == airkv.AIR_KV_E_INVALID_ARG
    with pytest.raises(ValueError):
        rotary.frequencies(64, scaling="other")


def test_a_missing_pool_or_output_is_refused():
    lib, m = _lib.load(), ctypes.c_float()
    out = np.zeros(4, np.float32)
    for got in (lib.air_rotary_frequencies(8, 10.0, 0, 1.0, 0.0, 0.0, 0.0, None, ctypes.byref(m)),
                lib.air_rotary_frequencies(8, 10.0, 0, 1.0, 0.0, 0.0, 0.0, out.ctypes.data, None),
                lib.air_rotary_frequencies(8, 10.0, 9, 1.0, 0.0, 0.0, 0.0, out.ctypes.data, ctypes.byref(m)),
                lib.air_kv_append_rotary(None, None, None, 0, 0, None, 0, None, 0, 0, None, None, 1, None, 8, 0, 1.0, None, 0),
                lib.air_kv_rotate(None, None, None, 1, 1, None, None, None, 1, None, 8, 0)):
        assert got == airkv.AIR_KV_E_INVALID_ARG
