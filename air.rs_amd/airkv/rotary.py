"""Frequencies of rotary positions (air_rotary_frequencies): as trained, or scaled for
contexts longer than a model was trained on.  KvPool.append_rotary and KvPool.rotate take
them as a float32 tensor on the device."""
from __future__ import annotations

import ctypes

import numpy as np

from . import _lib

SCALINGS = ("plain", "linear", "base", "bands", "ramp")


def frequencies(rot_dim, base=10000.0, scaling="plain", factor=1.0, trained_len=0.0, low=1.0, high=None):
    """(float32 array [rot_dim / 2], magnitude).  `scaling`: "plain"; "linear" (positions divided by
    factor); "base" (a larger base); "bands" (by wavelength against trained_len, between low and
    high turns); "ramp" (by pair, between those that turn `high` and `low` times over trained_len,
    with a magnitude).  `high` is 4 for bands and 32 for the ramp where it is left out."""
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}")
    if high is None:
        high = 32.0 if scaling == "ramp" else 4.0
    out, magnitude = np.empty(max(0, rot_dim) // 2, np.float32), ctypes.c_float()
    _lib.check(_lib.load().air_rotary_frequencies(rot_dim, base, SCALINGS.index(scaling), factor, trained_len, low, high,
                                                  out.ctypes.data_as(ctypes.c_void_p), ctypes.byref(magnitude)),
               "air_rotary_frequencies")
    return out, magnitude.value
