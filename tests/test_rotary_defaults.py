"""Frequencies with what the caller leaves out, and past a double's range (CPU)."""
import numpy as np
import pytest

import airkv
from airkv import rotary


def _same(x, y):
    return np.array_equal(x[0], y[0]) and x[1] == y[1]


def test_each_scaling_has_its_own_default_of_high():
    """Between 1 and 4 turns for "bands", 1 and 32 for "ramp": the published rules' choices."""
    for scaling, high in (("bands", 4.0), ("ramp", 32.0)):
        got = rotary.frequencies(128, 10000.0, scaling, 8.0, 4096.0)
        assert _same(got, rotary.frequencies(128, 10000.0, scaling, 8.0, 4096.0, 1.0, high))
        assert not _same(got, rotary.frequencies(128, 10000.0, scaling, 8.0, 4096.0, 1.0, 36.0 - high))
        # a low above the default is refused as a low above any high
        with pytest.raises(airkv.AirKvError):
            rotary.frequencies(128, 10000.0, scaling, 8.0, 4096.0, low=high)


def test_a_base_past_the_largest_double_is_refused():
    """base * factor^(rot_dim / (rot_dim - 2)): infinite, it gave the frequencies 1, 0, 0, ..."""
    assert np.isfinite(rotary.frequencies(64, 1e6, "base", 1e250)[0]).all()
    for rot, factor in ((4, 1e200), (64, 1e305)):
        with pytest.raises(airkv.AirKvError) as e:
            rotary.frequencies(rot, 1e6, "base", factor)
        assert e.value.code == airkv.AIR_KV_E_INVALID_ARG
