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
