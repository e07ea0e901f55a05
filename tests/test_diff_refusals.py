"""Calls of differential attention and of compaction that are refused before anything
else is looked at (no GPU)."""
import ctypes

import airkv
from airkv import _lib


def test_a_missing_pool_is_refused():
    lib, n = _lib.load(), ctypes.c_size_t()
    size = ctypes.byref(n)
    for got in (lib.air_paged_diff_decode_workspace_size(None, 8, 1, 1, 64, size),
                lib.air_paged_diff_decode(None, None, None, airkv.F32, 8, None, 0, None, None, 1, 1, 0.125, 64, None, 0.0, 1.0, None,
                                          0, None, airkv.F32),
                lib.air_paged_diff_prefill_workspace_size(None, 8, 1, 1, size),
                lib.air_paged_diff_prefill(None, None, None, airkv.F32, 8, None, 0, None, 1, 1, None, None, 1, 1, 0.125, None, 0.0,
                                           1.0, None, 0, None, airkv.F32),
                lib.air_kv_compact(None, None, None, None, 1, 1, None, None, 1),
                lib.air_kv_session_compact(None, None, None, 0)):
        assert got == airkv.AIR_KV_E_INVALID_ARG
