"""The differential prefill's work division (air.rs_amd/csrc/kernels/
diff_prefill_plan.hpp) on the CPU, and what the new entry points refuse before any
device work."""
import ctypes
import os
import shutil
import subprocess
import tempfile

import pytest

import airkv

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "..", "air.rs_amd", "csrc")


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_work_division():
    with tempfile.TemporaryDirectory() as d:
        exe = os.path.join(d, "check")
        subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=undefined",
                        "-I", CSRC, "-o", exe, os.path.join(HERE, "diff_prefill_plan_check.cpp")], check=True)
        out = subprocess.run([exe], capture_output=True, text=True, timeout=300)
        print(out.stdout)
        assert out.returncode == 0, out.stdout + out.stderr
        assert ", 0 wrong" in out.stdout


def test_null_pool_is_refused():
    L = airkv.load()
    n = ctypes.c_size_t()
    assert L.air_paged_diff_decode_workspace_size(None, 8, 1, 1, 64, ctypes.byref(n)) == airkv.AIR_KV_E_INVALID_ARG
    assert L.air_paged_diff_prefill_workspace_size(None, 8, 1, 1, ctypes.byref(n)) == airkv.AIR_KV_E_INVALID_ARG
    assert L.air_paged_diff_decode(None, None, None, airkv.BF16, 8, None, 0, None, None, 1, 1, 1.0, 64, None, 0.0, 1.0,
                                   None, 0, None, airkv.BF16) == airkv.AIR_KV_E_INVALID_ARG
    assert L.air_paged_diff_prefill(None, None, None, airkv.BF16, 8, None, 0, None, 1, 1, None, None, 1, 1, 1.0, None,
                                    0.0, 1.0, None, 0, None, airkv.BF16) == airkv.AIR_KV_E_INVALID_ARG
    assert L.air_kv_compact(None, None, None, None, 1, 1, None, None, 1) == airkv.AIR_KV_E_INVALID_ARG
    assert L.air_kv_session_compact(None, None, None, 0) == airkv.AIR_KV_E_INVALID_ARG
