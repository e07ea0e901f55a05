"""The spans by which entry points find arguments that overlap: tests/span_check.cpp, built with g++."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_spans(tmp_path):
    exe = str(tmp_path / "span_check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=undefined", "-I",
                    os.path.join(HERE, "..", "air.rs_amd", "csrc"), "-o", exe, os.path.join(HERE, "span_check.cpp")], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stdout + out.stderr
