"""Scratch memory of the decoding handles: whose buffer a call gets, on the CPU."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROCM = "/opt/rocm/include"


@pytest.mark.skipif(not os.path.isdir(ROCM), reason="no HIP headers")
def test_no_two_streams_share_a_buffer(tmp_path):
    """Threads' own streams have one name: their buffers are kept apart by the thread."""
    exe = str(tmp_path / "scratch_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I" + ROCM, "-pthread",
                    os.path.join(HERE, "scratch_check.cc"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
