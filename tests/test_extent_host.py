"""Which buffers the decoding calls take to overlap, on the CPU."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROCM = "/opt/rocm/include"


@pytest.mark.skipif(not os.path.isdir(ROCM), reason="no HIP headers")
def test_parts_side_by_side_do_not_overlap(tmp_path):
    """Queries, keys and values side by side in a row, in a head or in a head's rows share no byte; what shares one is
    always found."""
    exe = str(tmp_path / "extent_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I" + ROCM, os.path.join(HERE, "extent_check.cc"),
                    "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
