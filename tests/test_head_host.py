"""Log probabilities straight from a head: its calls on the host, without a GPU."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not installed")
def test_memory_that_runs_out_is_an_error(tmp_path):
    """PBX_ENOMEM wherever an allocation of a call fails, and no exception past the C entry points."""
    exe, src = str(tmp_path / "head"), os.path.join(ROOT, "purebee_amd", "csrc", "runtime")
    r = subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-Wall", "-Wno-unused-result", "-D__HIP_PLATFORM_AMD__",
                        "-I", os.path.join(ROOT, "include"), "-I", src, "-I", os.path.join(ROCM, "include"),
                        os.path.join(ROOT, "tests", "head_host_main.cpp"), os.path.join(src, "pbx_head.cpp"),
                        os.path.join(src, "pbx_gemm.cpp"), "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, (r.returncode, r.stdout, r.stderr[-3000:])
    refused, planned = (int(x) for x in r.stdout.split()[1::2])
    assert refused > 100 and planned > 1000
