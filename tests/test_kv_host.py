"""The paged KV cache's calls on the host, against a GPU that is not there: what errors leave."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not installed")
    exe = str(tmp_path_factory.mktemp("kv") / "host")
    r = subprocess.run(["g++", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                        "-std=c++17", "-Wall", "-Wno-unused-result", "-D__HIP_PLATFORM_AMD__",
                        "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "purebee_amd", "csrc", "runtime"),
                        "-I", os.path.join(ROCM, "include"), os.path.join(ROOT, "tests", "kv_host_main.cpp"),
                        os.path.join(ROOT, "purebee_amd", "csrc", "runtime", "pbx_kv.cpp"), "-o", exe],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    env = dict(os.environ)
    env.pop("LD_PRELOAD", None)

    def run(what):
        r = subprocess.run([exe, what], capture_output=True, text=True, env=env, timeout=120)
        assert r.returncode == 0, r.stderr[-3000:]

    return run


def test_a_compaction_that_fails_midway(host):
    """Sequences keep what had not moved, and batches over the rest are refused."""
    host("failed_compactions")


def test_a_refused_set_changes_nothing(host):
    """Neither the sequences nor the batch, which goes on with the rows that it had."""
    host("refused_sets")


def test_memory_that_runs_out_is_an_error(host):
    """PBX_ENOMEM, nothing changed, and no exception past the C entry points."""
    host("memory_runs_out")
