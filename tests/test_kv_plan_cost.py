"""Planning a batch costs what the batch is, not what the cache could hold."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not installed")
def test_plans_do_not_cost_by_the_sequences_that_could_be(tmp_path):
    """Two sequences' rows, planned and taken back, in caches of 64 and of 2^20 sequence ids: the least of 300 times each.
    (A byte for every id, cleared each time, made it a hundred times as long.)"""
    exe = str(tmp_path / "cost")
    r = subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-I", os.path.join(ROOT, "include"),
                        "-I", os.path.join(ROOT, "purebee_amd", "csrc", "runtime"),
                        os.path.join(ROOT, "tests", "kv_plan_cost_main.cpp"), "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-3000:]
    few, many = (float(x) for x in r.stdout.split()[1:])
    assert many <= 10 * few, (few, many)
