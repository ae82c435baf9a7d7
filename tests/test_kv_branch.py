"""Forks and compactions of the paged KV cache: the host bookkeeping under
AddressSanitizer + UBSan, and the refusals that need no GPU."""
import os
import shutil
import subprocess

import numpy as np
import pytest

from purebee_amd import native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not installed")
def test_sequences_keep_their_rows(tmp_path):
    exe = str(tmp_path / "branch")
    r = subprocess.run(["g++", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                        "-std=c++17", "-Wall", "-I", os.path.join(ROOT, "include"),
                        "-I", os.path.join(ROOT, "purebee_amd", "csrc", "runtime"),
                        os.path.join(ROOT, "tests", "kv_branch_main.cpp"), "-o", exe],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    env = dict(os.environ)
    env.pop("LD_PRELOAD", None)
    r = subprocess.run([exe], capture_output=True, text=True, env=env, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    words = r.stdout.split()
    met = dict(zip(words[::2], (int(x) for x in words[1::2])))
    assert min(met[k] for k in ("grown", "copies", "packs", "refused", "forks")) > 1000  # every side was met
    assert met["launches"] > 20  # compactions with fewer free pages than they fill


def test_null_handles_are_refused():
    L = native.load_library()
    for rc in (L.pbx_kv_fork(None, 0, None, None, None), L.pbx_kv_compact(None, 0, None, None, None)):
        assert rc == -1
        assert b"not a live cache" in L.pbx_last_error(None)


def test_lists_of_numbers():
    """What sequences and positions may be given as."""
    for a in ([3, 1, 2**31 - 1], (3, 1, 2**31 - 1), np.array([3, 1, 2**31 - 1]), np.array([3, 1, 2**31 - 1], np.uint32),
              np.array([3, 0, 1, 0, 2**31 - 1, 0], np.int32)[::2]):
        got = native._i32(a)
        assert got.dtype == np.int32 and got.flags.c_contiguous and got.tolist() == [3, 1, 2**31 - 1]
    for empty in ([], np.zeros(0, np.int64), np.zeros(0, np.int32), range(0)):
        assert native._i32(empty).shape == (0,)
    for a in ([2**31], np.array([-2**31 - 1]), np.array([2**31], np.uint32), np.array([2**63], np.uint64)):
        with pytest.raises(OverflowError):
            native._i32(a)
    for a in ([[1, 2], [3, 4]], np.ones((2, 2), np.int32), np.ones((2, 2), np.int64)):
        with pytest.raises(ValueError):
            native._i32(a)
