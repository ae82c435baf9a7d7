"""The paged KV cache's host bookkeeping (purebee_amd/csrc/runtime/pbx_kv_plan.h)
under host AddressSanitizer + UBSan, and the refusals that need no GPU."""
import ctypes
import os
import shutil
import subprocess

import pytest

import purebee_amd as pb
from purebee_amd import native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not installed")
def test_plans_stay_inside_their_pages(tmp_path):
    exe = str(tmp_path / "plan")
    r = subprocess.run(["g++", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                        "-std=c++17", "-Wall", "-I", os.path.join(ROOT, "include"),
                        "-I", os.path.join(ROOT, "purebee_amd", "csrc", "runtime"),
                        os.path.join(ROOT, "tests", "kv_plan_main.cpp"), "-o", exe],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    env = dict(os.environ)
    env.pop("LD_PRELOAD", None)
    r = subprocess.run([exe], capture_output=True, text=True, env=env, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    taken, refused = (int(x) for x in r.stdout.split()[1::2])
    assert taken > 1000 and refused > 100  # both sides were met


def test_null_handles_are_refused():
    L = native.load_library()
    out = ctypes.c_void_p()
    cfg = native.KvConfig()
    assert L.pbx_kv_create(None, ctypes.byref(cfg), ctypes.byref(out)) == -1
    assert b"ctx is NULL" in L.pbx_last_error(None)
    assert L.pbx_kv_free(None) == 0 and L.pbx_kv_batch_free(None) == 0
    n, size = ctypes.c_int(), ctypes.c_size_t()
    for rc in (L.pbx_kv_info(None, ctypes.byref(n), ctypes.byref(size)),
               L.pbx_kv_length(None, 0, ctypes.byref(n)), L.pbx_kv_truncate(None, 0, 0),
               L.pbx_kv_batch_create(None, ctypes.byref(out)), L.pbx_kv_batch_set(None, 0, None, None, None),
               L.pbx_kv_batch_rows(None, ctypes.byref(n)),
               L.pbx_kv_append_dev(None, 0, None, 0, None, 0, None, 0, None, 0),
               L.pbx_kv_attention_dev(None, 0, None, 0, 0.0, None, 0),
               L.pbx_kv_read_dev(None, 0, None, 0, None, 0),
               L.pbx_logprobs_workspace(None, 1, 10, 0, ctypes.byref(size)),
               L.pbx_logprobs_dev(None, None, 0, 1, 10, None, 0, None, None, None, None, None, 0)):
        assert rc == -1
        assert L.pbx_last_error(None)


def test_constants_of_the_header():
    src = open(os.path.join(ROOT, "include", "pbx.h")).read()
    for name, value in (("PBX_KV_BLOCK", native.KV_BLOCK), ("PBX_LOGPROBS_TOP_MAX", native.LOGPROBS_TOP_MAX),
                        ("PBX_ROPE_NONE", native.ROPE["none"]), ("PBX_ROPE_PAIRS", native.ROPE["pairs"]),
                        ("PBX_ROPE_HALVES", native.ROPE["halves"])):
        line = next(x for x in src.splitlines() if x.startswith("#define " + name + " "))
        assert int(line.split()[2]) == value
    assert pb.KvCache and pb.KvBatch
