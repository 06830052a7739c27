"""The paged cache's argument checks and index arithmetic (host code of the
library, csrc/paged_args.hpp) on the CPU, under AddressSanitizer and
UndefinedBehaviorSanitizer; the calls' refusals that need no device."""
import ctypes
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
SRC = os.path.join(HERE, "sanitize", "paged_args_check.cpp")


def test_paged_args_under_sanitizers(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    exe = str(tmp_path / "paged_args_check")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-g", "-O1", "-fsanitize=address,undefined",
                    "-fno-sanitize-recover=all", "-o", exe, SRC], check=True, capture_output=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "all cases held" in r.stdout, r.stdout + r.stderr[-3000:]


def test_structs_have_the_header_sizes(pkg):
    """The C structs' sizes on this ABI, as ctypes lays the mirrors out."""
    assert ctypes.sizeof(pkg.PagedKV) == 64
    assert ctypes.sizeof(pkg.PagedBatch) == 40
    assert ctypes.sizeof(pkg.LoraAdapterDesc) == 24


def test_null_context_is_refused(pkg):
    lib, inv = pkg.lib(), pkg.QORA_HIP_E_INVALID
    assert lib.qora_hip_paged_append(None, None, None, 1, None, 0, None, 0, None, 0, None, 0, None, None, 0, 0,
                                     None) == inv
    assert lib.qora_hip_paged_attn_prepare(None, 1, 1, 1, 1, 64, None) == inv
    assert lib.qora_hip_paged_attn_run(None, 0, None, None, None, 0, None, 0, None) == inv
    assert lib.qora_hip_paged_attn_release(None, 0) == inv
    assert lib.qora_hip_lora_upload(None, None, 1, 32, 32, 1, None) == inv
    assert lib.qora_hip_lora_release(None, 0) == inv
    assert lib.qora_hip_gemm_lora(None, 0, 0, None, None, 1, None, None) == inv
