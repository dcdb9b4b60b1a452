"""The host code of windowed and linear attention against the AddressSanitizer +
UndefinedBehaviorSanitizer build (see test_sanitizers.py; CPU only)."""
import glob
import os
import subprocess

import pytest

from tests.conftest import ROOT
from tests.test_sanitizers import _run


def test_bounded_host_code_under_asan_ubsan():
    subprocess.run(["make", "-s", "-j8", "-C", os.path.join(ROOT, "loom-dataflow_amd", "csrc"),
                    "asan"], check=True, capture_output=True)
    lib = os.path.join(ROOT, "loom-dataflow_amd", "_build_asan", "libloom_hip_asan.so")
    rt = sorted(glob.glob("/opt/rocm/lib/llvm/lib/clang/*/lib/linux/libclang_rt.asan-x86_64.so"))
    if not rt:
        pytest.skip("clang's ASan runtime is not installed")
    assert " passed" in _run({"LD_PRELOAD": rt[-1], "LOOM_HIP_LIB": lib},
                             ["tests/test_bounded_validation.py"])
