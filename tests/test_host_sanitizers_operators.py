"""The checks of arguments of the norm, the drawing of tokens and the clipping, as
tests/test_host_sanitizers.py runs the other CPU tests: in a child process with the
host side of the library under AddressSanitizer and UndefinedBehaviorSanitizer."""
import glob
import os

import pytest

from test_host_sanitizers import HOST_LIB, _child


def test_refusals_under_asan_and_ubsan():
    rt = sorted(glob.glob("/opt/rocm/lib/llvm/lib/clang/*/lib/linux/libclang_rt.asan-x86_64.so"))
    if not rt or not os.path.exists(HOST_LIB):
        pytest.skip("host sanitizer build or clang's ASan runtime absent")
    out = _child({"ORDA_HIP_LIB": HOST_LIB, "LD_PRELOAD": rt[-1]},
                 ["-m", "pytest", "tests/test_rms_norm_cpu.py", "tests/test_sampling_cpu.py", "tests/test_clip_cpu.py", "-q",
                  "-m", "not gpu", "-p", "no:cacheprovider"])
    assert " passed" in out, out[-2000:]
