"""The checks of tests/test_paged_calls.py again, against the host-side ASan + UBSan build that
tests/test_abi_sanitized.py makes (no GPU: they return before a launch)."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT
from test_abi_sanitized import CSRC, HIPCC, SAN_LIB, _asan_runtime


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc is needed to build the sanitizer variant")
def test_the_paged_calls_under_asan_and_ubsan():
    rt = _asan_runtime()
    if rt is None:
        pytest.skip("the clang AddressSanitizer runtime is not installed")
    build = subprocess.run(["make", "-C", CSRC, "-j8", "sanitize"], capture_output=True, text=True, timeout=900)
    assert build.returncode == 0, build.stdout[-2000:] + build.stderr[-2000:]
    env = dict(os.environ, LD_PRELOAD=rt, DMLA_LIBRARY=SAN_LIB,
               ASAN_OPTIONS="detect_leaks=0:halt_on_error=1:alloc_dealloc_mismatch=0:detect_odr_violation=0",
               UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1")
    run = subprocess.run([sys.executable, "-m", "pytest", os.path.join(ROOT, "tests", "test_paged_calls.py"), "-q", "-x", "-p", "no:cacheprovider"],
                         cwd=ROOT, env=env, capture_output=True, text=True, timeout=900)
    log = run.stdout[-4000:] + run.stderr[-4000:]
    assert run.returncode == 0 and " passed" in run.stdout, log
    assert "AddressSanitizer" not in run.stderr and "runtime error" not in run.stderr, log
