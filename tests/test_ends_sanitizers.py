"""The norms', embedding's and distillation's host checks under AddressSanitizer and UBSan (no GPU needed)."""

import os
import pathlib
import subprocess
import sys

import pytest

ROOT = pathlib.Path(__file__).resolve().parents[1]


def test_host_checks_are_clean_under_asan_and_ubsan():
    from mfattn import build

    if os.environ.get("PYTEST_XDIST_WORKER"):
        pytest.skip("its build shares objects with another test's")
    runtime = build.sanitizer_runtime()
    if runtime is None:
        pytest.skip("no clang AddressSanitizer runtime under /opt/rocm/llvm")
    env = dict(os.environ, LD_PRELOAD=str(runtime), MFATTN_LIB=str(build.build_sanitized()),
               ASAN_OPTIONS="detect_leaks=0:halt_on_error=1",
               UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1")
    proc = subprocess.run(
        [sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider", "-m", "not gpu",
         "tests/test_ends_checks.py", "tests/test_ends_sizes.py"], cwd=ROOT, env=env,
        capture_output=True, text=True, timeout=600)
    report = proc.stdout[-3000:] + proc.stderr[-3000:]
    assert "AddressSanitizer" not in proc.stderr and "runtime error" not in proc.stderr, report
    assert proc.returncode == 0 and "passed" in proc.stdout, report
