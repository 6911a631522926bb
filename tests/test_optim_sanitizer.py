"""Bounds and undefined-behaviour check of the optimizer-side kernels without a
GPU, as tests/test_sanitizer.py does it for the collectives' kernels."""
import glob
import os
import subprocess
import sys

import pytest

from conftest import HOST_CLANG, ROOT
from optim_oracle import cpu_library


@pytest.fixture(scope="module")
def sanitizer_run():
    runtimes = glob.glob("/opt/rocm/lib/llvm/lib/clang/*/lib/linux/libclang_rt.asan-x86_64.so")
    if not os.path.exists(HOST_CLANG) or not runtimes:
        pytest.skip("no host clang++ with a shared AddressSanitizer runtime")
    lib = cpu_library(os.path.join(ROOT, "tests", "build", "libpccl_optim_cpu_san.so"),
                      ("-O0", "-fsanitize=address,undefined", "-fno-sanitize=vptr", "-shared-libsan", "-fno-omit-frame-pointer"))
    env = dict(os.environ, LD_PRELOAD=runtimes[0], ASAN_OPTIONS="detect_leaks=0:abort_on_error=0:exitcode=86",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=0")
    return subprocess.run([sys.executable, os.path.join(ROOT, "tests", "optim_asan_check.py"), lib],
                          capture_output=True, text=True, env=env, timeout=900)


def test_optimizer_kernels_stay_in_bounds(sanitizer_run):
    p = sanitizer_run
    assert p.returncode == 0, (p.stdout[-2000:], p.stderr[-4000:])
    assert "AddressSanitizer" not in p.stderr, p.stderr[-4000:]
    assert "ASAN CHECK OK" in p.stdout


def test_optimizer_kernels_show_no_undefined_behaviour(sanitizer_run):
    p = sanitizer_run
    assert "runtime error" not in p.stderr, p.stderr[-4000:]
    assert "ASAN CHECK OK" in p.stdout
