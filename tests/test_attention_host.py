"""The C entries of the paged-cache operators on the CPU: attention.cpp over the
stand-in of the HIP runtime (tests/native/operators_driver.cpp), under
ThreadSanitizer."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
NATIVE = os.path.join(HERE, "native")
CSRC = os.path.join(HERE, "..", "sym_amd", "csrc")
SHARED = ["plan", "program", "runtime", "workers", "indexed", "transfer", "capi", "hip_fake"]  # that the Makefile builds


@pytest.fixture(scope="module")
def results(tmp_path_factory):
    if shutil.which("g++") is None or not os.path.isdir("/opt/rocm/include/hip"):
        pytest.skip("g++ or the HIP headers are missing")
    exe = str(tmp_path_factory.mktemp("operators") / "operators_driver")
    subprocess.run(["make", "-s", "-j8", "-C", NATIVE], check=True, capture_output=True)
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=thread", "-pthread", "-D__HIP_PLATFORM_AMD__",
                    "-I/opt/rocm/include", "-I" + CSRC, "-I" + NATIVE, "-o", exe, os.path.join(NATIVE, "operators_driver.cpp"),
                    os.path.join(CSRC, "attention.cpp")] +
                   [os.path.join(NATIVE, "_build", o + ".o") for o in SHARED] + ["-ldl"], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=100,
                       env=dict(os.environ, TSAN_OPTIONS="halt_on_error=0 exitcode=66 report_signal_unsafe=0"))
    assert r.returncode == 0 and "ThreadSanitizer" not in r.stderr, r.stdout + r.stderr[-4000:]
    return dict(line.split(": ", 1) for line in r.stdout.splitlines())


def test_calls_do_not_wait_for_transfers(results):
    """A transfer holds its context until the GPU has done it; the operators take
    nothing of the context that it uses."""
    assert results["tables"] == results["tables beside a transfer"] == "ok" and results["launches"] == "2"


def test_a_quarantined_context_takes_no_calls(results):
    assert results["tables of a quarantined context"] == "resources_closed"
