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


def test_results_that_share_elements_are_refused(results):
    """A result in which several rows or heads lie at one place would be written by
    several threads; any other strides are taken."""
    assert results["results of any strides that are judged otherwise than by brute force"] == "0"
    for what in ("append", "append, head-major", "append, pages inside slots", "attend"):
        assert results[what] == "ok", what
    for what in ("append, one page twice", "append, slots that share elements", "append, heads that share elements",
                 "attend, one row for all", "attend, one head for all"):
        assert results[what] == "invalid_argument", what


def test_sizes_that_no_launch_holds_are_refused(results):
    """Rather than launched, which fails and leaves its error to the next call."""
    for what in ("65534 blocks of heads", "65535 blocks of heads and values", "2^23 - 2 requests"):
        assert results[what] == "ok", what
    for what in ("65536 blocks of heads", "65538 blocks of heads and values", "2^23 - 1 requests"):
        assert results[what] == "unsupported_layout", what


def test_workspace_sizes_while_others_clear_them(monkeypatch):
    """Every size of the backward's workspace is found, also where it is cleared
    between a thread's look and its answer."""
    torch = pytest.importorskip("torch")
    from sym_amd import _native as N
    from sym_amd import attention as A

    class Cleared(dict):
        """As if another thread cleared it between any two steps of this one."""
        def _clear(self):
            dict.clear(self)

        def __contains__(self, key):
            found = dict.__contains__(self, key)
            self._clear()
            return found

        def __setitem__(self, key, value):
            dict.__setitem__(self, key, value)
            self._clear()

        def __len__(self):
            n = dict.__len__(self)
            self._clear()
            return n

        def get(self, key, default=None):
            value = dict.get(self, key, default)
            self._clear()
            return value

    monkeypatch.setattr(A, "_rooms", Cleared())
    positions = (N.ctypes.c_int32 * 4)()
    rot = A._ROTATION.pack(N.ctypes.addressof(positions), 0, 0, 0, 0, 0, 32, 4, 6, 2, 64, 0, 0, 0, 0, 16, 1e-6)
    sizes = [A._rotate_room(rot, torch.Size((4, 6, 64)), torch.Size((4, 2, 64)), torch.float16) for _ in range(3)]
    assert sizes[0] > 0 and len(set(sizes)) == 1


def test_a_workspace_holds_what_the_workgroups_leave():
    """Two parts a workgroup of an item's rows, each a sum of the head's width, a
    maximum and a sum of weights, and the schedule: 256 workgroups at 256 rows, 512
    below."""
    pytest.importorskip("torch")
    from sym_amd import attention as A
    for rows, item, groups in ((1, 16, 512), (16, 64, 512), (32, 128, 512), (64, 256, 256), (500, 256, 256)):
        for dim, width in ((64, 64), (72, 128), (128, 128)):
            want = groups * 2 * item * (width + 2) * 4 + 8 * 3
            assert A.tree_attention_workspace(2 * rows, 2, 32, 8, dim, 16) == want, (rows, dim)
    assert A.tree_attention_workspace(1000, 2, 32, 8, 256, 16) == 512 * 2 * 64 * 258 * 4 + 8 * 3


@pytest.mark.parametrize("heads,kv,dim", [(32, 8, 128), (8, 8, 64), (16, 1, 256)])
def test_a_workspace_for_steps_of_several_sizes(heads, kv, dim):
    """All rows in one request and eight bytes a request are enough for any smaller
    step; the size of the largest step itself is not, but where its rows of a request
    are already those of the largest item (64 in 16 heads of 256)."""
    pytest.importorskip("torch")
    from sym_amd import attention as A
    rows, requests = 256, 64
    kept = A.tree_attention_workspace(rows, 1, heads, kv, dim, 16) + 8 * requests
    sizes = {(r, b): A.tree_attention_workspace(r, b, heads, kv, dim, 16) for r in range(0, rows + 1, 3) for b in range(0, requests + 1, 3)}
    assert max(sizes.values()) <= kept
    assert (max(sizes.values()) > A.tree_attention_workspace(rows, requests, heads, kv, dim, 16)) == (dim < 256)
