"""What caches of pages ask of the host and of a launch, on the CPU from the library's own source."""
import atexit
import functools
import os
import shutil
import subprocess
import tempfile

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@functools.lru_cache(maxsize=None)
def _program():
    """The check program's path: the host side from its source, the kernel tables from the built library."""
    hipcc = "/opt/rocm/bin/hipcc" if os.path.exists("/opt/rocm/bin/hipcc") else shutil.which("hipcc")
    if not hipcc:
        pytest.skip("hipcc not found")
    from leap_amd.attention import load_library
    load_library()
    lib = os.path.join(ROOT, "leap_amd")
    tmp = tempfile.mkdtemp()
    atexit.register(shutil.rmtree, tmp, ignore_errors=True)
    exe = os.path.join(tmp, "pages_rules_check")
    r = subprocess.run([hipcc, "-x", "hip", "--offload-arch=gfx950", "-O2", "-std=c++17", "-Xclang", "-target-feature",
                        "-Xclang", "-packed-fp32-ops", "-I", os.path.join(ROOT, "leap_amd", "csrc"), "-I",
                        os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "pages_rules_check.cpp"), "-o", exe,
                        "-L", lib, "-lleap_hip_attention", f"-Wl,-rpath,{lib}"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return exe


def test_every_launch_covers_its_work_inside_its_workspace():
    r = subprocess.run([_program(), "launches"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


def test_tables_change_without_memory_and_a_full_pool_has_its_own_code():
    r = subprocess.run([_program(), "memory"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
