"""What prompts, trees and 8-bit steps are cut into, on the CPU from the
library's own source: kernels and workspace for every call, and the host-pointer
calls' checks."""
import atexit
import functools
import os
import shutil
import subprocess
import tempfile
from collections import namedtuple

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# rows of a tile (16 or 256), whether one launch stores and attends, chunks of the longest sequence, spread over the XCDs
Plan = namedtuple("Plan", "rows fused splits spread")


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
    exe = os.path.join(tmp, "many_rules_check")
    r = subprocess.run([hipcc, "-x", "hip", "--offload-arch=gfx950", "-O2", "-std=c++17", "-Xclang", "-target-feature",
                        "-Xclang", "-packed-fp32-ops", "-I", os.path.join(ROOT, "leap_amd", "csrc"), "-I",
                        os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "many_rules_check.cpp"), "-o", exe,
                        "-L", lib, "-lleap_hip_attention", f"-Wl,-rpath,{lib}"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return exe


@functools.lru_cache(maxsize=None)
def plan(nh, nkv, hd, cache, lens, pos, step=False):
    """The Plan of a call over sequences of `lens` new tokens after `pos` cached rows."""
    most = max(lens)
    last = max(p + n - 1 for n, p in zip(lens, pos) if n)
    line = [nh, nkv, hd, int(cache == "q8"), int(step), len(lens), sum(lens), most, last]
    r = subprocess.run([_program(), "plan"], input=" ".join(map(str, line)), capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    rows, fused, splits, spread = map(int, r.stdout.split())
    return Plan(rows, bool(fused), splits, bool(spread))


def test_every_call_has_kernels_and_workspace():
    r = subprocess.run([_program()], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


# Calls on either side of the lines between tiles of 16 and of 256 rows, one
# launch and two, one chunk and more: each side as it measured faster.
@pytest.mark.parametrize("nh,nkv,hd,cache,lens,pos,rows,fused", [
    (32, 8, 128, "f32", (64,), (0,), 16, False),
    (32, 8, 128, "f32", (64,), (4032,), 256, True),
    (32, 8, 128, "f32", (16,) * 8, (1008,) * 8, 16, True),
    (32, 8, 128, "f32", (8,), (0,), 16, True),
    (32, 4, 64, "f32", (16,) * 32, (496,) * 32, 16, False),
    (32, 8, 128, "q8", (100,), (3996,), 16, False),
    (32, 8, 128, "q8", (32,) * 32, (480,) * 32, 256, False),
    (32, 4, 64, "q8", (64,) * 32, (448,) * 32, 256, False),
    (32, 8, 128, "f32", (8192,), (0,), 256, False),
])
def test_calls_take_the_side_that_measured_faster(nh, nkv, hd, cache, lens, pos, rows, fused):
    p = plan(nh, nkv, hd, cache, lens, pos)
    assert (p.rows, p.fused) == (rows, fused), p


def test_begins_that_go_backwards_are_refused_before_any_parent_is_read():
    r = subprocess.run([_program(), "refuse"], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
