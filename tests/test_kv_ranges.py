"""CPU: the index arithmetic of the paged cache's kernels, which host and device
share (csrc/srw_kv.hpp), in a program of its own (tests/kv_ranges/): what a call
reads and writes stays inside its arrays, whatever its lengths."""

from __future__ import annotations

import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
HIPCC = "/opt/rocm/bin/hipcc"


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if not os.path.exists(HIPCC) or shutil.which("g++") is None:
        pytest.skip("needs hipcc")
    exe = tmp_path_factory.mktemp("kv_ranges") / "kv_ranges"
    root = os.path.dirname(HERE)
    build = subprocess.run([HIPCC, "--offload-host-only", "-O1", "-std=c++17",
                            "-Xarch_host", "-fsanitize=undefined", "-Xarch_host", "-fno-sanitize-recover=all", "-Wall", "-Wno-unused-function",
                            "-I", os.path.join(root, "include"), "-I", os.path.join(root, "dawn-srw_amd", "csrc"),
                            os.path.join(HERE, "kv_ranges", "kv_ranges.hip"), "-o", str(exe)],
                           capture_output=True, text=True)
    assert build.returncode == 0, build.stderr[-3000:]
    return str(exe)


def _run(program, what):
    got = subprocess.run([program, what], capture_output=True, text=True, timeout=120)
    assert got.returncode == 0, got.stdout[-3000:] + got.stderr[-1000:]
    assert " 0 failures" in got.stdout


def test_rows_of_units_are_rows_of_the_call(program):
    """kv_write loads, for 16 positions, rows of their own sequence's new tokens
    only: none of a sequence without new tokens, whose neighbours' rows may end
    or begin the tensor."""
    _run(program, "rows")


def test_spans_hold_what_rows_see(program):
    """Tiles and keys of rows against the definition, with windows and first tokens
    up to 2^31 - 1 and rows before the first position."""
    _run(program, "spans")


@pytest.mark.skipif(shutil.which("make") is None or not os.path.exists(HIPCC), reason="needs make and hipcc")
def test_entry_points_clean_under_asan_ubsan():
    """Descriptions, workspace sizes and refusals over the whole range of a call's
    fields (tests/kv_ranges/kv_sanitize.c)."""
    folder = os.path.join(HERE, "kv_ranges")
    build = subprocess.run(["make", "-C", folder, "-j4"], capture_output=True, text=True)
    assert build.returncode == 0, build.stdout[-2000:] + build.stderr[-2000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:abort_on_error=1:verify_asan_link_order=0",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    run = subprocess.run([os.path.join(folder, "_build", "kv_sanitize")], capture_output=True, text=True, env=env,
                         timeout=300)
    out = run.stdout + run.stderr
    assert run.returncode == 0 and " 0 failures" in out, out[-4000:]
    assert "runtime error" not in out and "AddressSanitizer" not in out
