"""CPU: the whole-number arithmetic of sampling that host and device share
(csrc/srw_sample.hpp), in a program of its own (tests/sample_ranges/) whose undefined
behaviour ends it."""

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
    exe = tmp_path_factory.mktemp("sample_ranges") / "sample_ranges"
    root = os.path.dirname(HERE)
    build = subprocess.run([HIPCC, "--offload-host-only", "-O1", "-std=c++17",
                            "-Xarch_host", "-fsanitize=undefined", "-Xarch_host", "-fno-sanitize-recover=all", "-Wall", "-Wno-unused-function",
                            "-I", os.path.join(root, "include"), "-I", os.path.join(root, "dawn-srw_amd", "csrc"),
                            os.path.join(HERE, "sample_ranges", "sample_ranges.hip"), "-o", str(exe)],
                           capture_output=True, text=True)
    assert build.returncode == 0, build.stderr[-3000:]
    return str(exe)


def _run(program, what):
    got = subprocess.run([program, what], capture_output=True, text=True, timeout=120)
    assert got.returncode == 0, got.stdout[-3000:] + got.stderr[-1000:]
    assert " 0 failures" in got.stdout and not got.stdout.startswith("0 checks")


def test_shares_of_a_sum_are_exact(program):
    """u and p times sums of up to 62 bits, against 128 bits."""
    _run(program, "shares")


def test_the_largest_float_under_a_number(program):
    """Of numbers that round to a zero of either sign too."""
    _run(program, "unders")


def test_octaves_of_any_temperature(program):
    """Where a logit lies under the largest, for logits over temperatures up to 2^30."""
    _run(program, "octaves")
