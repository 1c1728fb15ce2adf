"""CPU: which tensors kv_copy takes together: their layers may lie between each other's,
and share no byte (csrc/srw_kv.hpp in a program of its own, tests/kv_blocks/)."""

from __future__ import annotations

import ctypes
import os
import shutil
import subprocess

import pytest

from tests.test_serving_host import _copy

HERE = os.path.dirname(os.path.abspath(__file__))
HIPCC = "/opt/rocm/bin/hipcc"


@pytest.mark.skipif(not os.path.exists(HIPCC) or shutil.which("g++") is None, reason="needs hipcc")
def test_blocks_meet_where_they_share_a_byte(tmp_path):
    exe, root = tmp_path / "kv_blocks", os.path.dirname(HERE)
    build = subprocess.run([HIPCC, "--offload-host-only", "-O1", "-std=c++17",
                            "-Xarch_host", "-fsanitize=undefined", "-Xarch_host", "-fno-sanitize-recover=all", "-Wall", "-Wno-unused-function",
                            "-I", os.path.join(root, "include"), "-I", os.path.join(root, "dawn-srw_amd", "csrc"),
                            os.path.join(HERE, "kv_blocks", "kv_blocks.hip"), "-o", str(exe)], capture_output=True, text=True)
    assert build.returncode == 0, build.stderr[-3000:]
    got = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert got.returncode == 0 and " 0 failures" in got.stdout, got.stdout[-3000:] + got.stderr[-1000:]


LAYER = 100 * 64 + 100 * 4      # both tensors' pages of a layer, one behind the other


@pytest.mark.parametrize("change", [
    dict(dst=[1 << 20, (1 << 20) + 6396], src=[1 << 20, (1 << 20) + 6396], src_layer_stride=[LAYER] * 2, dst_layer_stride=[LAYER] * 2),
    dict(dst=[1 << 20, (1 << 20) + 6400], src=[1 << 20, (1 << 20) + 6400], src_layer_stride=[LAYER - 4] * 2, dst_layer_stride=[LAYER - 4] * 2),
    dict(dst=[1 << 20, (1 << 20) + 6400 + 2 * LAYER], src=[1 << 20, (1 << 20) + 6400], src_layer_stride=[LAYER] * 2,
         dst_layer_stride=[LAYER] * 2, n_layers=3),
], ids=["first", "next", "other"])
def test_layers_that_share_bytes_are_refused(pkg, change):
    from dawn_srw_amd import _capi as C
    c, keep = _copy(C, **change)
    assert C.load_library().srw_kv_copy(ctypes.byref(c), None) == C.SRW_EINVAL
