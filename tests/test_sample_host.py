"""CPU: sampling's workspaces and the numbers its calls are described by."""

from __future__ import annotations

import ctypes

import pytest

from tests.test_serving_host import _sample


@pytest.fixture(scope="module")
def C(pkg):
    from dawn_srw_amd import _capi
    _capi.load_library()
    return _capi


@pytest.mark.parametrize("top_k", ["none", "array", "number", "all"])
@pytest.mark.parametrize("top_p", [1.0, 0.9])
@pytest.mark.parametrize("V", [1024, 1025, 2048, 2049, 8192, 8193])
def test_workspaces_of_sampling(C, V, top_p, top_k):
    """Rows are their own lists up to 2 048 logits, or 1 024 where there may be a top-k;
    longer ones have a number and a sum for each run of 8 192, and for top-p 512 running
    sums, wherever they begin."""
    lib, n = C.load_library(), ctypes.c_size_t(7)
    kw = {"none": {}, "array": dict(top_k=4096), "number": dict(top_k_all=50), "all": dict(top_k_all=V)}[top_k]
    own = V <= (2048 if top_k == "none" else 1024)
    runs = 3 * -(-V // 8192)
    al = lambda b: (b + 255) // 256 * 256  # noqa: E731
    want = 0 if own or top_k == "number" else al(al(4 * runs) + 8 * runs) + (4096 * runs if top_p < 1 else 0)
    for at, stride in ((4096, V), (4100, V + 1), (4108, V + 7)):
        d = _sample(C, B=3, V=V, row_stride=stride, logits=at, top_p_all=top_p, **kw)
        assert lib.srw_sample_workspace_size(ctypes.byref(d), ctypes.byref(n)) == C.SRW_OK and n.value == want
        if want:
            assert lib.srw_sample(ctypes.byref(d), None, 0, None) == C.SRW_EWORKSPACE
