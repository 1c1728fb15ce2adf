"""CPU: sampling's workspaces and the numbers its calls are described by."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

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


def test_temperatures_past_float32_are_infinite(pkg):
    """As a tensor's would be: every token alike."""
    from dawn_srw_amd import sampling
    for x in (1e39, 10 ** 40, 1.7e308, math.inf):
        at, number = sampling._parameter("temperature", x, torch.device("cpu"), torch.float32, 1)
        assert (at, number) == (0, math.inf)
    assert sampling._parameter("temperature", 3.4028234e38, torch.device("cpu"), torch.float32, 1) == (0, 3.4028234e38)


@pytest.mark.gpu
def test_rows_at_such_temperatures(pkg, dev):
    print("[gpu] sample hot", flush=True)
    logits = torch.randn(3, 700, generator=torch.Generator().manual_seed(1)).to(dev)
    u = torch.tensor([0.1, 0.5, 0.9], device=dev)
    want = pkg.sample(logits, u, temperature=math.inf)
    for x in (1e39, 10 ** 40):
        got = pkg.sample(logits, u, temperature=x)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert want[0].tolist() == [70, 350, 629]     # (float32 0.9 lies under 0.9, 0.1 over 0.1)
