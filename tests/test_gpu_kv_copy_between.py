"""GPU: kv_copy of tensors whose layers lie between each other's in one allocation."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("L,n", [(1, 6), (3, 6), (24, 40)])
def test_keys_and_values_by_layer(pkg, dev, L, n):
    print(f"[gpu] kv_copy between {L} {n}", flush=True)
    g = torch.Generator().manual_seed(L)
    kv = torch.randn(L, 2, n, 2, 16, 64, generator=g).to(torch.bfloat16).to(dev)
    want = kv.clone()
    src, dst = [0, 3, 3], [1, 4, n - 1]
    want[:, :, dst] = want[:, :, src]
    pkg.kv_copy([kv[:, 0], kv[:, 1]], src, dst)
    assert torch.equal(kv, want)
    # to the values' half of another allocation, from the keys' of this one
    other = torch.zeros_like(kv)
    pkg.kv_copy([kv[:, 0]], src, dst, to=[other[:, 1]])
    assert torch.equal(other[:, 1, dst], kv[:, 0, src]) and not other[:, 0].any() and not other[:, 1, 0].any()
    # keys onto values of the same allocation: no byte of them is shared
    pkg.kv_copy([kv[:, 0]], src, dst, to=[kv[:, 1]])
    want[:, 1, dst] = want[:, 0, src]
    assert torch.equal(kv, want)


def test_a_tensor_that_begins_within_another_is_refused(pkg, dev):
    kv = torch.zeros(3, 12, 64, device=dev)
    for n, first in ((8, 0), (8, 1), (8, 4), (5, 4)):
        with pytest.raises(ValueError):
            pkg.kv_copy([kv[:, :n], kv[:, first:first + n]], [0], [1])
    pkg.kv_copy([kv[:, :6], kv[:, 6:]], [0], [1])
