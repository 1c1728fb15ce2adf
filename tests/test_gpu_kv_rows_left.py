"""GPU: rows of paged_attention's out that no sequence names (cu's last entry below
T, its first above 0) keep what they hold, in calls whose positions are split and
joined too.  The named rows against float64, bound as in test_gpu_kv.py."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_kv import BAR, BF, F64, I32, Cache, _attend64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("past,n", [(100, 3), (9000, 3), (9000, 40)], ids=["whole", "split", "split_many_rows"])
def test_rows_that_no_sequence_names(pkg, dev, past, n):
    print(f"[gpu] rows left {past} {n}", flush=True)
    H, dh = 2, 64
    g = torch.Generator().manual_seed(past + n)
    c = Cache(pkg, dev, "bf16", H, dh, 64, [past + n], seed=31)
    k, v = (torch.randn(past + n, H, dh, generator=g).to(BF) for _ in range(2))
    pkg.kv_write(c.pages, k.to(dev), v.to(dev), c.table, c.len_t, torch.tensor([0, past + n], dtype=I32, device=dev))
    T = n + 5
    q = torch.randn(T, 2 * H, dh, generator=g).to(BF)
    for first in (0, 2):
        cu = torch.tensor([first, first + n], dtype=I32, device=dev)
        out = torch.full((T, 2 * H, dh), 7.0, dtype=BF, device=dev)
        pkg.paged_attention(q.to(dev), c.pages, c.table, c.len_t, cu, max_new=n, out=out)
        out = out.cpu()
        assert (out[:first] == 7).all() and (out[first + n:] == 7).all()
        want, size = _attend64(q[first:first + n].to(F64), k.to(F64), v.to(F64), past, dh ** -0.5, 0, 0)
        assert ((out[first:first + n].to(F64) - want).abs() <= BAR * size).all()
