"""GPU: the ends of the range of the paged cache's calls, against plain float64
implementations on the CPU (bounds as in test_gpu_kv.py)."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_kv import BF, F32, I32, KINDS, Cache, _codes, _cu

pytestmark = pytest.mark.gpu


# -- the cache -------------------------------------------------------------------

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("counts", [[0, 5, 3], [5, 0, 3], [5, 3, 0], [0, 0, 0, 1, 0], [0, 18, 0]], ids=str)
def test_write_beside_sequences_without_new_tokens(pkg, dev, kind, counts):
    """Sequences that hold earlier positions and have no new token, before, between
    and behind others: nothing of theirs changes, the others' rows are stored.  k
    and v fill their tensors, so that there is no row before the first or behind
    the last."""
    past = [7, 21, 9, 30, 16][:len(counts)]
    print(f"[gpu] kv write beside empty counts {kind} {counts}", flush=True)
    c = Cache(pkg, dev, kind, 2, 64, 16, [n + m for n, m in zip(counts, past)], seed=201)
    g = torch.Generator().manual_seed(202)
    old = [torch.randn(sum(past), 2, 64, generator=g).to(BF) for _ in range(2)]
    new = [torch.randn(sum(counts), 2, 64, generator=g).to(BF) for _ in range(2)]
    past_t, past_cu, cu = torch.tensor(past, dtype=I32, device=dev), _cu(dev, past), _cu(dev, counts)
    pkg.kv_write(c.pages, *(t.to(dev) for t in old), c.table, past_t, past_cu)
    pkg.kv_write(c.pages, *(t.to(dev) for t in new), c.table, c.len_t, cu)

    def held(t):
        if kind == "bf16":
            return t.to(F32)
        codes, sc = _codes(t, kind)
        return codes.to(F32) * sc[..., None]

    for want, got in zip(old, pkg.kv_read(c.pages, c.table, past_t, past_cu, total=sum(past), dtype=F32)):
        assert torch.equal(got.cpu(), held(want))
    for want, got in zip(new, pkg.kv_read(c.pages, c.table, c.len_t, cu, total=sum(counts), dtype=F32)):
        assert torch.equal(got.cpu(), held(want))
