"""GPU: attention to kept pages gives the same bits in every run, whatever its workspace
and output held before, in one and in several splits."""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_kv import BF, KINDS, Cache, _fill

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens,n", [([9000], 30), ([9000, 700, 20, 5000], 60), ([400] * 40, 12)], ids=["deep", "splits", "whole"])
def test_the_same_bits_every_time(pkg, dev, kind, lens, n):
    print(f"[gpu] kept attention again {kind} {lens[:4]} {n}", flush=True)
    H, dh, P, G = 2, 128, 64, 8
    c = Cache(pkg, dev, kind, H, dh, P, lens, seed=n)
    g = torch.Generator().manual_seed(n)
    _fill(pkg, dev, c, g)
    B = len(lens)
    q = torch.randn(B, H * G, dh, generator=g).to(BF).to(dev)
    keep = torch.full((B, H, n), -1, dtype=torch.int32)
    for b, t in enumerate(lens):
        pages = -(-t // P)
        for h in range(H):
            some = torch.randperm(pages, generator=g)[:n].sort().values
            keep[b, h, :len(some)] = some.to(torch.int32)
    keep = keep.to(dev)
    first = None
    for fill in (0.0, math.nan, 1e30, -math.inf):
        held = [torch.full((1 << k,), fill, device=dev) for k in range(6, 22) for _ in range(3)]
        del held                                  # (what workspaces and outputs will hold)
        out = pkg.paged_attention(q, c.pages, c.table, c.len_t, keep=keep)
        given = torch.full_like(out, fill)
        pkg.paged_attention(q, c.pages, c.table, c.len_t, keep=keep, out=given)
        first = out.clone() if first is None else first
        assert torch.equal(out, first) and torch.equal(given, first)
    assert torch.isfinite(first).all()
