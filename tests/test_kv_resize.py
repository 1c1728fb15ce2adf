"""PagedKvCache.resize on another stream than the one its tensors were allocated on: they
are not given out again before the copy has read them."""

from __future__ import annotations

import pytest
import torch


def test_the_copys_stream_is_recorded(pkg, monkeypatch):
    """CPU: every old tensor, behind the copy and before it is dropped."""
    from dawn_srw_amd import kv
    log = []

    class Old:
        is_cuda, device = True, "the device"

        def record_stream(self, stream):
            log.append((self, stream))

    cache = pkg.PagedKvCache(1, 4, 1, 64, page_size=16, device="cpu")
    old = [Old(), Old()]
    cache._tensors = lambda: old
    monkeypatch.setattr(kv, "kv_copy", lambda tensors, src, dst, to: log.append("copy"))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: ("stream of", device))
    cache.resize(9)
    assert log == ["copy"] + [(t, ("stream of", "the device")) for t in old] and cache.n_pages == 9


@pytest.mark.gpu
def test_memory_of_old_tensors_waits_for_the_copy(pkg, dev):
    print("[gpu] resize streams", flush=True)
    a, b = torch.cuda.Stream(dev), torch.cuda.Stream(dev)
    n = 64
    with torch.cuda.stream(a):
        cache = pkg.PagedKvCache(2, n, 2, 64, page_size=64, device=dev)
        seq = cache.add()
        cache.extend([seq], [64 * n])
        g = torch.Generator().manual_seed(1)
        cache.k.copy_(torch.randn(cache.k.shape, generator=g))
        cache.v.copy_(torch.randn(cache.v.shape, generator=g))
        pages, want = list(cache._pages[seq]), (cache.k.cpu(), cache.v.cpu())
    torch.cuda.synchronize()
    shape = tuple(cache.k.shape)
    with torch.cuda.stream(b):
        torch.cuda._sleep(200_000_000)      # (some 100 ms: the copy stays behind it)
        cache.resize(n + 3)
    with torch.cuda.stream(a):              # what the allocator would give out
        other = [torch.full(shape, 7.0, dtype=torch.bfloat16, device=dev) for _ in range(4)]
    torch.cuda.synchronize()
    at = cache._pages[seq]
    assert torch.equal(cache.k[:, at].cpu(), want[0][:, pages]) and torch.equal(cache.v[:, at].cpu(), want[1][:, pages])
    assert all((t == 7).all() for t in other)
