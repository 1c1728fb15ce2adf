"""GPU: kv_copy (pages copied onto other pages in all layers) and the sequences of a
PagedKvCache that branch, move and change places.  Copies are equal bit for bit."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32
FP8 = torch.float8_e4m3fn


def _bytes(t):
    return t.contiguous().view(torch.uint8).cpu()


def _random(shape, dtype, g, dev):
    n = 1
    for s in shape:
        n *= s
    size = torch.empty(0, dtype=dtype).element_size()
    return torch.randint(0, 256, (n * size,), generator=g, dtype=torch.uint8).view(dtype).reshape(shape).to(dev)


LAYOUTS = {
    "bf16": [((6, 64, 64), BF), ((6, 64, 64), BF)],
    "fp8": [((2, 16, 128), FP8), ((2, 128, 16), FP8), ((2, 16), F32), ((2, 16), F32)],
    "index": [((3, 16, 64), torch.int8), ((3, 64, 16), torch.int8), ((3, 16), F32), ((3, 16), F32), ((3, 64), torch.int8), ((3,), F32)],
    "odd": [((7, 3), F32), ((1,), I32), ((5, 4), torch.uint8)],
    "large": [((8, 256, 128), BF)],
}


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("L,n,pairs", [(1, 2, 1), (3, 40, 13), (2, 700, 300), (5, 30, 0)])
def test_pages_get_what_others_hold(pkg, dev, layout, L, n, pairs):
    print(f"[gpu] kv_copy {layout} {L} {n} {pairs}", flush=True)
    if layout == "large" and n > 100:
        n, pairs = 60, 20
    g = torch.Generator().manual_seed(n + pairs)
    t = [_random((L, n, *s), d, g, dev) for s, d in LAYOUTS[layout]]
    order = torch.randperm(n, generator=g).tolist()
    dst, rest = order[:pairs], order[pairs:]
    src = [rest[i // 2 % len(rest)] for i in range(pairs)]         # several times
    want = [_bytes(x).reshape(L, n, -1).clone() for x in t]
    for w in want:
        w[:, dst] = w[:, src]
    version = [x._version for x in t]
    pkg.kv_copy(t, src, dst)
    for x, w, v in zip(t, want, version):
        assert torch.equal(_bytes(x).reshape(L, n, -1), w)
        assert x._version == v + (1 if pairs else 0)


def test_to_other_tensors_and_of_one_layer(pkg, dev):
    print("[gpu] kv_copy to others", flush=True)
    g = torch.Generator().manual_seed(2)
    shapes = [((2, 16, 64), torch.int8), ((2, 64, 16), torch.int8), ((2, 16), F32), ((2, 16), F32)]
    a = [_random((3, 9, *s), d, g, dev) for s, d in shapes]
    b = [_random((3, 5, *s), d, g, dev) for s, d in shapes]
    want = [_bytes(x).reshape(3, 5, -1) for x in b]
    held = [_bytes(x).reshape(3, 9, -1) for x in a]
    for w, h in zip(want, held):
        w[:, [4, 0, 2]] = h[:, [0, 8, 8]]
    pkg.kv_copy(a, [0, 8, 8], range(4, -1, -2)[:0] or [4, 0, 2], to=b)
    for x, w, y, h in zip(b, want, a, held):
        assert torch.equal(_bytes(x).reshape(3, 5, -1), w) and torch.equal(_bytes(y).reshape(3, 9, -1), h)
    # one layer's pages; every second layer of a tensor
    pages = pkg.KvPages(*(x[1] for x in a))
    pkg.kv_copy(pages, [3], [4])
    for x, h in zip(a, held):
        h[1, 4] = h[1, 3]
        assert torch.equal(_bytes(x).reshape(3, 9, -1), h)
    pkg.kv_copy([x[::2] for x in a], (1,), (2,))
    for x, h in zip(a, held):
        h[::2, 2] = h[::2, 1]
        assert torch.equal(_bytes(x).reshape(3, 9, -1), h)


def test_offsets_past_32_bits(pkg, dev):
    print("[gpu] kv_copy past 4 GiB", flush=True)
    n = 36000                                     # pages of 128 KiB: 4.7 GB
    t = torch.zeros(1, n, 1 << 17, dtype=torch.uint8, device=dev)
    t[0, 5] = 7
    t[0, n - 1] = 9
    pkg.kv_copy([t], [5, n - 1], [n - 2, 6])
    assert (t[0, n - 2] == 7).all() and (t[0, 6] == 9).all() and not t[0, n - 3].any()


def test_unaligned_and_streams(pkg, dev):
    """Tensors that begin 4 bytes behind a 16-byte border; another stream; a graph."""
    print("[gpu] kv_copy alignment, streams, capture", flush=True)
    g = torch.Generator().manual_seed(4)
    flat = _random((1 + 2 * 6 * 32,), F32, g, dev)
    t = flat[1:].view(2, 6, 32)
    want = t.clone()
    want[:, 1] = want[:, 5]
    pkg.kv_copy([t], [5], [1])
    assert torch.equal(t.view(I32), want.view(I32))
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        pkg.kv_copy([t], [2], [0])
    side.synchronize()
    assert torch.equal(t[:, 0].view(I32), t[:, 2].view(I32))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.kv_copy([t], [4, 4], [3, 1])
    for seed in range(3):
        t.copy_(torch.randn(2, 6, 32, generator=torch.Generator().manual_seed(seed)))
        want = t.clone()
        want[:, 3] = want[:, 1] = want[:, 4]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(t, want)


def test_refusals(pkg, dev):
    t = torch.zeros(2, 8, 16, device=dev)
    u = torch.zeros(2, 4, 16, device=dev)
    many = torch.zeros(1, 100, 4, device=dev)
    bad = [(ValueError, ([], [], []), {}), (ValueError, ([t], [0], []), {}), (ValueError, ([t], [0], [8]), {}),
           (ValueError, ([t], [-1], [1]), {}), (ValueError, ([t], [0], [2 ** 40]), {}), (ValueError, ([t], [0, 1], [2, 2]), {}),
           (ValueError, ([t], [0, 1], [1, 2]), {}), (ValueError, ([t], [3], [3]), {}),
           (ValueError, ([many], list(range(40)), list(range(39, 79))), {}),
           (ValueError, ([many], [0] * 40, [50] + list(range(50, 89))), {}),
           (ValueError, ([t, t], [0], [1]), {}), (ValueError, ([t, u], [0], [1]), {}),
           (ValueError, ([t], [0], [1]), dict(to=[t[:, :4]])), (ValueError, ([t], [0], [1]), dict(to=[t.clone(), u])),
           (ValueError, ([t], [0], [5]), dict(to=[u])), (ValueError, ([t], [0], [1]), dict(to=[u[:1]])),
           (ValueError, ([t], [0], [1]), dict(to=[u.to(I32)])), (ValueError, ([t.cpu()], [0], [1]), {}),
           (ValueError, ([t.transpose(1, 2)], [0], [1]), {}), (ValueError, ([t[..., 0]], [0], [1]), {}),
           (ValueError, ([t.to(torch.uint8)[..., :3].contiguous()], [0], [1]), {}), (ValueError, ([t[0]], [0], [1]), dict(to=[u[0, 0]])),
           (ValueError, ([t[:1].expand(2, -1, -1)], [0], [1]), {}), (ValueError, ([t[:, :0]], [0], [1]), {}),
           (TypeError, ([t], [0.5], [1]), {}), (TypeError, ([t], torch.tensor([0], device=dev), [1]), {}),
           (ValueError, ([t] * 9, [0], [1]), {}), (NotImplementedError, ([t.clone().requires_grad_()], [0], [1]), {})]
    before = t.clone()
    for i, (err, args, kw) in enumerate(bad):
        with pytest.raises(err):
            pkg.kv_copy(*args, **kw)
            print("not refused:", i, flush=True)
    assert torch.equal(t, before)


# -- sequences ---------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, torch.int8], ids=["bf16", "int8"])
def test_forked_sequences_go_their_own_ways(pkg, dev, dtype):
    """Sequences that branch at every kind of place, write, free, move and change
    tensors; what each holds is what was written into it."""
    print(f"[gpu] forks {dtype}", flush=True)
    H, dh, P = 2, 64, 16
    cache = pkg.PagedKvCache(2, 40, H, dh, page_size=P, dtype=dtype, indexed=dtype != BF)
    g = torch.Generator().manual_seed(1)
    held = {}

    def write(seqs, counts):
        table, lens, cu, most = cache.extend(seqs, counts)
        k = torch.randint(-127, 128, (sum(counts), H, dh), generator=g).float()
        k[..., 0] = 127.0                          # codes of these numbers are they themselves
        for layer in range(2):
            pkg.kv_write(cache.layer(layer), (k + 0).to(dev), (k * (layer + 1)).to(dev), table, lens, cu)
        at = 0
        for s, n in zip(seqs, counts):
            held[s] = torch.cat([held.get(s, k[:0]), k[at:at + n]])
            at += n

    def check():
        table, lens, cu, _ = cache.extend(list(held), [0] * len(held))
        everything = torch.tensor([0] + [len(x) for x in held.values()]).cumsum(0).to(I32).to(dev)
        for layer in range(2):
            k, v = pkg.kv_read(cache.layer(layer), table, lens, everything, total=sum(map(len, held.values())), dtype=F32)
            want = torch.cat(list(held.values()))
            assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), (want * (layer + 1)))

    def fork(s):
        new = cache.fork(s)
        held[new] = held[s]
        return new

    a = cache.add()
    write([a], [37])
    used = 40 - cache.free_pages
    b, c = fork(a), fork(a)
    assert 40 - cache.free_pages == used
    check()
    write([b, a, c], [1, 2, 0])                    # b's and a's last page are copied, c keeps the old one
    assert 40 - cache.free_pages == used + 2
    check()
    write([c], [1])                                # c's alone by now: no copy
    assert 40 - cache.free_pages == used + 2
    write([a, b], [9, 10])                         # up to and over the page's end
    check()
    d = fork(b)                                    # at a page's end: nothing to copy
    assert len(held[b]) % P == 0
    before = cache.free_pages
    write([d], [3])
    assert cache.free_pages == before - 1
    check()
    cache.free(a)
    del held[a]
    check()
    moved = cache.compact()
    top = max(p for pages in cache._pages.values() for p in pages)
    assert top == 40 - cache.free_pages - 1 and moved >= 0
    check()
    write([b, c, d], [5, 20, 14])
    cache.resize(64)
    assert cache.n_pages == cache.k.shape[1] == 64
    check()
    write([b, c, d], [30, 1, 2])
    cache.resize(64 - cache.free_pages)
    assert cache.free_pages == 0
    check()
    with pytest.raises(MemoryError):
        cache.resize(3)
    e = fork(c)
    with pytest.raises(MemoryError):               # no page for the copy
        write([e], [1])
    del held[e]
    cache.free(e)
    check()
    for s in list(held):
        cache.free(s)
    assert cache.free_pages == cache.n_pages and not cache._more
