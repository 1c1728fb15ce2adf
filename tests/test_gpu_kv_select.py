"""GPU: the index of the paged cache's pages (kv_index), the choice of pages by it
(kv_select) and the attention to these alone (paged_attention with keep), against
plain implementations on the CPU.

* index: a mean's sum is exact in float64 on both sides (up to 256 numbers of 8 bits,
  or of 8 bits times a float32 scale, whose exponents lie within 2^20), so codes and
  scales equal the float32 formula's bit for bit;
* places: scores are whole numbers under 2^24 times a float32, rounded once: equal;
* attention: the bound of test_gpu_kv.py, over the kept positions."""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_kv import BAR, BF, F32, F64, I32, KINDS, Cache, _cu, _fill

pytestmark = pytest.mark.gpu
NAN = math.nan


def _codes(x):
    """(codes, scale) of float64 rows rounded to float32."""
    x = x.to(F32)
    m = x.abs().amax(-1)
    fine = (m > 2.0 ** -100) & torch.isfinite(m)
    top = torch.full_like(m, 127.0)
    c = torch.round(torch.where(fine[..., None], x * torch.where(fine, top / m, torch.zeros(()))[..., None], torch.zeros(())))
    scale = torch.where(fine, m / top, torch.zeros(()))
    return c.to(torch.int8), torch.where(torch.isfinite(m), scale, torch.full_like(m, NAN))


def _index_of(c):
    """{page: (codes, scale)} of every page of every sequence."""
    got = {}
    for b, n in enumerate(c.lens):
        k, _ = c.held(b)
        for j in range(-(-n // c.P)):
            part = k[j * c.P:min(n, (j + 1) * c.P)]
            got[c.rows[b][j]] = _codes(part.sum(0) / len(part))
    return got


def _empty_index(pkg, dev, c, fill=3):
    n = c.pages.n_pages
    return pkg.KvIndex(torch.full((n, c.H, c.dh), fill, dtype=torch.int8, device=dev), torch.full((n, c.H), float(fill), device=dev))


# -- the index -----------------------------------------------------------------------

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("P", [16, 32, 64, 128, 256])
def test_index_of_new_tokens(pkg, dev, kind, dh, P):
    """Whole sequences, then further tokens of some: entries of the pages they touch
    are the mean of what these hold by then, all others stay."""
    print(f"[gpu] kv_index {kind} {dh} {P}", flush=True)
    lens = [1, P, P + 1, 3 * P - 1, 17]
    c = Cache(pkg, dev, kind, 3, dh, P, lens, seed=P + dh)
    g = torch.Generator().manual_seed(P)
    _fill(pkg, dev, c, g)
    index = _empty_index(pkg, dev, c)
    pkg.kv_index(c.pages, index, c.table, c.len_t, _cu(dev, lens), total=sum(lens))
    want = _index_of(c)
    codes, scale = index.codes.cpu(), index.scale.cpu()
    for page in range(c.pages.n_pages):
        if page in want:
            assert torch.equal(codes[page], want[page][0]) and torch.equal(scale[page], want[page][1]), page
        else:
            assert (codes[page] == 3).all() and (scale[page] == 3).all()
    # the last 1, 0, 2, P and 17 positions alone
    index = _empty_index(pkg, dev, c)
    counts = [1, 0, 2, P, 17]
    for total in (sum(counts), None):
        pkg.kv_index(c.pages, index, c.table, c.len_t, _cu(dev, counts), total=total)
    codes = index.codes.cpu()
    touched = {c.rows[b][j] for b, n in enumerate(counts) if n for j in range((lens[b] - n) // P, (lens[b] - 1) // P + 1)}
    for page in range(c.pages.n_pages):
        assert torch.equal(codes[page], want[page][0]) if page in touched else (codes[page] == 3).all()
    # single tokens
    index = _empty_index(pkg, dev, c)
    pkg.kv_index(c.pages, index, c.table, c.len_t)
    codes = index.codes.cpu()
    touched = {c.rows[b][(n - 1) // P] for b, n in enumerate(lens)}
    for page in range(c.pages.n_pages):
        assert torch.equal(codes[page], want[page][0]) if page in touched else (codes[page] == 3).all()


@pytest.mark.parametrize("kind", KINDS)
def test_index_of_zeros_infinities_and_missing_pages(pkg, dev, kind):
    print(f"[gpu] kv_index edges {kind}", flush=True)
    P = 16
    c = Cache(pkg, dev, kind, 1, 64, P, [80], seed=4)
    k = torch.randn(80, 1, 64, generator=torch.Generator().manual_seed(1))
    k[:16] = 0
    k[16:32] = 2.0 ** -110
    k[40, 0, 5], k[50, 0, 0] = math.inf, NAN
    v = torch.ones_like(k)
    pkg.kv_write(c.pages, k.to(dev), v.to(dev), c.table, c.len_t, _cu(dev, [80]))
    index = _empty_index(pkg, dev, c)
    table = c.table.clone()
    table[0, 4] = -1
    pkg.kv_index(c.pages, index, table, c.len_t, _cu(dev, [80]))
    codes, scale = index.codes.cpu()[c.rows[0]], index.scale.cpu()[c.rows[0]]
    assert not codes[0].any() and not codes[1].any() and scale[0] == 0 and scale[1] == 0
    assert torch.isnan(scale[2]).all() and torch.isnan(scale[3]).all() and not codes[2:4].any()
    assert (codes[4] == 3).all() and scale[4] == 3
    # lengths of zero, tables without columns, entries that name no page
    for lens, cu in (([0], [0, 1]), ([-5], [0, 3]), ([10 ** 9], [0, 5])):
        pkg.kv_index(c.pages, index, table, torch.tensor(lens, dtype=I32, device=dev), torch.tensor(cu, dtype=I32, device=dev))
    pkg.kv_index(c.pages, index, table[:, :0], c.len_t, _cu(dev, [80]), total=80)
    pkg.kv_index(c.pages, index, torch.full_like(table, 99), c.len_t, _cu(dev, [80]))
    assert torch.equal(index.codes.cpu()[c.rows[0]], codes)


# -- the choice ----------------------------------------------------------------------

def _select(q, codes, scale, rows, lens, counts, P, n, first, last):
    """keep [T, H, n] by the definition."""
    H, dh = codes.shape[1:]
    G = q.shape[1] // H
    out, at = [], 0
    cq, _ = _codes(q.to(F64).reshape(q.shape[0], H, G, dh).sum(2))
    for b, m in enumerate(counts):
        ids = torch.tensor([r if 0 <= r < codes.shape[0] else -1 for r in rows[b]], dtype=torch.long)
        for i in range(m):
            pos = lens[b] - m + i
            own = min(pos // P, len(ids) - 1) if pos >= 0 else -1
            for h in range(H):
                dots = codes[ids, h].to(torch.int64) @ cq[at + i, h].to(torch.int64)
                score = dots.to(F32) * scale[ids, h]
                have = [j for j in range(own + 1) if ids[j] >= 0]
                ends = [j for j in have if j < first or j > own - last]
                rest = [j for j in have if j not in set(ends)]
                nan = [j for j in rest if math.isnan(score[j])]
                rest = nan + sorted((j for j in rest if j not in set(nan)), key=lambda j: (-score[j].item(), j))
                take = sorted(ends + rest[:max(0, n - len(ends))])
                out.append(take + [-1] * (n - len(take)))
        at += m
    return torch.tensor(out, dtype=I32).reshape(at, H, n)


@pytest.mark.parametrize("counts", [None, [1, 3, 0, 9, 2], [5, 4, 8, 1, 1]], ids=str)
@pytest.mark.parametrize("n,first,last", [(1, 0, 1), (4, 1, 2), (9, 2, 3), (40, 1, 1), (7, 6, 1)])
@pytest.mark.parametrize("dh,G,P", [(64, 1, 16), (128, 4, 32)])
def test_places_of_the_largest_scores(pkg, dev, counts, n, first, last, dh, G, P):
    print(f"[gpu] kv_select {counts} {n} {first} {last} {dh} {G} {P}", flush=True)
    H = 2
    lens = [11 * P + 3, 5, P, 30 * P, 2 * P + 1]
    c = Cache(pkg, dev, "bf16", H, dh, P, lens, seed=n)
    g = torch.Generator().manual_seed(dh + n)
    N = c.pages.n_pages
    codes = torch.randint(-127, 128, (N, H, dh), generator=g, dtype=torch.int8)
    scale = torch.rand(N, H, generator=g)
    codes[::7] = 0                                                   # equal scores
    scale[3::11] = 0
    scale[5::13] = NAN
    index = pkg.KvIndex(codes.to(dev), scale.to(dev))
    m = counts or [1] * 5
    T = sum(m)
    wide = torch.randn(T, H * G + 1, dh + 8, generator=g).to(BF)
    q = wide[:, 1:, 8:]                                              # strided
    q[0, 0] = 0
    table = c.table.clone()
    table[0, 4], table[3, 9] = -1, N                                 # evicted, no page
    rows = [list(r) for r in table.tolist()]
    keep = pkg.kv_select(wide.to(dev)[:, 1:, 8:], c.pages, index, table, c.len_t, None if counts is None else _cu(dev, m),
                         n=n, first=first, last=last)
    assert keep.dtype == I32 and keep.shape == (T, H, n)
    want = _select(q, codes, scale, rows, lens, m, P, n, first, last)
    assert torch.equal(keep.cpu(), want)


def test_tables_of_very_many_pages(pkg, dev):
    """More pages than a workgroup holds keys of."""
    print("[gpu] kv_select many pages", flush=True)
    H, dh, P, N = 1, 64, 16, 500
    g = torch.Generator().manual_seed(9)
    pages = pkg.KvPages(*(torch.zeros(s, dtype=BF, device=dev) for s in ((N, H, P, dh), (N, H, dh, P))))
    codes = torch.randint(-127, 128, (N, H, dh), generator=g, dtype=torch.int8)
    scale = torch.rand(N, H, generator=g)
    index = pkg.KvIndex(codes.to(dev), scale.to(dev))
    for width, counts in ((12288, None), (30001, None), (9000, [6])):
        rows = [torch.randint(0, N, (width,), generator=g).tolist()]
        table = torch.tensor(rows, dtype=I32, device=dev)
        lens = [width * P - 3]
        q = torch.randn(sum(counts or [1]), 2, dh, generator=g).to(BF)
        keep = pkg.kv_select(q.to(dev), pages, index, table, torch.tensor(lens, dtype=I32, device=dev),
                             None if counts is None else _cu(dev, counts), n=100, first=3, last=2)
        want = _select(q, codes, scale, rows, lens, counts or [1], P, 100, 3, 2)
        assert torch.equal(keep.cpu(), want)


def test_select_rows_that_no_sequence_names_and_empty_ones(pkg, dev):
    print("[gpu] kv_select rows", flush=True)
    c = Cache(pkg, dev, "int8", 2, 64, 16, [40, 3], seed=1)
    g = torch.Generator().manual_seed(1)
    _fill(pkg, dev, c, g)
    index = _empty_index(pkg, dev, c)
    q = torch.randn(9, 2, 64, generator=g).to(BF).to(dev)
    # (the outputs' memory is new: only the named rows are looked at)
    cu = torch.tensor([1, 3, 8], dtype=I32, device=dev)              # five tokens of a sequence of three
    keep = pkg.kv_select(q, c.pages, index, c.table, c.len_t, cu, n=2)
    assert keep[1:3].tolist() == [[[0, 2], [0, 2]]] * 2
    assert keep[3:8].tolist() == [[[-1, -1]] * 2] * 2 + [[[0, -1]] * 2] * 3
    none = pkg.kv_select(q[:0], c.pages, index, c.table[:0], c.len_t[:0], n=2)
    assert none.shape == (0, 2, 2)
    bare = pkg.kv_select(q[:2], c.pages, index, c.table[:, :0], c.len_t, n=3)
    assert (bare == -1).all()


# -- attention to kept pages -----------------------------------------------------------

def _attend_kept(q, k, v, keep, pos, P, scale):
    """One token: (out, sum of p |v|) [Hq, dh] over the kept pages of k, v [len, H, dh]."""
    Hq, dh = q.shape
    H = k.shape[1]
    G = Hq // H
    out, mag = torch.zeros(Hq, dh, dtype=F64), torch.zeros(Hq, dh, dtype=F64)
    for h in range(H):
        at = [j * P + s for j in keep[h] if j >= 0 for s in range(P) if j * P + s <= pos and j * P + s < len(k)]
        if at:
            kk, vv = k[at, h], v[at, h]
            p = torch.softmax(q[h * G:(h + 1) * G].to(F64) @ kk.T * scale, -1)
            out[h * G:(h + 1) * G], mag[h * G:(h + 1) * G] = p @ vv, p @ vv.abs()
    return out, mag


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dh,G,P", [(64, 1, 16), (64, 8, 64), (128, 4, 32), (128, 20, 256), (64, 3, 128)])
@pytest.mark.parametrize("counts,n", [(None, 3), (None, 60), ([4, 1, 0, 7], 5)], ids=str)
def test_attention_to_kept_pages(pkg, dev, kind, dh, G, P, counts, n):
    print(f"[gpu] kept {kind} {dh} {G} {P} {counts} {n}", flush=True)
    H = 2
    lens = [13 * P + 5, 1, P, 4 * P - 1]
    c = Cache(pkg, dev, kind, H, dh, P, lens, seed=n + dh)
    g = torch.Generator().manual_seed(dh * n)
    _fill(pkg, dev, c, g)
    m = counts or [1] * 4
    T = sum(m)
    cu = None if counts is None else _cu(dev, m)
    q = torch.randn(T, H * G, dh, generator=g).to(BF)
    index = _empty_index(pkg, dev, c)
    pkg.kv_index(c.pages, index, c.table, c.len_t, _cu(dev, lens))
    keep = pkg.kv_select(q.to(dev), c.pages, index, c.table, c.len_t, cu, n=n, first=1, last=1)
    out = pkg.paged_attention(q.to(dev), c.pages, c.table, c.len_t, cu, keep=keep).cpu().to(F64)
    at = 0
    for b, cnt in enumerate(m):
        k, v = c.held(b)
        for i in range(cnt):
            want, size = _attend_kept(q[at], k, v, keep[at].tolist(), lens[b] - cnt + i, P, dh ** -0.5)
            assert ((out[at] - want).abs() <= BAR * size).all(), (b, i)
            at += 1


def test_any_lists(pkg, dev):
    """Lists of a caller's own: unused entries anywhere, places outside the table, not
    yet there or named twice, pages that are none; a token that sees nothing gets
    zeros; rows that no sequence names stay."""
    print("[gpu] kept lists", flush=True)
    P, H, dh = 16, 1, 64
    c = Cache(pkg, dev, "int8", H, dh, P, [100, 40], seed=6)
    g = torch.Generator().manual_seed(7)
    _fill(pkg, dev, c, g)
    table = c.table.clone()
    table[0, 2] = -1
    lists = [[0, 1, 3, 3], [-1, 2, -1, 5], [-1, -1, -1, -1], [6, 6, 7, 2 ** 31 - 1], [1, 1, 1, 1], [-2 ** 31, 0, 4, 99]]
    real = [[0, 1, 3], [5], [], [6], [1], [0, 4]]
    keep = torch.tensor(lists, dtype=I32, device=dev)[:, None].contiguous()
    T = len(lists)
    q = torch.randn(T + 1, 2, dh, generator=g).to(BF)
    keep = torch.cat([keep, keep[:1]])
    cu = torch.tensor([0, T - 1, T], dtype=I32, device=dev)
    out = torch.full((T + 1, 2, dh), 5.0, dtype=BF, device=dev)
    pkg.paged_attention(q.to(dev), c.pages, table, c.len_t, cu, keep=keep, out=out)
    out = out.cpu().to(F64)
    assert (out[T] == 5).all()
    for t in range(T):
        b, pos = (0, 100 - (T - 1) + t) if t < T - 1 else (1, 39)
        k, v = c.held(b)
        want, size = _attend_kept(q[t], k, v, [real[t]], pos, P, dh ** -0.5)
        assert ((out[t] - want).abs() <= BAR * size).all(), t
    assert not out[2].any()


@pytest.mark.parametrize("kind", KINDS)
def test_long_lists_in_splits(pkg, dev, kind):
    """One token over lists of hundreds of pages: splits, joined."""
    print(f"[gpu] kept splits {kind}", flush=True)
    P, H, dh, G = 64, 2, 128, 8
    c = Cache(pkg, dev, kind, H, dh, P, [20011], seed=3)
    g = torch.Generator().manual_seed(3)
    _fill(pkg, dev, c, g)
    q = torch.randn(1, H * G, dh, generator=g).to(BF)
    k, v = c.held(0)
    for n in (313, 200, 20):
        keep = torch.stack([torch.sort(torch.randperm(313, generator=g)[:n]).values for _ in range(H)])[None].to(I32)
        out = pkg.paged_attention(q.to(dev), c.pages, c.table, c.len_t, keep=keep.to(dev)).cpu().to(F64)[0]
        want, size = _attend_kept(q[0], k, v, keep[0].tolist(), 20010, P, dh ** -0.5)
        assert ((out - want).abs() <= BAR * size).all()
        if n == 313:     # all of them: the call without lists
            dense = pkg.paged_attention(q.to(dev), c.pages, c.table, c.len_t).cpu().to(F64)[0]
            assert ((dense - out).abs() <= 2 * BAR * size).all()


def test_large_scores_infinities_and_nan(pkg, dev):
    """Rows that leave the hot loop: large scores, values that are not finite, in kept
    pages and in others (which no one sees)."""
    print("[gpu] kept odd values", flush=True)
    P, H, dh = 16, 1, 64
    c = Cache(pkg, dev, "bf16", H, dh, P, [160], seed=8)
    g = torch.Generator().manual_seed(8)
    k, v = torch.randn(160, H, dh, generator=g), torch.randn(160, H, dh, generator=g)
    k[20] *= 3000
    v[33, 0, 3], v[34, 0, 4], v[100, 0, 5] = math.inf, NAN, NAN
    pkg.kv_write(c.pages, k.to(dev), v.to(dev), c.table, c.len_t, _cu(dev, [160]))
    q = torch.randn(1, 4, dh, generator=g).to(BF)
    for lst in ([0, 1, 3], [0, 2, 4], [3, 4, 5], [0, 3, 5, 7, 9]):
        keep = torch.tensor(lst, dtype=I32, device=dev)[None, None]
        out = pkg.paged_attention(q.to(dev), c.pages, c.table, c.len_t, keep=keep).cpu().to(F64)[0]
        kk, vv = c.held(0)
        want, size = _attend_kept(q[0], kk, vv, [lst], 159, P, dh ** -0.5)
        odd = ~torch.isfinite(want)
        # (weights of exactly zero leave a NaN as in the definition or drop it: not here)
        assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out[odd & ~torch.isnan(want)], want[odd & ~torch.isnan(want)])
        assert ((out - want).abs()[~odd] <= (BAR + 2e-3) * size[~odd]).all()


def test_streams_capture_and_growing_sequences(pkg, dev):
    """A captured step (write, index, select, attend) that follows lens as they grow."""
    print("[gpu] kept capture", flush=True)
    P, H, dh, G, B = 16, 2, 64, 2, 3
    c = Cache(pkg, dev, "int8", H, dh, P, [200, 90, 17], seed=12)
    g = torch.Generator().manual_seed(12)
    _fill(pkg, dev, c, g)
    index = _empty_index(pkg, dev, c, 0)
    pkg.kv_index(c.pages, index, c.table, c.len_t, _cu(dev, c.lens))
    lens = torch.tensor([150, 60, 1], dtype=I32, device=dev)
    k, v, q = (torch.randn(B, h, dh, generator=g).to(BF).to(dev) for h in (H, H, H * G))

    def step():
        pkg.kv_write(c.pages, k, v, c.table, lens)
        pkg.kv_index(c.pages, index, c.table, lens)
        keep = pkg.kv_select(q, c.pages, index, c.table, lens, n=4, first=1, last=1)
        return keep, pkg.paged_attention(q, c.pages, c.table, lens, keep=keep)

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        lens += 1 + i
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        first = [t.clone() for t in got]
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(first, want))


def test_refusals(pkg, dev):
    c = Cache(pkg, dev, "bf16", 2, 64, 16, [40, 20], seed=1)
    N = c.pages.n_pages
    codes, scale = torch.zeros(N, 2, 64, dtype=torch.int8, device=dev), torch.zeros(N, 2, device=dev)
    index = pkg.KvIndex(codes, scale)
    q = torch.zeros(2, 4, 64, dtype=BF, device=dev)
    for err, args in ((ValueError, (codes[0], scale)), (TypeError, (codes.float(), scale)), (ValueError, (codes, scale[:1])),
                      (TypeError, (codes, scale.double())), (ValueError, (codes.cpu(), scale.cpu())),
                      (ValueError, (codes.transpose(0, 1), scale)), (TypeError, (codes, None)),
                      (NotImplementedError, (codes, scale.clone().requires_grad_()))):
        with pytest.raises(err):
            pkg.KvIndex(*args)
    small = pkg.KvIndex(codes[:1], scale[:1])
    sel = lambda **kw: pkg.kv_select(kw.pop("q", q), c.pages, kw.pop("index", index), c.table, c.len_t,  # noqa: E731
                                     **{**dict(n=4), **kw})
    for err, kw in ((ValueError, dict(n=0)), (ValueError, dict(n=2, first=2)), (ValueError, dict(last=0)),
                    (ValueError, dict(first=-1)), (TypeError, dict(n=1.5)), (ValueError, dict(index=small)),
                    (ValueError, dict(q=q[:1])), (ValueError, dict(q=q[:, :3])), (TypeError, dict(q=q.float())),
                    (NotImplementedError, dict(q=q.clone().requires_grad_()))):
        with pytest.raises(err):
            sel(**kw)
    with pytest.raises(ValueError):
        pkg.kv_index(c.pages, small, c.table, c.len_t)
    with pytest.raises(TypeError):
        pkg.kv_index(c.pages, index, c.table, c.len_t.long())
    keep = sel()
    for err, kw in ((ValueError, dict(keep=keep, window=4)), (ValueError, dict(keep=keep[:1])), (TypeError, dict(keep=keep.long())),
                    (ValueError, dict(keep=keep[..., :0])), (ValueError, dict(keep=keep[:, :1])), (ValueError, dict(keep=keep.cpu())),
                    (ValueError, dict(keep=keep[..., ::2])), (ValueError, dict(keep=[1]))):
        with pytest.raises(err):
            pkg.paged_attention(q, c.pages, c.table, c.len_t, **kw)


@pytest.mark.parametrize("counts", [None, [3]], ids=str)
@pytest.mark.parametrize("width", [90, 700, 3500])
@pytest.mark.parametrize("kind", ["zeros", "levels", "near", "infinite", "nan", "spread", "holes"])
def test_borders_among_scores_of_any_kind(pkg, dev, kind, width, counts):
    """Equal scores beyond what is counted one by one, infinities, neighbours in the last
    bit, scores of sixty orders of magnitude, pages that are missing."""
    print(f"[gpu] kv_select {kind} {width} {counts}", flush=True)
    H, dh, P, N = 1, 64, 16, 400
    g = torch.Generator().manual_seed(width + len(kind))
    pages = pkg.KvPages(*(torch.zeros(s, dtype=BF, device=dev) for s in ((N, H, P, dh), (N, H, dh, P))))
    codes = torch.randint(-127, 128, (N, H, dh), generator=g, dtype=torch.int8)
    scale = 0.5 + torch.rand(N, H, generator=g)
    rows = [torch.randint(0, N, (width,), generator=g).tolist()]
    if kind == "zeros":
        codes.zero_()
    elif kind == "levels":
        codes[:] = codes[:1]
        scale = torch.randint(1, 4, (N, H), generator=g).float()
    elif kind == "near":
        codes[:] = codes[:1]
        scale = torch.nextafter(torch.ones(N, H), torch.full((N, H), 2.0)) + torch.randint(0, 5, (N, H), generator=g) * 2.0 ** -23
    elif kind == "infinite":
        scale[::2] = math.inf
    elif kind == "nan":
        scale[torch.rand(N, H, generator=g) < 0.6] = NAN
    elif kind == "spread":
        scale = 10 ** (60 * torch.rand(N, H, generator=g, dtype=F64) - 30).float().clamp_min(1e-38)
    else:
        rows[0] = [r if j % 3 else -1 for j, r in enumerate(rows[0])]
    index = pkg.KvIndex(codes.to(dev), scale.to(dev))
    table = torch.tensor(rows, dtype=I32, device=dev)
    lens = [width * P - 2]
    q = torch.randn(sum(counts or [1]), 2, dh, generator=g).to(BF)
    for n, first, last in ((20, 1, 2), (70, 0, 1), (width // 2, 2, 3), (width - 1, 1, 1), (width + 5, 0, 1)):
        keep = pkg.kv_select(q.to(dev), pages, index, table, torch.tensor(lens, dtype=I32, device=dev),
                             None if counts is None else _cu(dev, counts), n=n, first=first, last=last)
        assert torch.equal(keep.cpu(), _select(q, codes, scale, rows, lens, counts or [1], P, n, first, last))
