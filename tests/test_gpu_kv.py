"""GPU: the paged key/value cache (kv_write, kv_read) and paged_attention
against plain implementations in float64 on the CPU.

Bounds, from the formats and the sums alone:

* written codes equal the float32 formula's (x * (top / m), to the nearest) bit
  for bit, so what is read back is within half a step of the source: m / 254 a
  value in int8; in fp8 2^-4 of the value, or 2^-10 of m / 448 below the normal
  range.  float32's own roundings add less than 1e-6 of m.
* attention: the weights are rounded to bf16 (8 significant bits, to the
  nearest: 2^-8 of each at most), the output again (2^-8); the scores' float32
  sums of up to 128 products move a weight by less than 2e-4 of itself at these
  inputs.  So |error| <= (2^-7 + 2^-16 + 3e-4) sum_j p_j |v_j| for every element."""

from __future__ import annotations

import ctypes
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
KINDS = {"bf16": BF, "int8": torch.int8, "fp8": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "fp8": 448.0}
BAR = 2.0 ** -7 + 2.0 ** -16 + 3e-4


class Cache:
    """Pages whose every slot starts as NaN (or as codes under NaN scales),
    page ids in a shuffled order, tables with unused entries of -1."""

    def __init__(self, pkg, dev, kind, H, dh, P, lens, spare=2, seed=0):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // P) for n in lens]
        n_pages = sum(need) + spare
        self.kind, self.H, self.dh, self.P, self.lens = kind, H, dh, P, list(lens)
        dt = KINDS[kind]
        if kind == "int8":
            k, v = (torch.randint(-128, 128, s, generator=g, dtype=torch.int8)
                    for s in ((n_pages, H, P, dh), (n_pages, H, dh, P)))
        else:
            k, v = (torch.full(s, float("nan")).to(dt) for s in ((n_pages, H, P, dh), (n_pages, H, dh, P)))
        sc = [None, None] if kind == "bf16" else [torch.full((n_pages, H, P), float("nan")) for _ in range(2)]
        self.pages = pkg.KvPages(*(t if t is None else t.to(dev) for t in (k, v, *sc)))
        order = torch.randperm(n_pages, generator=g).tolist()
        width = max(need + [1])
        rows, at = [], 0
        for n in need:
            rows.append(order[at:at + n] + [-1] * (width - n))
            at += n
        self.rows = rows
        self.table = torch.tensor(rows, dtype=I32, device=dev)
        self.len_t = torch.tensor(lens, dtype=I32, device=dev)

    def held(self, b):
        """(k, v) [lens[b], H, dh] float64 from the pages themselves."""
        p, n = self.pages, self.lens[b]
        ids = torch.tensor(self.rows[b][:-(-n // self.P)], dtype=torch.long)
        k, v = (_values(t).cpu()[ids] for t in (p.k, p.v))
        v = v.transpose(-1, -2)
        if self.kind != "bf16":
            k = k * p.k_scale.cpu().to(F64)[ids][..., None]
            v = v * p.v_scale.cpu().to(F64)[ids][..., None]
        return tuple(t.transpose(1, 2).reshape(-1, self.H, self.dh)[:n] for t in (k, v))


def _values(t):
    return t.to(F32).to(F64) if t.dtype != torch.float8_e4m3fn else t.cpu().to(F32).to(F64)


def _cu(dev, counts):
    return torch.tensor([0] + list(itertools.accumulate(counts)), dtype=I32, device=dev)


def _attend64(q, k, v, first, scale, window, sinks, seen=None):
    """(out, sum of p |v|) [n, Hq, dh] of rows at positions first ...; seen
    [len]: positions that have a page."""
    n, Hq, dh = q.shape
    G = Hq // k.shape[1]
    pos = torch.arange(n)[:, None] + first
    key = torch.arange(k.shape[0])[None]
    see = key <= pos
    if window:
        see &= (key > pos - window) | (key < sinks)
    if seen is not None:
        see &= seen[None]
    out, mag = torch.zeros(n, Hq, dh, dtype=F64), torch.zeros(n, Hq, dh, dtype=F64)
    for h in range(Hq):
        kk, vv = k[:, h // G], v[:, h // G]
        s = (q[:, h].to(F64) @ torch.nan_to_num(kk).T * scale).masked_fill(~see, -math.inf)
        any_ = see.any(1, keepdim=True)
        p = torch.where(any_, torch.softmax(s.masked_fill(~any_, 0.0), -1), torch.zeros((), dtype=F64))
        p = torch.where(see, p, torch.zeros((), dtype=F64))
        vv = torch.where(see.any(0)[:, None], vv, torch.zeros((), dtype=F64))
        out[:, h], mag[:, h] = p @ vv, p @ vv.abs()
    return out, mag


def _fill(pkg, dev, c, g, src=BF):
    """Every position of every sequence written in one call; the sources."""
    T = sum(c.lens)
    k, v = (torch.randn(T, c.H, c.dh, generator=g) * torch.exp(0.5 * torch.randn(T, c.H, 1, generator=g)) for _ in range(2))
    k, v = k.to(src), v.to(src)
    pkg.kv_write(c.pages, k.to(dev), v.to(dev), c.table, c.len_t, _cu(dev, c.lens))
    return k, v


def _codes(x, kind):
    """The float32 formula on the CPU: (codes, scales)."""
    x = x.to(F32)
    m = x.abs().amax(-1)
    fine = m > 2.0 ** -100
    top = torch.full_like(m, TOP[kind])                       # (a number / a tensor is two roundings)
    y = x * torch.where(fine, top / m, torch.zeros(()))[..., None]
    c = torch.round(y).to(torch.int8) if kind == "int8" else y.to(torch.float8_e4m3fn)
    return c, torch.where(fine, m / top, torch.zeros(()))


# -- the cache -----------------------------------------------------------------

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dh,H,P", [(64, 1, 16), (64, 6, 64), (128, 3, 32), (128, 2, 256)])
@pytest.mark.parametrize("src", [BF, F32], ids=["bf16", "f32"])
def test_write_read(pkg, dev, kind, dh, H, P, src):
    """Whole sequences, then single tokens behind them: codes, scales and what
    is read back; slots that no call names keep their bits."""
    lens = [1, 0, 15, 16, 17, P, P + 1, 2 * P + 5, 77]
    print(f"[gpu] kv write/read {kind} dh{dh} H{H} P{P} {src}", flush=True)
    c = Cache(pkg, dev, kind, H, dh, P, [n + 1 for n in lens], seed=1)
    before = (c.pages.k.clone(), c.pages.v.clone())
    g = torch.Generator().manual_seed(2)
    T = sum(lens)
    k, v = (torch.randn(T, H, dh, generator=g).mul(3).to(src) for _ in range(2))
    k[0, 0], v[T - 1] = 0, 0                                  # rows of nothing
    k[1, 0, 3] = 3e38 if src == F32 else 2.0 ** 100           # a row of one large value
    v[2, 0] = v[2, 0] * 2.0 ** -60
    cu = _cu(dev, lens)
    before_lens = torch.tensor(lens, dtype=I32, device=dev)
    pkg.kv_write(c.pages, k.to(dev), v.to(dev), c.table, before_lens, cu)
    one = [torch.randn(len(lens), H, dh, generator=g).to(src) for _ in range(2)]
    pkg.kv_write(c.pages, one[0].to(dev), one[1].to(dev), c.table, c.len_t)   # cu None: one token each
    got = pkg.kv_read(c.pages, c.table, before_lens, cu, total=T, dtype=F32)
    last = pkg.kv_read(c.pages, c.table, c.len_t, dtype=F32)
    half = pkg.kv_read(c.pages, c.table, before_lens, cu, total=T)
    for x, y, z, o, w in zip((k, v), got, half, one, last):
        for a, b in ((x, y), (o, w)):
            b = b.cpu()
            if kind == "bf16":
                assert torch.equal(b, a.to(BF).to(F32))
                continue
            codes, sc = _codes(a, kind)
            assert torch.equal(b, codes.to(F32) * sc[..., None])
            m = a.to(F64).abs().amax(-1, keepdim=True)
            step = m / 254 if kind == "int8" else torch.maximum(a.to(F64).abs() / 16, m / 448 / 1024)
            assert ((b.to(F64) - a.to(F64)).abs() <= step + 1e-6 * m).all()
        assert torch.equal(z, y.to(BF))
    # untouched slots
    used = torch.zeros(c.pages.n_pages, P, dtype=torch.bool)
    for b, n in enumerate(c.lens):
        for p in range(n):
            used[c.rows[b][p // P], p % P] = True
    raw = lambda t: t.view(torch.uint8 if t.element_size() == 1 else torch.int16).cpu()  # noqa: E731
    keep = ~used
    assert torch.equal(raw(c.pages.k).transpose(1, 2)[keep], raw(before[0]).transpose(1, 2)[keep])
    assert torch.equal(raw(c.pages.v).permute(0, 3, 1, 2)[keep], raw(before[1]).permute(0, 3, 1, 2)[keep])


@pytest.mark.parametrize("kind", KINDS)
def test_read_holds_what_the_pages_hold(pkg, dev, kind):
    c = Cache(pkg, dev, kind, 2, 64, 32, [45, 3, 100], seed=3)
    _fill(pkg, dev, c, torch.Generator().manual_seed(4))
    k, v = pkg.kv_read(c.pages, c.table, c.len_t, _cu(dev, c.lens), total=148, dtype=F32)
    at = 0
    for b, n in enumerate(c.lens):
        for x, y in zip((k, v), c.held(b)):
            # one product in float32
            assert torch.allclose(x[at:at + n].cpu().to(F64), y, rtol=1e-7, atol=0)
        at += n


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_write_of_infinities_and_small_rows(pkg, dev, kind):
    c = Cache(pkg, dev, kind, 2, 64, 16, [6], seed=5)
    x = torch.randn(6, 2, 64, generator=torch.Generator().manual_seed(6))
    x[1, 0, 5], x[2, 1, 63], x[3, 0, 0] = math.inf, -math.inf, math.nan
    x[4, 0] *= 2.0 ** -105
    x[5, 1] *= 2.0 ** -90
    print(f"[gpu] kv write of infinities {kind}", flush=True)
    for src in (F32, BF):
        y = x.to(src)
        pkg.kv_write(c.pages, y.to(dev), (2 * y).to(dev), c.table, c.len_t, _cu(dev, [6]))
        for t, s in zip(pkg.kv_read(c.pages, c.table, c.len_t, _cu(dev, [6]), total=6, dtype=F32), (y, 2 * y)):
            t = t.cpu()
            bad = ~torch.isfinite(s).all(-1)
            assert torch.isnan(t[bad]).all() and torch.isfinite(t[~bad]).all()
            assert (t[4, 0] == 0).all() and (t[5, 1] != 0).any()


def test_strided_rows_and_missing_pages(pkg, dev):
    """Rows in a wider tensor (as the two routes of one call give them), rows
    that have to be copied first, positions without pages."""
    T, H, dh, P = 40, 3, 64, 16
    c = Cache(pkg, dev, "bf16", H, dh, P, [T], seed=7)
    g = torch.Generator().manual_seed(8)
    wide = torch.randn(T, 2, H * dh, generator=g).to(BF).to(dev)
    k, v = wide[:, 0].view(T, H, dh), wide[:, 1].view(T, H, dh)
    odd = torch.randn(T * H * dh + 1, generator=g).to(BF).to(dev)[1:].view(T, H, dh)
    cu = _cu(dev, [T])
    print("[gpu] kv strided rows", flush=True)
    for a, b in ((k, v), (odd, v.transpose(0, 1).contiguous().transpose(0, 1)), (v, torch.flip(odd, [2]))):
        pkg.kv_write(c.pages, a, b, c.table, c.len_t, cu)
        ra, rb = pkg.kv_read(c.pages, c.table, c.len_t, cu, total=T)
        assert torch.equal(ra, a) and torch.equal(rb, b)
    table = c.table.clone()
    table[0, 1], table[0, 2] = -1, c.pages.n_pages           # neither names a page
    keep = (c.pages.k.clone(), c.pages.v.clone())
    pkg.kv_write(c.pages, odd, odd, table, c.len_t, cu)
    ra, rb = pkg.kv_read(c.pages, table, c.len_t, cu, total=T)
    for t in (ra, rb):
        assert torch.equal(t[:16], odd[:16]) and (t[16:] == 0).all()
    for t, u in zip((c.pages.k, c.pages.v), keep):           # their pages were not touched
        ids = torch.tensor([i for i in range(c.pages.n_pages) if i != c.rows[0][0]], device=dev)
        assert torch.equal(t[ids].view(torch.int16), u[ids].view(torch.int16))
    # more new tokens than the sequence is long, more positions than the table holds
    short = torch.tensor([25], dtype=I32, device=dev)
    ra, _ = pkg.kv_read(c.pages, c.table, short, cu, total=T)
    assert (ra[:15] == 0).all() and torch.equal(ra[15:31], odd[:16])
    long = torch.tensor([60], dtype=I32, device=dev)
    pkg.kv_write(c.pages, odd, odd, c.table, long, cu)
    ra, _ = pkg.kv_read(c.pages, c.table, long, cu, total=T)
    assert torch.equal(ra[:28], odd[:28]) and (ra[28:] == 0).all()


# -- attention -------------------------------------------------------------------

def _check(pkg, dev, kind, dh, H, G, P, new, past, window=0, sinks=0, scale=None, max_new=None, seed=0, holes=()):
    lens = [n + m for n, m in zip(new, past)]
    c = Cache(pkg, dev, kind, H, dh, P, lens, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    _fill(pkg, dev, c, g)
    for b, i in holes:                                        # pages that a sequence gave back
        c.table[b, i] = -1
    T = sum(new)
    q = torch.randn(T, H * G, dh, generator=g).to(BF)
    cu = None if max(new) == 1 and min(new) == 1 else _cu(dev, new)
    got = pkg.paged_attention(q.to(dev), c.pages, c.table, c.len_t, cu, max_new=max(new) if max_new is None else max_new,
                              window=window, sinks=sinks, scale=scale)
    torch.cuda.synchronize()
    assert got.dtype == BF and got.shape == q.shape
    at, worst = 0, 0.0
    for b, n in enumerate(new):
        if n == 0:
            continue
        seen = torch.ones(lens[b], dtype=torch.bool)
        for bb, i in holes:
            if bb == b:
                seen[i * P:(i + 1) * P] = False
        k, v = c.held(b)
        by = 1 / math.sqrt(dh) if scale is None else scale
        want, mag = _attend64(q[at:at + n], k, v, past[b], by, window, sinks, seen)
        err = (got[at:at + n].cpu().to(F64) - want).abs()
        assert torch.isfinite(got[at:at + n]).all()
        assert (err <= BAR * mag + 1e-30).all(), (b, float((err / (BAR * mag + 1e-30)).max()))
        worst = max(worst, float((err / (mag + 1e-30)).max()))
        at += n
    print(f"  worst |error| / sum p|v|: {worst:.2e} (bar {BAR:.2e})", flush=True)
    return got


# single tokens: one position, around a tile of 64, a page, four waves' tiles, splits
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dh,H,G,P", [(64, 6, 1, 64), (64, 2, 4, 16), (128, 2, 8, 32), (128, 1, 16, 128), (64, 1, 20, 32),
                                      (64, 2, 40, 64), (64, 1, 130, 64)])
def test_single_tokens(pkg, dev, kind, dh, H, G, P):
    past = [0, 1, 15, 16, 62, 63, 64, 65, 255, 256, 300, 1025]
    print(f"[gpu] attention single tokens {kind} dh{dh} H{H} G{G} P{P}", flush=True)
    _check(pkg, dev, kind, dh, H, G, P, [1] * len(past), past, seed=11)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dh,G", [(64, 1), (128, 4), (64, 24)])
def test_one_long_sequence(pkg, dev, kind, dh, G):
    """Few rows over many positions: split and joined."""
    print(f"[gpu] attention long {kind} dh{dh} G{G}", flush=True)
    _check(pkg, dev, kind, dh, 1, G, 64, [1], [9001], seed=12)
    _check(pkg, dev, kind, dh, 1, G, 64, [3, 1], [9001, 20], seed=13)


# chunks: rows of 16, 32 and 128 a workgroup, their neighbours, nothing before,
# much before, sequences without new tokens
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dh,H,G,P", [(64, 2, 1, 64), (64, 1, 3, 16), (128, 2, 2, 32), (128, 1, 8, 256)])
def test_chunks(pkg, dev, kind, dh, H, G, P):
    print(f"[gpu] attention chunks {kind} dh{dh} H{H} G{G} P{P}", flush=True)
    _check(pkg, dev, kind, dh, H, G, P, [2, 5, 0, 4], [0, 61, 7, 130], seed=21)
    _check(pkg, dev, kind, dh, H, G, P, [31, 1, 16], [0, 64, 200], seed=22)
    _check(pkg, dev, kind, dh, H, G, P, [129, 0, 1, 128, 70, 300], [0, 5, 0, 0, 333, 64], seed=23)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dh,H,G,P", [(64, 2, 1, 16), (64, 1, 4, 64), (128, 1, 2, 64)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 4), (64, 4), (65, 70), (130, 16), (1000, 4)])
def test_windows(pkg, dev, kind, dh, H, G, P, window, sinks):
    print(f"[gpu] attention window {window} sinks {sinks} {kind} dh{dh} G{G} P{P}", flush=True)
    _check(pkg, dev, kind, dh, H, G, P, [1, 1, 1, 1], [0, 70, 333, 1200], window, sinks, seed=31)
    _check(pkg, dev, kind, dh, H, G, P, [200, 3, 66], [0, 500, 131], window, sinks, seed=32)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_chunk_split_over_a_long_axis(pkg, dev, kind):
    print(f"[gpu] attention split chunk {kind}", flush=True)
    _check(pkg, dev, kind, 64, 1, 1, 64, [100, 60], [7000, 100], seed=41)
    _check(pkg, dev, kind, 128, 1, 2, 32, [70], [5000], window=3000, sinks=5, seed=42)


# tables far wider than the sequences: splits of what a row tile sees, more of
# them than it has tiles, joined by one, four or all groups of a workgroup
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dh,H,G,new,past,width", [
    (64, 2, 1, [1, 1, 1], [2000, 0, 129], 2048),             # one token each, many splits of few rows
    (128, 1, 8, [1] * 40, [40 * i for i in range(40)], 128),  # some splits of more rows
    (64, 1, 1, [60, 1, 40], [333, 70, 0], 512),              # 32 rows a workgroup
    (128, 2, 2, [300, 0, 129], [900, 5, 0], 300),            # 128 rows a workgroup
    (64, 1, 1, [300, 2], [1500, 3000], 2048),                # the same, many splits of many rows
])
@pytest.mark.parametrize("window", [0, 700])
def test_tables_wider_than_their_sequences(pkg, dev, kind, dh, H, G, new, past, width, window):
    print(f"[gpu] attention wide table {kind} dh{dh} H{H} G{G} new {new[:3]} width {width} window {window}", flush=True)
    sinks = 4 if window else 0
    lens = [n + m for n, m in zip(new, past)]
    c = Cache(pkg, dev, kind, H, dh, 64, lens, seed=81)
    g = torch.Generator().manual_seed(82)
    _fill(pkg, dev, c, g)
    table = torch.full((len(new), width), -1, dtype=I32, device=dev)
    table[:, :c.table.shape[1]] = c.table
    q = torch.randn(sum(new), H * G, dh, generator=g).to(BF)
    cu = None if max(new) == 1 else _cu(dev, new)
    got = pkg.paged_attention(q.to(dev), c.pages, table, c.len_t, cu, max_new=max(new), window=window, sinks=sinks)
    torch.cuda.synchronize()
    at = 0
    for b, n in enumerate(new):
        if n == 0:
            continue
        k, v = c.held(b)
        want, mag = _attend64(q[at:at + n], k, v, past[b], 1 / math.sqrt(dh), window, sinks)
        err = (got[at:at + n].cpu().to(F64) - want).abs()
        assert (err <= BAR * mag + 1e-30).all(), (b, float((err / (BAR * mag + 1e-30)).max()))
        at += n


@pytest.mark.parametrize("max_new", [0, 1, 5, 1000])
def test_max_new_is_a_hint(pkg, dev, max_new):
    print(f"[gpu] attention max_new {max_new}", flush=True)
    _check(pkg, dev, "bf16", 64, 2, 3, 32, [40, 1, 7], [10, 99, 0], max_new=max_new, seed=51)


@pytest.mark.parametrize("kind", KINDS)
def test_pages_given_back(pkg, dev, kind):
    """Positions without a page are not seen, whatever else is; a row left
    with nothing gives zeros."""
    print(f"[gpu] attention holes {kind}", flush=True)
    _check(pkg, dev, kind, 64, 2, 2, 16, [1, 1, 1], [100, 31, 5], seed=61, holes=[(0, 0), (0, 3), (1, 1), (2, 0)])
    _check(pkg, dev, kind, 64, 1, 2, 32, [90, 40], [50, 0], seed=62, holes=[(0, 1), (0, 2), (1, 0)])
    got = _check(pkg, dev, kind, 128, 1, 1, 32, [40], [0], seed=63, holes=[(0, 0)])
    assert (got[:32] == 0).all() and (got[32:] != 0).any()


def test_rows_before_the_first_position(pkg, dev):
    """More new tokens than positions: the first rows see nothing."""
    c = Cache(pkg, dev, "bf16", 2, 64, 16, [20], seed=71)
    g = torch.Generator().manual_seed(72)
    _fill(pkg, dev, c, g)
    print("[gpu] attention rows before position 0", flush=True)
    for n, most in ((30, 30), (30, 4), (22, 22)):
        q = torch.randn(n, 2, 64, generator=g).to(BF)
        got = pkg.paged_attention(q.to(dev), c.pages, c.table, c.len_t, _cu(dev, [n]), max_new=most).cpu()
        assert (got[:n - 20] == 0).all()
        k, v = c.held(0)
        want, mag = _attend64(q[n - 20:], k, v, 0, 0.125, 0, 0)
        assert ((got[n - 20:].to(F64) - want).abs() <= BAR * mag).all()
    zero = torch.zeros(1, dtype=I32, device=dev)
    assert (pkg.paged_attention(q[:1].to(dev), c.pages, c.table, zero) == 0).all()
    none = pkg.KvPages(*(torch.empty(s, dtype=BF, device=dev) for s in ((0, 2, 16, 64), (0, 2, 64, 16))))
    assert (pkg.paged_attention(q[:1].to(dev), none, c.table, c.len_t) == 0).all()
    assert (pkg.kv_read(none, c.table, c.len_t)[0] == 0).all()
    pkg.kv_write(none, q[:1].to(dev), q[:1].to(dev), c.table, c.len_t)
    empty = q[:0].to(dev)
    assert pkg.paged_attention(empty, c.pages, c.table, c.len_t, _cu(dev, [0])).shape == (0, 2, 64)


@pytest.mark.parametrize("n", [1, 100])
def test_large_scores_and_scales(pkg, dev, n):
    """Rows whose weight lies on one key, equal scores, a negative scale."""
    print(f"[gpu] attention scales {n}", flush=True)
    for scale in (50.0, 0.0, -1.0, 1e-8):
        if scale == 50.0:
            # scores of size 400 * 50: float32 keeps them to 2^-8, which moves
            # a weight by 1%; the largest wins all the same
            c = Cache(pkg, dev, "bf16", 1, 64, 64, [n + 200], seed=81)
            g = torch.Generator().manual_seed(82)
            _fill(pkg, dev, c, g)
            q = torch.randn(n, 1, 64, generator=g).to(BF)
            got = pkg.paged_attention(q.to(dev), c.pages, c.table, c.len_t, _cu(dev, [n]), max_new=n, scale=scale).cpu()
            k, v = c.held(0)
            want, mag = _attend64(q, k, v, 200, scale, 0, 0)
            assert ((got.to(F64) - want).abs() <= (BAR + 0.02) * mag.amax(-1, keepdim=True)).all()
        else:
            _check(pkg, dev, "int8", 64, 1, 2, 32, [n], [200], scale=scale, seed=83)


@pytest.mark.parametrize("n", [1, 20, 200])
def test_infinite_and_nan_keys(pkg, dev, n):
    """Scores of -inf weigh nothing, NaN and +inf make the rows that see them
    NaN, later tokens' do not reach earlier rows."""
    print(f"[gpu] attention infinities {n}", flush=True)
    g = torch.Generator().manual_seed(91)
    past = 150
    L = past + n
    c = Cache(pkg, dev, "bf16", 1, 64, 64, [L], seed=92)
    k, v = (torch.randn(L, 1, 64, generator=g).to(BF) for _ in range(2))
    q = torch.randn(n, 1, 64, generator=g).abs().to(BF)      # so that -inf in a key gives -inf
    cu = _cu(dev, [L])

    def run(k, v):
        pkg.kv_write(c.pages, k.to(dev), v.to(dev), c.table, c.len_t, cu)
        return pkg.paged_attention(q.to(dev), c.pages, c.table, c.len_t, _cu(dev, [n]), max_new=n).cpu()

    kk = k.clone()
    kk[5, 0, 3] = kk[past - 1, 0, 7] = -math.inf
    got = run(kk, v)
    seen = torch.ones(L, dtype=torch.bool)
    seen[5] = seen[past - 1] = False
    want, mag = _attend64(q, k.to(F64), v.to(F64), past, 0.125, 0, 0, seen)
    assert ((got.to(F64) - want).abs() <= BAR * mag).all()
    for bad in (math.nan, math.inf):
        kk = k.clone()
        kk[L - 1, 0, 3] = bad                                 # the last token's key
        got = run(kk, v)
        assert torch.isnan(got[n - 1]).all() and torch.isfinite(got[:n - 1]).all()
        vv = v.clone()
        vv[L - 1, 0, 3] = bad                                 # its value: that dim of its own row
        got = run(k, vv)
        want, mag = _attend64(q, k.to(F64), v.to(F64), past, 0.125, 0, 0)
        assert not torch.isfinite(got[n - 1, 0, 3])
        ok = torch.ones(n, 1, 64, dtype=torch.bool)
        ok[n - 1, 0, 3] = False
        assert ((got.to(F64) - want).abs() <= BAR * mag)[ok].all()


def test_rows_do_not_depend_on_the_batch(pkg, dev):
    """A sequence's rows are the same, bit for bit, alone and among others of
    one table width."""
    c = Cache(pkg, dev, "int8", 2, 64, 32, [200, 90, 333], seed=101)
    g = torch.Generator().manual_seed(102)
    _fill(pkg, dev, c, g)
    new = [20, 1, 150]
    q = torch.randn(sum(new), 4, 64, generator=g).to(BF).to(dev)
    print("[gpu] attention batch independence", flush=True)
    whole = pkg.paged_attention(q, c.pages, c.table, c.len_t, _cu(dev, new), max_new=150)
    at = 0
    for b, n in enumerate(new):
        alone = pkg.paged_attention(q[at:at + n], c.pages, c.table[b:b + 1], c.len_t[b:b + 1], _cu(dev, [n]), max_new=150)
        assert torch.equal(alone, whole[at:at + n])
        assert torch.equal(whole, pkg.paged_attention(q, c.pages, c.table, c.len_t, _cu(dev, new), max_new=150))
        at += n


def test_strided_queries_other_streams_and_capture(pkg, dev):
    c = Cache(pkg, dev, "fp8", 2, 64, 32, [200, 1000], seed=111)
    g = torch.Generator().manual_seed(112)
    _fill(pkg, dev, c, g)
    wide = torch.randn(2, 3, 4, 64, generator=g).to(BF).to(dev)
    q = wide[:, 1]
    print("[gpu] attention strides, streams, capture", flush=True)
    want = pkg.paged_attention(q.contiguous(), c.pages, c.table, c.len_t)
    assert torch.equal(pkg.paged_attention(q, c.pages, c.table, c.len_t), want)
    odd = torch.empty(2 * 4 * 64 + 1, dtype=BF, device=dev)[1:].view(2, 4, 64)
    odd.copy_(q)
    assert torch.equal(pkg.paged_attention(odd, c.pages, c.table, c.len_t), want)
    out = torch.empty(2, 4, 64, dtype=BF, device=dev)
    assert pkg.paged_attention(q, c.pages, c.table, c.len_t, out=out) is out and torch.equal(out, want)
    padded = torch.full((2, c.table.shape[1] + 3), 7, dtype=I32, device=dev)[:, :c.table.shape[1]]
    padded.copy_(c.table)
    assert torch.equal(pkg.paged_attention(q, c.pages, padded, c.len_t), want)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = pkg.paged_attention(q, c.pages, c.table, c.len_t)
    side.synchronize()
    assert torch.equal(other, want)
    k = torch.randn(2, 2, 64, generator=g).to(BF).to(dev)
    graph = torch.cuda.CUDAGraph()
    cap = torch.cuda.Stream(dev)
    cap.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.graph(graph, stream=cap):
        pkg.kv_write(c.pages, k, k, c.table, c.len_t)
        got = pkg.paged_attention(q, c.pages, c.table, c.len_t)
    for rep in range(3):
        k.normal_(generator=torch.Generator(device=dev).manual_seed(rep))
        graph.replay()
        torch.cuda.synchronize()
        mine = got.clone()
        pkg.kv_write(c.pages, k, k, c.table, c.len_t)
        assert torch.equal(pkg.paged_attention(q, c.pages, c.table, c.len_t), mine), rep


def test_offsets_past_32_bits(pkg, dev):
    """Pages whose first byte lies past 2^32, in a cache of 5 GB a tensor."""
    H, P, dh = 8, 256, 128
    n_pages = 10000
    k = torch.empty(n_pages, H, P, dh, dtype=BF, device=dev)
    v = torch.empty(n_pages, H, dh, P, dtype=BF, device=dev)
    assert k.numel() * 2 > 2 ** 32
    pages = pkg.KvPages(k, v)
    g = torch.Generator().manual_seed(121)
    n = 300
    table = torch.tensor([[n_pages - 1, n_pages - 2]], dtype=I32, device=dev)
    lens, cu = torch.tensor([n], dtype=I32, device=dev), _cu(dev, [n])
    x, y = (torch.randn(n, H, dh, generator=g).to(BF) for _ in range(2))
    print("[gpu] kv offsets past 32 bits", flush=True)
    pkg.kv_write(pages, x.to(dev), y.to(dev), table, lens, cu)
    a, b = pkg.kv_read(pages, table, lens, cu, total=n)
    assert torch.equal(a.cpu(), x) and torch.equal(b.cpu(), y)
    for m in (1, 40):
        q = torch.randn(m, H, dh, generator=g).to(BF)
        got = pkg.paged_attention(q.to(dev), pages, table, lens, _cu(dev, [m]), max_new=m).cpu()
        want, mag = _attend64(q, x.to(F64), y.to(F64), n - m, 1 / math.sqrt(dh), 0, 0)
        assert ((got.to(F64) - want).abs() <= BAR * mag).all()


def test_refusals(pkg, dev):
    C = pkg._capi
    c = Cache(pkg, dev, "int8", 2, 64, 16, [20, 5], seed=131)
    p, q = c.pages, torch.zeros(2, 4, 64, dtype=BF, device=dev)
    kv = torch.zeros(2, 2, 64, dtype=BF, device=dev)
    ok = (q, p, c.table, c.len_t)
    print("[gpu] kv refusals", flush=True)

    def refuses(kind, f, *a, **kw):
        with pytest.raises(kind):
            f(*a, **kw)

    att = pkg.paged_attention
    refuses(TypeError, att, q.float(), *ok[1:])
    refuses(ValueError, att, q[:, :3], *ok[1:])
    refuses(ValueError, att, q[..., :32], *ok[1:])
    refuses(ValueError, att, q.cpu(), *ok[1:])
    refuses(ValueError, att, q[:1], *ok[1:])                                   # needs cu
    refuses(ValueError, att, *ok, sinks=2)
    refuses(ValueError, att, *ok, window=-1)
    refuses(TypeError, att, q, p, c.table.long(), c.len_t)
    refuses(TypeError, att, q, p, c.table, c.len_t.long())
    refuses(ValueError, att, q, p, c.table[:1], c.len_t)
    refuses(ValueError, att, q, p, c.table, c.len_t, c.len_t)
    refuses(ValueError, att, q, p, c.table.t().contiguous().t(), c.len_t)
    refuses(ValueError, att, *ok, out=torch.empty(2, 4, 32, dtype=BF, device=dev))
    refuses(ValueError, pkg.kv_write, p, kv[:, :1], kv[:, :1], c.table, c.len_t)
    refuses(TypeError, pkg.kv_write, p, kv, kv.float(), c.table, c.len_t)
    refuses(TypeError, pkg.kv_write, p, kv.half(), kv.half(), c.table, c.len_t)
    refuses(ValueError, pkg.kv_read, p, c.table, c.len_t, _cu(dev, [1, 1]))    # total
    refuses(TypeError, pkg.kv_read, p, c.table, c.len_t, dtype=torch.float16)
    refuses(TypeError, pkg.KvPages, p.k.float(), p.v.float())
    refuses(TypeError, pkg.KvPages, p.k, p.v)                                  # scales
    refuses(ValueError, pkg.KvPages, p.k, p.k, p.k_scale, p.v_scale)
    odd = [torch.zeros(s, dtype=BF, device=dev) for s in ((2, 1, 24, 64), (2, 1, 64, 24))]
    refuses(C.SrwError, att, q, pkg.KvPages(*odd), c.table, c.len_t)
    thin = [torch.zeros(s, dtype=BF, device=dev) for s in ((2, 1, 16, 32), (2, 1, 32, 16))]
    refuses(C.SrwError, att, q[..., :32].contiguous(), pkg.KvPages(*thin), c.table, c.len_t)
    refuses(C.SrwError, att, *ok, window=3, scale=math.inf)
    # a workspace that is missing or too small
    lib = C.load_library()
    long = Cache(pkg, dev, "bf16", 1, 64, 64, [9000], seed=132)
    from dawn_srw_amd.kv import _address
    q1, out = torch.zeros(1, 1, 64, dtype=BF, device=dev), torch.zeros(1, 1, 64, dtype=BF, device=dev)
    a = C.SrwAttention(C.SrwKv(*_address(long.pages, long.table, long.len_t, None, 1)), q1.data_ptr(), out.data_ptr(), 64, 64, 1, 1,
                       0, 0, 1.0)
    need = ctypes.c_size_t(0)
    assert lib.srw_attention_workspace_size(ctypes.byref(a), ctypes.byref(need)) == C.SRW_OK and need.value > 0
    assert lib.srw_attention(ctypes.byref(a), None, need.value, None) == C.SRW_EWORKSPACE
    ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
    assert lib.srw_attention(ctypes.byref(a), ws.data_ptr(), need.value - 1, None) == C.SRW_EWORKSPACE
    torch.cuda.synchronize()


def test_calls_without_the_native_host_side(pkg, dev, monkeypatch):
    """The general path, which the native host side hands calls to that it does
    not take, makes the same calls."""
    from dawn_srw_amd import kv
    new, past = [3, 1, 70], [40, 200, 0]
    c = Cache(pkg, dev, "int8", 2, 64, 32, [n + m for n, m in zip(new, past)], seed=141)
    g = torch.Generator().manual_seed(142)
    _fill(pkg, dev, c, g)
    k, v = (torch.randn(74, 2, 64, generator=g).to(BF).to(dev) for _ in range(2))
    q = torch.randn(74, 4, 64, generator=g).to(BF).to(dev)
    cu = _cu(dev, new)

    def calls():
        pkg.kv_write(c.pages, k, v, c.table, c.len_t, cu)
        return (*pkg.kv_read(c.pages, c.table, c.len_t, cu, total=74, dtype=F32),
                pkg.paged_attention(q, c.pages, c.table, c.len_t, cu, max_new=70, window=50, sinks=3),
                c.pages.k.clone(), c.pages.v.clone(), pkg.KvPages(c.pages.k, c.pages.v, c.pages.k_scale, c.pages.v_scale)._at)

    class Nothing:
        def __getattr__(self, name):
            return lambda *args: None

    print("[gpu] kv without the native host side", flush=True)
    native = calls()
    monkeypatch.setattr(kv, "_host", Nothing())
    for a, b in zip(native, calls()):
        assert a == b if isinstance(a, tuple) else torch.equal(a, b)


def test_pages_are_looked_at_in_every_call(pkg, dev):
    """Tensors whose memory became another's, names that cannot be put on other
    tensors, tensors whose shape no longer fits."""
    print("[gpu] pages looked at anew", flush=True)
    lens = torch.tensor([20], dtype=I32, device=dev)
    table = torch.tensor([[1, 0]], dtype=I32, device=dev)
    cu = _cu(dev, [20])
    g = torch.Generator().manual_seed(91)
    rows = torch.randn(20, 1, 64, generator=g).to(BF).to(dev)
    pages = pkg.KvPages(torch.zeros(2, 1, 16, 64, dtype=BF, device=dev), torch.zeros(2, 1, 64, 16, dtype=BF, device=dev))
    old, old_v = pages.k.data, pages.v.data
    pages.k.data, pages.v.data = torch.zeros_like(old), torch.zeros_like(old_v)
    pkg.kv_write(pages, rows, rows, table, lens, cu)
    assert (old == 0).all() and (old_v == 0).all()
    assert torch.equal(pages.k[1, 0], rows[:16, 0]) and torch.equal(pages.v[0, 0, :, :4].T, rows[16:, 0])
    for name in ("k", "v", "k_scale", "v_scale"):
        with pytest.raises(AttributeError):
            setattr(pages, name, old)
    pages.v.data = torch.zeros(2, 1, 16, 64, dtype=BF, device=dev)
    for call in (lambda: pkg.kv_write(pages, rows, rows, table, lens, cu),
                 lambda: pkg.kv_read(pages, table, lens, cu, total=20),
                 lambda: pkg.paged_attention(rows, pages, table, lens, cu)):
        with pytest.raises(ValueError):
            call()


def test_tensors_that_want_gradients_are_refused(pkg, dev):
    print("[gpu] no gradients", flush=True)
    lens, table = torch.tensor([1], dtype=I32, device=dev), torch.tensor([[0]], dtype=I32, device=dev)
    pages = pkg.KvPages(torch.zeros(1, 1, 16, 64, dtype=BF, device=dev), torch.zeros(1, 1, 64, 16, dtype=BF, device=dev))
    x = torch.ones(1, 1, 64, dtype=BF, device=dev)
    w = x.clone().requires_grad_()
    for call in (lambda: pkg.kv_write(pages, w, x, table, lens), lambda: pkg.kv_write(pages, x, w, table, lens),
                 lambda: pkg.paged_attention(w, pages, table, lens)):
        with pytest.raises(NotImplementedError):
            call()
    with torch.no_grad():
        pkg.kv_write(pages, w, w, table, lens)
        assert torch.equal(pkg.paged_attention(w, pages, table, lens), x)
