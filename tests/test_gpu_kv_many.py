"""GPU: paged_attention's kernel for many rows (128 a workgroup) -- pages smaller
and larger than its tiles, windows, missing pages, values that are not finite,
whole and split -- against plain float64 on the CPU (bounds as in
test_gpu_kv.py).  Every call is asserted to run on it, and in how many splits."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from tests.test_gpu_kv import BAR, BF, F32, F64, I32, KINDS, Cache, _attend64, _cu, _fill

pytestmark = pytest.mark.gpu


def plan(pkg, q, pages, table, lens, cu, max_new=0, window=0, sinks=0):
    """(rows a workgroup, splits) of the call."""
    from dawn_srw_amd.kv import _address
    C = pkg._capi
    a = C.SrwAttention(C.SrwKv(*_address(pages, table, lens, cu, q.shape[0])), q.data_ptr(), q.data_ptr(), q.stride(0),
                       q.stride(1), q.shape[1], max_new, window, sinks, 1.0)
    rows, splits = ctypes.c_int32(-1), ctypes.c_int32(-1)
    C.check(C.load_library().srw_attention_plan(ctypes.byref(a), ctypes.byref(rows), ctypes.byref(splits)))
    return rows.value, splits.value


def attend(pkg, split, q, pages, table, lens, cu, max_new, **kw):
    """The call, which has to run on the kernel for many rows, whole or split."""
    rows, splits = plan(pkg, q, pages, table, lens, cu, max_new, **{k: v for k, v in kw.items() if k in ("window", "sinks")})
    assert rows == 128 and (splits > 1) == split, (rows, splits)
    out = pkg.paged_attention(q, pages, table, lens, cu, max_new=max_new, **kw)
    torch.cuda.synchronize()
    return out


# whole: 5 604 rows over at most 768 positions; split: 912 rows in a table for 8 192
# positions, with windows by a max_new that promises little (a hint only)
WHOLE = dict(H=1, G=4, new=[700, 640, 0, 61], past=[60, 100, 37, 333])
SPLIT = dict(H=2, G=2, new=[150, 1, 0, 77], past=[0, 300, 5, 1000])


class Call:
    """A batch of chunks over pages of P positions and their outputs, checked."""

    def __init__(self, pkg, dev, kind, dh, P, split, seed, holes=()):
        s = SPLIT if split else WHOLE
        self.pkg, self.split, self.new, self.past, self.P, self.dh = pkg, split, s["new"], s["past"], P, dh
        lens = [n + m for n, m in zip(self.new, self.past)]
        c = self.c = Cache(pkg, dev, kind, s["H"], dh, P, lens, seed=seed)
        g = torch.Generator().manual_seed(seed + 1)
        self.sources = _fill(pkg, dev, c, g)
        width = (8192 if split else 768) // P
        self.table = torch.full((len(lens), width), -1, dtype=I32, device=dev)
        self.table[:, :c.table.shape[1]] = c.table
        self.holes = [(b, i) for b, i in holes if i * P < lens[b]]
        for b, i in self.holes:
            self.table[b, i] = -1
        self.cu = _cu(dev, self.new)
        self.q = torch.randn(sum(self.new), s["H"] * s["G"], dh, generator=g).to(BF)
        self.dev = dev

    def run(self, window=0, sinks=0, **kw):
        most = 8192 if self.split and window else max(self.new)
        return attend(self.pkg, self.split, self.q.to(self.dev), self.c.pages, self.table, self.c.len_t, self.cu, most,
                      window=window, sinks=sinks, **kw).cpu()

    def sequences(self):
        """(b, rows, positions that have a page) of each sequence with new tokens."""
        at = 0
        for b, n in enumerate(self.new):
            if n:
                seen = torch.ones(self.c.lens[b], dtype=torch.bool)
                for bb, i in self.holes:
                    if bb == b:
                        seen[i * self.P:(i + 1) * self.P] = False
                yield b, slice(at, at + n), seen
            at += n

    def check(self, got, window=0, sinks=0, scale=None):
        for b, rows, seen in self.sequences():
            k, v = self.c.held(b)
            want, mag = _attend64(self.q[rows], k, v, self.past[b], scale or self.dh ** -0.5, window, sinks, seen)
            err = (got[rows].to(F64) - want).abs()
            assert torch.isfinite(got[rows]).all()
            assert (err <= BAR * mag + 1e-30).all(), (b, float((err / (BAR * mag + 1e-30)).max()))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("P", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("split", [False, True], ids=["whole", "split"])
def test_pages_and_windows(pkg, dev, kind, dh, P, split):
    print(f"[gpu] many rows {kind} dh{dh} P{P} split {split}", flush=True)
    call = Call(pkg, dev, kind, dh, P, split, 301)
    for window, sinks in ((0, 0), (1, 0), (70, 5), (130, 70), (300, 0), (1 << 30, 0)):
        call.check(call.run(window, sinks), window, sinks)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dh,P", [(64, 16), (64, 64), (64, 128), (128, 16), (128, 32), (128, 64)])
@pytest.mark.parametrize("split", [False, True], ids=["whole", "split"])
def test_missing_pages(pkg, dev, kind, dh, P, split):
    """Pages given back at the front, in the middle (some of a tile's, all of a
    tile's) and at the end; the first rows of a sequence see nothing."""
    print(f"[gpu] many rows, holes {kind} dh{dh} P{P} split {split}", flush=True)
    tile = max(1, 64 // P)
    holes = [(0, 0), (0, tile), *((0, 2 * tile + i) for i in range(tile)), (1, 1), (1, 5), (3, 0), (3, 3)]
    call = Call(pkg, dev, kind, dh, P, split, 311, holes)
    for window, sinks in ((0, 0), (70, 5)):
        got = call.run(window, sinks)
        call.check(got, window, sinks)
        if split and not window:
            assert (got[:min(P, call.new[0])] == 0).all()


@pytest.mark.parametrize("P", [16, 64, 128])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("split", [False, True], ids=["whole", "split"])
def test_infinite_and_nan_values(pkg, dev, dh, P, split):
    """Values that are not finite are those of the rows that see them, exactly."""
    print(f"[gpu] many rows, infinities dh{dh} P{P} split {split}", flush=True)
    call = Call(pkg, dev, "bf16", dh, P, split, 321)
    k, v = (t.clone() for t in call.sources)
    first = [sum(call.c.lens[:b]) for b in range(len(call.new))]
    # (sequence, position, dim, value); the last sequence has 77 or 61 new tokens
    last = len(call.new) - 1
    L = call.c.lens[last]
    bad = [(0, 0, 3, math.inf), (0, 70, 9, -math.inf), (0, 90, 11, math.inf), (0, 95, 11, -math.inf), (0, 20, 12, math.nan),
           (last, 5, 3, math.inf), (last, L - 30, 7, -math.inf), (last, L - 1, 8, math.nan)]
    for b, p, d, x in bad:
        v[first[b] + p, 0, d] = x
    pkg.kv_write(call.c.pages, k.to(dev), v.to(dev), call.table, call.c.len_t, _cu(dev, call.c.lens))
    got = call.run().to(F64)
    G = SPLIT["G"] if split else WHOLE["G"]
    for b, rows, _ in call.sequences():
        kk, vv = (t[first[b]:first[b] + call.c.lens[b]].to(F64) for t in (k, call.sources[1]))
        want, mag = _attend64(call.q[rows], kk, vv, call.past[b], dh ** -0.5, 0, 0)
        for bb, p, d, x in bad:
            if bb == b:  # heads of key head 0, tokens at p and later
                want[max(0, p - call.past[b]):, :G, d] += x
        fine = torch.isfinite(want)
        assert ((got[rows] - want).abs() <= BAR * mag)[fine].all()
        assert torch.equal(got[rows][~fine].nan_to_num(7.0, 1e300, -1e300), want[~fine].nan_to_num(7.0, 1e300, -1e300))


@pytest.mark.parametrize("split", [False, True], ids=["whole", "split"])
def test_infinite_and_nan_keys(pkg, dev, split):
    """Keys of -inf weigh nothing; the rows that see a NaN are NaN, no earlier ones."""
    print(f"[gpu] many rows, keys split {split}", flush=True)
    call = Call(pkg, dev, "bf16", 64, 32, split, 331)
    k, v = (t.clone() for t in call.sources)
    call.q = call.q.abs()                                     # so that -inf in a key gives -inf
    n = call.new[0]
    k[5, 0, 3] = k[70, 0, 9] = -math.inf
    k[call.c.lens[0] - 1, 0, 5] = math.nan                    # the last token's of the first sequence
    pkg.kv_write(call.c.pages, k.to(dev), v.to(dev), call.table, call.c.len_t, _cu(dev, call.c.lens))
    got = call.run().to(F64)
    G = SPLIT["G"] if split else WHOLE["G"]
    kk, vv = (t[:call.c.lens[0], :1].to(F64) for t in call.sources)
    seen = torch.ones(call.c.lens[0], dtype=torch.bool)
    seen[5] = seen[70] = False
    want, mag = _attend64(call.q[:n, :G], kk, vv, call.past[0], 0.125, 0, 0, seen)
    assert ((got[:n - 1, :G] - want[:-1]).abs() <= BAR * mag[:-1]).all()
    assert torch.isnan(got[n - 1, :G]).all() and torch.isfinite(got[n:]).all()


@pytest.mark.parametrize("n,width", [(1, 0), (20, 0), (200, 400)], ids=str)
@pytest.mark.parametrize("P", [16, 64])
def test_nan_codes_of_later_positions(pkg, dev, n, width, P):
    """A caller's own fp8 pages may hold NaN's codes: in the rows that see them, no
    earlier ones."""
    print(f"[gpu] fp8 NaN codes n{n} P{P}", flush=True)
    past = 300
    L = past + n
    c = Cache(pkg, dev, "fp8", 1, 64, P, [L], seed=341)
    g = torch.Generator().manual_seed(342)
    k, v = _fill(pkg, dev, c, g)
    kk, vv = c.held(0)
    at = [(L - 1, 3), (max(L - 10, 0), 5)]
    raw = c.pages.v.view(torch.uint8)
    for p, d in at:
        raw[c.rows[0][p // P], 0, d, p % P] = 0x7f if d == 3 else 0xff
    table = c.table
    if width:
        table = torch.full((1, width * 64 // P), -1, dtype=I32, device=dev)
        table[:, :c.table.shape[1]] = c.table
    q = torch.randn(n, 2, 64, generator=g).to(BF)
    got = pkg.paged_attention(q.to(dev), c.pages, table, c.len_t, _cu(dev, [n]), max_new=n).cpu().to(F64)
    want, mag = _attend64(q, kk, vv, past, 0.125, 0, 0)
    for p, d in at:
        want[max(0, p - past):, :, d] = math.nan
    fine = torch.isfinite(want)
    assert ((got - want).abs() <= BAR * mag)[fine].all() and torch.isnan(got[~fine]).all()


@pytest.mark.parametrize("kind,P", [("bf16", 16), ("bf16", 256), ("int8", 16), ("int8", 128), ("fp8", 64)])
def test_offsets_past_32_bits(pkg, dev, kind, P):
    """Pages whose first byte lies past 2^32."""
    H, dh = 8, 128
    size = H * P * dh * (2 if kind == "bf16" else 1)
    n_pages = 2 ** 32 // size + 40
    dt = KINDS[kind]
    k = torch.empty(n_pages, H, P, dh, dtype=dt, device=dev)
    v = torch.empty(n_pages, H, dh, P, dtype=dt, device=dev)
    sc = [] if kind == "bf16" else [torch.empty(n_pages, H, P, device=dev) for _ in range(2)]
    assert (n_pages - 30) * size > 2 ** 32
    pages = pkg.KvPages(k, v, *sc)
    g = torch.Generator().manual_seed(351)
    n = 300
    need = -(-n // P)
    table = torch.full((1, 16384 // P), -1, dtype=I32, device=dev)
    table[0, :need] = torch.arange(n_pages - 1, n_pages - 1 - need, -1)
    lens, cu = torch.tensor([n], dtype=I32, device=dev), _cu(dev, [n])
    x, y = (torch.randn(n, H, dh, generator=g).to(BF) for _ in range(2))
    print(f"[gpu] many rows, offsets past 32 bits {kind} P{P}", flush=True)
    pkg.kv_write(pages, x.to(dev), y.to(dev), table, lens, cu)
    a, b = (t.cpu().to(F64) for t in pkg.kv_read(pages, table, lens, cu, total=n, dtype=F32))
    q = torch.randn(40, H, dh, generator=g).to(BF)
    got = attend(pkg, True, q.to(dev), pages, table, lens, _cu(dev, [40]), 40).cpu()
    want, mag = _attend64(q, a, b, n - 40, dh ** -0.5, 0, 0)
    assert ((got.to(F64) - want).abs() <= BAR * mag).all()


def test_rows_before_the_first_position(pkg, dev):
    """More new tokens than positions: the first rows see nothing."""
    print("[gpu] many rows before position 0", flush=True)
    c = Cache(pkg, dev, "bf16", 2, 64, 16, [250], seed=361)
    g = torch.Generator().manual_seed(362)
    _fill(pkg, dev, c, g)
    table = torch.full((1, 512), -1, dtype=I32, device=dev)
    table[:, :c.table.shape[1]] = c.table
    n = 400
    q = torch.randn(n, 2, 64, generator=g).to(BF)
    k, v = c.held(0)
    for window in (0, 100):
        got = attend(pkg, True, q.to(dev), c.pages, table, c.len_t, _cu(dev, [n]), 8192, window=window).cpu()
        assert (got[:150] == 0).all()
        want, mag = _attend64(q[150:], k, v, 0, 0.125, window, 0)
        assert ((got[150:].to(F64) - want).abs() <= BAR * mag).all()


@pytest.mark.parametrize("split", [False, True], ids=["whole", "split"])
def test_strided_queries_out_streams_and_capture(pkg, dev, split):
    print(f"[gpu] many rows, strides, streams, capture split {split}", flush=True)
    call = Call(pkg, dev, "int8", 64, 32, split, 371)
    want = call.run()
    T, Hq, dh = call.q.shape
    wide = torch.zeros(T, 3, Hq, dh, dtype=BF, device=dev)
    wide[:, 1] = call.q.to(dev)
    q, most = wide[:, 1], max(call.new)
    args = (call.c.pages, call.table, call.c.len_t, call.cu)
    assert torch.equal(attend(pkg, split, q, *args, most).cpu(), want)
    out = torch.empty(T, Hq, dh, dtype=BF, device=dev)
    assert pkg.paged_attention(q, *args, max_new=most, out=out) is out and torch.equal(out.cpu(), want)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = pkg.paged_attention(q, *args, max_new=most)
    side.synchronize()
    assert torch.equal(other.cpu(), want)
    graph, cap = torch.cuda.CUDAGraph(), torch.cuda.Stream(dev)
    cap.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.graph(graph, stream=cap):
        got = pkg.paged_attention(q, *args, max_new=most)
    for rep in range(3):
        wide.normal_(generator=torch.Generator(device=dev).manual_seed(rep))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, pkg.paged_attention(q, *args, max_new=most)), rep


@pytest.mark.parametrize("scale", [50.0, 0.0, -1.0])
def test_scales(pkg, dev, scale):
    print(f"[gpu] many rows, scale {scale}", flush=True)
    call = Call(pkg, dev, "int8", 64, 64, False, 381)
    got = call.run(scale=scale)
    if scale != 50.0:
        return call.check(got, scale=scale or 1e-300)
    # scores of size 50 x 40: float32's sums of 64 products move a weight by 1% (as in
    # test_large_scores_and_scales); the largest wins all the same
    for b, rows, seen in call.sequences():
        k, v = call.c.held(b)
        want, mag = _attend64(call.q[rows], k, v, call.past[b], scale, 0, 0, seen)
        assert ((got[rows].to(F64) - want).abs() <= (BAR + 0.02) * mag.amax(-1, keepdim=True)).all()
