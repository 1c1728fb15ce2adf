"""GPU: the ends of the range of the paged cache's calls, against plain float64
implementations on the CPU (bounds as in test_gpu_kv.py)."""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_kv import BAR, BF, F32, F64, I32, KINDS, Cache, _attend64, _codes, _cu

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


# -- attention -------------------------------------------------------------------

@pytest.mark.parametrize("dh,G", [(64, 1), (128, 2), (64, 24)])
@pytest.mark.parametrize("n,past", [(1, 300), (1, 9001), (20, 300)], ids=str)
def test_infinite_values(pkg, dev, dh, G, n, past):
    """A value of infinity weighs more than nothing in every row that sees it: that
    dim is the infinity, two of opposite signs make it NaN, and no other dim nor
    any row before it changes."""
    print(f"[gpu] attention infinite values dh{dh} G{G} n{n} past{past}", flush=True)
    L = past + n
    c = Cache(pkg, dev, "bf16", 1, dh, 64, [L], seed=211)
    g = torch.Generator().manual_seed(212)
    k, v = (torch.randn(L, 1, dh, generator=g).to(BF) for _ in range(2))
    q = torch.randn(n, G, dh, generator=g).to(BF)
    want, mag = _attend64(q, k.to(F64), v.to(F64), past, dh ** -0.5, 0, 0)
    bad = v.clone()
    bad[5, 0, 3] = bad[L - 1, 0, 21] = math.inf
    bad[70, 0, 9] = bad[L - 2, 0, 22] = -math.inf
    bad[130, 0, 11], bad[200, 0, 11] = math.inf, -math.inf
    bad[131, 0, 12] = math.nan
    want[..., 3], want[..., 9], want[..., 11], want[..., 12] = math.inf, -math.inf, math.nan, math.nan
    want[n - 1, :, 21] = math.inf                             # the last token's, which only it sees
    want[max(n - 2, 0):, :, 22] = -math.inf
    pkg.kv_write(c.pages, k.to(dev), bad.to(dev), c.table, c.len_t, _cu(dev, [L]))
    got = pkg.paged_attention(q.to(dev), c.pages, c.table, c.len_t, _cu(dev, [n]), max_new=n).cpu().to(F64)
    fine = torch.isfinite(want)
    assert ((got - want).abs() <= BAR * mag)[fine].all()
    assert torch.equal(got[~fine].nan_to_num(7.0, 1e300, -1e300), want[~fine].nan_to_num(7.0, 1e300, -1e300))


def _wide(c, width):
    """The table with unused entries behind it: calls of few tokens then take the
    kernel for many rows."""
    t = torch.full((c.table.shape[0], width), -1, dtype=I32, device=c.table.device)
    t[:, :c.table.shape[1]] = c.table
    return t


# single tokens, split over a long axis, 32 rows a workgroup, 128
SHAPES = [(1, 300, 1, 0), (1, 9001, 2, 0), (20, 300, 1, 0), (200, 300, 2, 400)]


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("n,past,G,width", SHAPES, ids=str)
@pytest.mark.parametrize("beside", [False, True], ids=["alone", "beside"])
def test_smallest_value_rows(pkg, dev, kind, n, past, G, width, beside):
    """Value rows from the smallest that is not held as zeros on, whose scales lie
    under 2^-100: attention reads them as they are read back.  Their weights'
    exponents are about 110, kept to 2^-18: within the bound's 3e-4."""
    print(f"[gpu] attention smallest value rows {kind} n{n} past{past} {beside}", flush=True)
    L = past + n
    c = Cache(pkg, dev, kind, 1, 64, 64, [L], seed=221)
    g = torch.Generator().manual_seed(222)
    k, v = (torch.randn(L, 1, 64, generator=g) for _ in range(2))
    v = v / v.abs().amax(-1, keepdim=True)
    size = torch.tensor([1.001 * 2.0 ** -100, 2.0 ** -99, 2.0 ** -95, 2.0 ** -92, 0.0])[torch.arange(L) % 5]
    if beside:
        size[::7] = 1.0
    v = v * size[:, None, None]
    q = torch.randn(n, G, 64, generator=g).to(BF)
    pkg.kv_write(c.pages, k.to(dev), v.to(dev), c.table, c.len_t, _cu(dev, [L]))
    table = _wide(c, width) if width else c.table
    got = pkg.paged_attention(q.to(dev), c.pages, table, c.len_t, _cu(dev, [n]), max_new=n).cpu().to(F64)
    kk, vv = c.held(0)
    want, mag = _attend64(q, kk, vv, past, 0.125, 0, 0)
    assert (mag > 0).all()
    err = ((got - want).abs() / mag).max()
    assert err <= BAR, float(err)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,past,G,width", SHAPES, ids=str)
@pytest.mark.parametrize("zero", [None, 0, 290], ids=str)
def test_scores_far_below_zero(pkg, dev, kind, n, past, G, width, zero):
    """Finite scores of -1.2e31 and -2.3e31 (in units of log2), alone and with one
    of zero among them: equal keys weigh the same, the others nothing."""
    print(f"[gpu] attention low scores {kind} n{n} past{past} {zero}", flush=True)
    L = past + n
    c = Cache(pkg, dev, kind, 1, 64, 64, [L], seed=231)
    g = torch.Generator().manual_seed(232)
    k = torch.full((L, 1, 64), 2.0 ** 50)
    k[1::3] *= 2
    if zero is not None:
        k[zero] = 0
    v = torch.randn(L, 1, 64, generator=g)
    q = torch.full((n, G, 64), -2.0 ** 50).to(BF)
    pkg.kv_write(c.pages, k.to(dev), v.to(dev), c.table, c.len_t, _cu(dev, [L]))
    table = _wide(c, width) if width else c.table
    got = pkg.paged_attention(q.to(dev), c.pages, table, c.len_t, _cu(dev, [n]), max_new=n).cpu().to(F64)
    kk, vv = c.held(0)
    kk = k.to(F64)                                           # 127 or 448 times a scale is off by a rounding, the same for all
    want, mag = _attend64(q, kk, vv, past, 0.125, 0, 0)
    assert ((got - want).abs() <= BAR * mag).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,past,G,width", SHAPES, ids=str)
@pytest.mark.parametrize("size", [3, 4, 6, 9, 12, 16, 18, 30, 50])
def test_equal_keys_weigh_the_same_at_any_size_of_scores(pkg, dev, kind, n, past, G, width, size):
    """Two groups of equal keys, at scores of 22 x 4^size (in units of log2) of
    either sign whose products take more bits than float32 holds: the larger
    group's members share the weight, in every tile, split and wave alike."""
    print(f"[gpu] attention scores of 22 x 4^{size} {kind} n{n} past{past}", flush=True)
    L = past + n
    c = Cache(pkg, dev, kind, 1, 64, 64, [L], seed=271)
    g = torch.Generator().manual_seed(272)
    k = torch.full((L, 1, 64), 1.5 * 2.0 ** size)
    k[1::3] = 1.25 * 2.0 ** size
    v = torch.randn(L, 1, 64, generator=g) * torch.exp(torch.randn(L, 1, 1, generator=g))
    pkg.kv_write(c.pages, k.to(dev), v.to(dev), c.table, c.len_t, _cu(dev, [L]))
    table = _wide(c, width) if width else c.table
    _, vv = c.held(0)
    for sign in (1, -1):
        q = torch.full((n, G, 64), sign * 1.25 * 2.0 ** size).to(BF)
        got = pkg.paged_attention(q.to(dev), c.pages, table, c.len_t, _cu(dev, [n]), max_new=n).cpu().to(F64)
        want, mag = _attend64(q, k.to(F64), vv, past, 0.125, 0, 0)
        err = ((got - want).abs() / mag).max()
        assert err <= BAR, (sign, float(err))


@pytest.mark.parametrize("sinks", [0, 4])
@pytest.mark.parametrize("width", [0, 2048])
def test_the_largest_window_hides_nothing(pkg, dev, sinks, width):
    """A window of 2^31 - 1, also for a call with rows before the first position."""
    print(f"[gpu] attention largest window sinks {sinks} width {width}", flush=True)
    n, L = 90, 80
    c = Cache(pkg, dev, "bf16", 1, 64, 64, [L], seed=241)
    g = torch.Generator().manual_seed(242)
    k, v = (torch.randn(L, 1, 64, generator=g).to(BF) for _ in range(2))
    q = torch.randn(n, 1, 64, generator=g).to(BF).to(dev)
    pkg.kv_write(c.pages, k.to(dev), v.to(dev), c.table, c.len_t, _cu(dev, [L]))
    table = _wide(c, width) if width else c.table
    want = pkg.paged_attention(q, c.pages, table, c.len_t, _cu(dev, [n]), max_new=n)
    assert (want[:10] == 0).all() and (want[10:] != 0).any(-1).all()
    for window in (1 << 20, (1 << 31) - 1):
        got = pkg.paged_attention(q, c.pages, table, c.len_t, _cu(dev, [n]), max_new=n, window=window, sinks=sinks)
        assert torch.equal(got, want), window


# -- what tensors the calls take ---------------------------------------------------

class _Nothing:
    """A native host side that takes no call."""

    def __getattr__(self, name):
        return lambda *args: None


@pytest.mark.parametrize("native", [True, False], ids=["native", "general"])
@pytest.mark.parametrize("T,H", [(1, 1), (1, 3), (5, 1)])
def test_odd_strides_of_single_tokens_and_heads(pkg, dev, monkeypatch, native, T, H):
    """The stride of a dimension of one element is no stride: slices of tensors of
    odd widths."""
    from dawn_srw_amd import kv
    print(f"[gpu] kv odd strides T{T} H{H}", flush=True)
    c = Cache(pkg, dev, "bf16", H, 64, 16, [T], seed=251)
    if not native:
        monkeypatch.setattr(kv, "_host", _Nothing())
    g = torch.Generator().manual_seed(252)
    wide = torch.randn(T, 3 * H * 64 + 3, generator=g).to(BF).to(dev)
    rows = [torch.as_strided(wide, (T, H, 64), (wide.stride(0), 64 if H > 1 else 67, 1), i * H * 64) for i in range(3)]
    cu = _cu(dev, [T])
    pkg.kv_write(c.pages, rows[0], rows[1], c.table, c.len_t, cu)
    for got, want in zip(pkg.kv_read(c.pages, c.table, c.len_t, cu, total=T), rows):
        assert torch.equal(got, want)
    got = pkg.paged_attention(rows[2], c.pages, c.table, c.len_t, cu)
    assert torch.equal(got, pkg.paged_attention(rows[2].clone(memory_format=torch.contiguous_format), c.pages, c.table,
                                                c.len_t, cu))


@pytest.mark.parametrize("native", [True, False], ids=["native", "general"])
def test_pages_of_another_shape_are_refused(pkg, dev, monkeypatch, native):
    """Tensors that got another shape after KvPages took them."""
    from dawn_srw_amd import kv
    print("[gpu] kv pages of another shape", flush=True)
    lens, table = torch.tensor([1], dtype=I32, device=dev), torch.tensor([[0]], dtype=I32, device=dev)
    for dh, P in ((128, 16), (64, 32)):
        pages = pkg.KvPages(torch.zeros(1, 1, 16, 64, dtype=BF, device=dev), torch.zeros(1, 1, 64, 16, dtype=BF, device=dev))
        pages.k.data, pages.v.data = (torch.zeros(s, dtype=BF, device=dev) for s in ((1, 1, P, dh), (1, 1, dh, P)))
        x = torch.ones(1, 1, dh, dtype=BF, device=dev)
        if not native:
            monkeypatch.setattr(kv, "_host", _Nothing())
        for call in (lambda: pkg.kv_write(pages, x, x, table, lens), lambda: pkg.kv_read(pages, table, lens),
                     lambda: pkg.paged_attention(x, pages, table, lens)):
            with pytest.raises(ValueError):
                call()


@pytest.mark.parametrize("native", [True, False], ids=["native", "general"])
def test_pages_and_tangents_that_want_gradients(pkg, dev, monkeypatch, native):
    """No gradient is dropped silently: neither of pages nor of forward mode."""
    from torch.autograd import forward_ad
    from dawn_srw_amd import kv
    print("[gpu] kv pages and tangents", flush=True)
    lens, table = torch.tensor([1], dtype=I32, device=dev), torch.tensor([[0]], dtype=I32, device=dev)
    k, v = (torch.zeros(s, dtype=BF, device=dev) for s in ((1, 1, 16, 64), (1, 1, 64, 16)))
    pages, x = pkg.KvPages(k, v), torch.ones(1, 1, 64, dtype=BF, device=dev)
    if not native:
        monkeypatch.setattr(kv, "_host", _Nothing())

    def refused(*calls):
        for call in calls:
            with pytest.raises(NotImplementedError):
                call()

    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        refused(lambda: pkg.kv_write(pages, d, x, table, lens), lambda: pkg.kv_write(pages, x, d, table, lens),
                lambda: pkg.paged_attention(d, pages, table, lens))
    pkg.kv_write(pages, x, x, table, lens)
    v.requires_grad_()
    refused(lambda: pkg.kv_write(pages, x, x, table, lens), lambda: pkg.kv_read(pages, table, lens),
            lambda: pkg.paged_attention(x, pages, table, lens))
    with torch.no_grad():
        assert torch.equal(pkg.paged_attention(x, pages, table, lens), x)


@pytest.mark.parametrize("native", [True, False], ids=["native", "general"])
@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_written_tensors_tell_their_version(pkg, dev, monkeypatch, native, kind):
    """What a call writes in place counts as changed: a gradient that was to use
    the old values is refused."""
    from dawn_srw_amd import kv
    print(f"[gpu] kv versions {kind}", flush=True)
    c = Cache(pkg, dev, kind, 1, 64, 16, [1], seed=261)
    if not native:
        monkeypatch.setattr(kv, "_host", _Nothing())
    x = torch.ones(1, 1, 64, dtype=BF, device=dev)
    held = [t for t in (c.pages.k, c.pages.v, c.pages.k_scale, c.pages.v_scale) if t is not None]
    before = [t._version for t in held]
    pkg.kv_write(c.pages, x, x, c.table, c.len_t)
    assert all(t._version > b for t, b in zip(held, before))
    out = torch.zeros(1, 1, 64, dtype=BF, device=dev)
    pkg.kv_read(c.pages, c.table, c.len_t)
    before = [t._version for t in (*held, out)]
    pkg.paged_attention(x, c.pages, c.table, c.len_t, out=out)
    assert [t._version for t in held] == before[:-1] and out._version > before[-1]
    w = torch.ones(1, 1, 64, device=dev, requires_grad=True)
    y = (w * out.float()).sum() + (w * out).sum()
    pkg.paged_attention(x, c.pages, c.table, c.len_t, out=out)
    with pytest.raises(RuntimeError):
        y.backward()
    with torch.inference_mode():                              # which keeps no versions
        other = pkg.KvPages(*(None if t is None else t.clone() for t in (c.pages.k, c.pages.v, c.pages.k_scale, c.pages.v_scale)))
        pkg.kv_write(other, x, x, c.table, c.len_t)
        pkg.paged_attention(x, other, c.table, c.len_t, out=torch.zeros_like(x))
