"""CPU: the host side of page copies, the pages' index and choice, attention to kept
pages and sampling -- C descriptions, the checks that return before any launch,
workspace sizes, and the bookkeeping of sequences that share pages."""

from __future__ import annotations

import ctypes
import os
import random
import subprocess

import pytest
import torch

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "srw_amd.h")


@pytest.fixture(scope="module")
def C(pkg):
    from dawn_srw_amd import _capi
    _capi.load_library()
    return _capi


def test_layouts_match_the_header(C, tmp_path):
    from dawn_srw_amd import kv, sampling
    structs = {"srw_kv_copy_t": C.SrwKvCopy, "srw_kv_index_t": C.SrwKvIndex, "srw_kv_select_t": C.SrwKvSelect,
               "srw_sample_t": C.SrwSample}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "srw_amd.h"', "int main(void){"]
    for name, cls in structs.items():
        lines.append(f'printf("{name} - %zu\\n", sizeof({name}));')
        for f, *_ in cls._fields_:
            lines.append(f'printf("{name} {f} %zu\\n", offsetof({name}, {f}));')
    lines.append('printf("tensors - %d\\n", SRW_KV_COPY_TENSORS);')
    lines.append("return 0;}")
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.dirname(HEADER), str(src), "-o", str(exe)],
                   check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n"):
        if line:
            name, f, n = line.split()
            if name == "tensors":
                assert int(n) == C.COPY_TENSORS
                continue
            cls = structs[name]
            assert int(n) == (ctypes.sizeof(cls) if f == "-" else getattr(cls, f).offset), line
    # the packed forms are the same bytes
    at = tuple(range(1, 17))
    assert kv._INDEX.pack(1, 2) == bytes(C.SrwKvIndex(1, 2))
    assert kv._SELECT.pack(*at, *range(17, 27)) == bytes(
        C.SrwKvSelect(C.SrwKv(*at), C.SrwKvIndex(17, 18), *range(19, 27)))
    n = C.COPY_TENSORS
    rows = [tuple(range(n * i, n * i + n)) for i in range(5)]
    as_arrays = [(ctypes.c_void_p * n)(*r) for r in rows[:2]] + [(ctypes.c_int64 * n)(*r) for r in rows[2:]]
    assert kv._COPY.pack(*range(5 * n), 3, 4, 5, 6, 7, 8, 9, 0) == bytes(C.SrwKvCopy(*as_arrays, 3, 4, 5, 6, 7, 8, 9, 0))
    rest = (0.5, 0.25, 0.125, 7, 1, 0)
    assert sampling._SAMPLE.pack(*range(1, 12), *rest) == bytes(C.SrwSample(*range(1, 12), *rest))


def _kv(C, **kw):
    f = dict(k=4096, v=4096, k_scale=4096, v_scale=4096, table=4096, lens=4096, cu=4096, B=2, T=5, n_pages=8,
             table_width=3, table_stride=3, n_kv_heads=2, head_dim=64, page_size=16, kind=C.SRW_KV_INT8)
    f.update(kw)
    return C.SrwKv(**f)


# -- what each entry point refuses before a launch ----------------------------------

def _copy(C, **kw):
    """Two tensors at made-up addresses, three pairs; nothing reads them on the host but
    the lists of pages."""
    f = dict(src=[1 << 20, 1 << 24], dst=[1 << 20, 1 << 24], page_bytes=[64, 4], src_layer_stride=[6400, 400],
             dst_layer_stride=[6400, 400], n_layers=2, n_src_pages=100, n_dst_pages=100, n_tensors=2,
             src_page=[0, 1, 1], dst_page=[2, 3, 4])
    f.update(kw)
    c, keep = C.SrwKvCopy(), []
    for name in ("src", "dst", "page_bytes", "src_layer_stride", "dst_layer_stride"):
        for i, x in enumerate(f[name]):
            getattr(c, name)[i] = x
    for name in ("src_page", "dst_page"):
        if f[name] is not None:
            a = (ctypes.c_int32 * max(1, len(f[name])))(*f[name])
            keep.append(a)
            setattr(c, name, ctypes.addressof(a))
    c.n_pairs = f.get("n_pairs", len(f["src_page"] or ()))
    for name in ("n_layers", "n_src_pages", "n_dst_pages", "n_tensors"):
        setattr(c, name, f[name])
    return c, keep


MANY = list(range(40))
COPY_BAD = [dict(n_tensors=9), dict(n_tensors=-1), dict(n_layers=-1), dict(n_src_pages=-1), dict(n_dst_pages=-1),
            dict(n_pairs=-1), dict(n_pairs=101), dict(src_page=None, n_pairs=3), dict(page_bytes=[64, 6]),
            dict(page_bytes=[0, 4]), dict(src=[(1 << 20) + 2, 1 << 24]), dict(src_layer_stride=[6396, 400]),
            dict(src_layer_stride=[6402, 400]), dict(src_page=[0, 1, 100]), dict(src_page=[0, -1, 1]),
            dict(dst_page=[2, 3, 100]), dict(dst_page=[2, 3, -1]), dict(dst_page=[2, 3, 2]), dict(src_page=[0, 2, 1]),
            dict(src_page=[2, 0, 1], dst_page=[2, 3, 4]),                            # onto itself
            dict(src_page=MANY, dst_page=[40 + i for i in MANY[:39]] + [40]),         # twice, many
            dict(src_page=MANY, dst_page=[40 + i for i in MANY[:39]] + [7]),          # read and written, many
            dict(dst=[(1 << 20) + 64, 1 << 24]), dict(dst=[1 << 21, (1 << 20) + 128]),   # tensors that meet
            dict(src=[1 << 20, 1 << 21], dst=[1 << 22, (1 << 22) + 64])]


@pytest.mark.parametrize("change", COPY_BAD, ids=str)
def test_copies_are_checked(C, change):
    c, keep = _copy(C, **change)
    assert C.load_library().srw_kv_copy(ctypes.byref(c), None) == C.SRW_EINVAL


def test_copies_of_nothing_and_beyond_the_limits(C):
    lib = C.load_library()
    for change in (dict(src_page=[], dst_page=[]), dict(n_layers=0), dict(n_tensors=0)):
        c, keep = _copy(C, **change)
        assert lib.srw_kv_copy(ctypes.byref(c), None) == C.SRW_OK
    for change in (dict(n_layers=65536), dict(n_dst_pages=1 << 31), dict(n_src_pages=1 << 31),
                   dict(page_bytes=[(1 << 30) + 4, 4])):
        c, keep = _copy(C, **change)
        assert lib.srw_kv_copy(ctypes.byref(c), None) == C.SRW_EUNSUPPORTED
    assert lib.srw_kv_copy(None, None) == C.SRW_EINVAL


def test_the_index_is_checked(C):
    lib = C.load_library()

    def call(codes=4096, scale=4096, **kw):
        return lib.srw_kv_index(ctypes.byref(_kv(C, **kw)), ctypes.byref(C.SrwKvIndex(codes, scale)), None)

    assert call(codes=4104) == call(scale=4098) == call(codes=None) == call(scale=None) == C.SRW_EINVAL
    assert call(B=-1) == call(lens=None) == call(k=None) == C.SRW_EINVAL
    assert call(head_dim=96) == call(page_size=8) == call(T=(1 << 29) + 1) == C.SRW_EUNSUPPORTED
    assert call(T=0) == call(n_pages=0) == C.SRW_OK
    assert lib.srw_kv_index(None, None, None) == C.SRW_EINVAL
    assert lib.srw_kv_index(ctypes.byref(_kv(C)), None, None) == C.SRW_EINVAL


def test_the_choice_is_checked(C):
    lib = C.load_library()

    def call(kv={}, codes=4096, **kw):
        f = dict(q=4096, keep=4096, q_token_stride=256, q_head_stride=64, n_heads=4, n=3, first=1, last=1)
        f.update(kw)
        return lib.srw_kv_select(ctypes.byref(C.SrwKvSelect(kv=_kv(C, **kv), index=C.SrwKvIndex(codes, 4096), **f)), None)

    for bad in (dict(q=4100), dict(keep=4098), dict(q_token_stride=-4), dict(q_head_stride=62), dict(q_token_stride=2),
                dict(n_heads=0), dict(n_heads=3), dict(n=0), dict(first=-1), dict(last=0), dict(first=2, last=2),
                dict(first=0x7fffffff, last=0x7fffffff), dict(codes=4100), dict(kv=dict(table=None))):
        assert call(**bad) == C.SRW_EINVAL, bad
    assert call(kv=dict(T=1 << 22)) == call(kv=dict(head_dim=80)) == C.SRW_EUNSUPPORTED
    assert call(kv=dict(T=0)) == C.SRW_OK
    assert lib.srw_kv_select(None, None) == C.SRW_EINVAL


def test_attention_to_kept_pages_is_checked(C):
    lib, n = C.load_library(), ctypes.c_size_t(7)

    def a(kv={}, **kw):
        f = dict(q=4096, out=4096, q_token_stride=256, q_head_stride=64, n_heads=4, scale=0.125)
        f.update(kw)
        return C.SrwAttention(kv=_kv(C, **kv), **f)

    def size(n_keep, **kw):
        return lib.srw_attention_kept_workspace_size(ctypes.byref(a(**kw)), n_keep, ctypes.byref(n))

    def run(keep, n_keep, **kw):
        return lib.srw_attention_kept(ctypes.byref(a(**kw)), keep, n_keep, None, 0, None)

    for bad in (dict(window=8), dict(window=8, sinks=1), dict(n_heads=3), dict(max_new=-1), dict(scale=float("nan")),
                dict(kv=dict(lens=None))):
        assert size(4, **bad) == run(4096, 4, **bad) == C.SRW_EINVAL, bad
    assert size(0) == size(-1) == run(4096, 0) == C.SRW_EINVAL
    assert run(None, 4) == run(4098, 4) == run(4096, 4, q=4100) == run(4096, 4, q_head_stride=60) == C.SRW_EINVAL
    assert size(4, kv=dict(T=0)) == C.SRW_OK and n.value == 0 and run(4096, 4, kv=dict(T=0)) == C.SRW_OK
    assert size(1 << 40) != C.SRW_OK
    assert lib.srw_attention_kept_workspace_size(ctypes.byref(a()), 4, None) == C.SRW_EINVAL
    # few rows over long lists: four tiles of 64 positions a split, a float2 and head_dim
    # floats for each row of each; the launch waits for the workspace
    one = dict(kv=dict(B=1, T=1, cu=None, page_size=64, table_width=500, table_stride=500))
    assert size(100, **one) == C.SRW_OK
    al = lambda b: (b + 255) // 256 * 256  # noqa: E731
    assert n.value == al(25 * 4 * 8) + al(25 * 4 * 64 * 4)
    assert run(4096, 100, **one) == C.SRW_EWORKSPACE
    many = dict(kv=dict(B=128, T=128, cu=None, page_size=64, table_width=500, table_stride=500))
    assert size(100, **many) == C.SRW_OK and n.value == 0


def _sample(C, **kw):
    f = dict(logits=4096, row_stride=100, B=2, V=100, u=4096, token=4096, logprob=4096, temperature_all=1.0, top_p_all=1.0,
             min_p_all=0.0, top_k_all=0, dtype=C.SRW_F32)
    f.update(kw)
    return C.SrwSample(**f)


def test_sampling_is_checked(C):
    lib, n = C.load_library(), ctypes.c_size_t(7)

    def size(**kw):
        return lib.srw_sample_workspace_size(ctypes.byref(_sample(C, **kw)), ctypes.byref(n))

    def run(**kw):
        return lib.srw_sample(ctypes.byref(_sample(C, **kw)), None, 0, None)

    nan = float("nan")
    for bad in (dict(B=-1), dict(V=0), dict(V=-4), dict(dtype=5), dict(logits=None), dict(logits=4098), dict(u=None),
                dict(u=4097), dict(token=None), dict(token=4100), dict(logprob=4098), dict(temperature=4098),
                dict(top_k=4098), dict(top_p=4097), dict(min_p=4098), dict(row_stride=-1), dict(temperature_all=-0.5),
                dict(temperature_all=nan), dict(top_k_all=-1), dict(top_p_all=1.5), dict(top_p_all=nan),
                dict(min_p_all=-0.1), dict(min_p_all=nan)):
        assert size(**bad) == run(**bad) == C.SRW_EINVAL, bad
    for far in (dict(B=(1 << 21) + 1), dict(V=(1 << 24) + 1), dict(B=1 << 14, V=1 << 24)):
        assert size(**far) == run(**far) == C.SRW_EUNSUPPORTED, far
    assert size(B=0) == run(B=0) == C.SRW_OK
    assert lib.srw_sample_workspace_size(ctypes.byref(_sample(C)), None) == C.SRW_EINVAL
    assert lib.srw_sample(None, None, 0, None) == C.SRW_EINVAL
    # a large vocabulary from the whole distribution: the parts' sums, no launch without
    big = dict(V=100000, row_stride=100000)
    assert size(**big) == C.SRW_OK and n.value > 0 and run(**big) == C.SRW_EWORKSPACE
    assert size(V=1000) == C.SRW_OK and n.value == 0


def test_python_refusals(pkg):
    """What the Python entry points say of tensors off the device and of bad numbers."""
    z = torch.zeros
    with pytest.raises(ValueError):
        pkg.sample(z(2, 5), z(2))
    with pytest.raises(ValueError):
        pkg.sample(z(5), z(2))
    with pytest.raises(ValueError):
        pkg.sample(None, z(2))
    for tensors, src, dst, to in (([z(1, 2, 3)], [0], [1], None), ([], [0], [1], None), ([z(1, 2, 4)] * 9, [0], [1], None),
                                  ([z(1, 2, 4)], [0, 1], [1], None), ([z(1, 2, 4)], [1 << 40], [1], None),
                                  ([z(1, 2, 4)], [0], [1], [z(1, 2, 4)] * 2)):
        with pytest.raises(ValueError):
            pkg.kv_copy(tensors, src, dst, to=to)
    with pytest.raises(TypeError):
        pkg.kv_copy([z(1, 2, 4)], torch.tensor([0]), [1])
    with pytest.raises(TypeError):
        pkg.kv_copy([z(1, 2, 4)], [0.5], [1])
    with pytest.raises((TypeError, ValueError)):
        pkg.KvIndex(z(4, 2, 64), z(4, 2))
    with pytest.raises(ValueError):
        pkg.PagedKvCache(1, 4, 1, 64, device="cpu").index(0)


# -- sequences that share pages ------------------------------------------------------

def _copied(log=None):
    def copy(tensors, src, dst, *, to=None):
        src, dst = list(src), list(dst)
        assert len(src) == len(dst) and len(set(dst)) == len(dst)
        if to is None:
            assert not set(src) & set(dst)
        for x, y in zip(tensors, tensors if to is None else to):
            y[:, dst] = x[:, src]
        if log is not None:
            log.append((src, dst))
    return copy


class Model:
    """What each sequence should hold, beside a cache whose k[0, page, 0, slot, 0] holds
    it."""

    def __init__(self, cache):
        self.c, self.has, self.next = cache, {}, 0

    def write(self, seqs, counts):
        table, lens, cu, most = self.c.extend(seqs, counts)
        for b, (s, n) in enumerate(zip(seqs, counts)):
            assert int(lens[b]) == len(self.has[s]) + n
            for _ in range(n):
                i = len(self.has[s])
                self.c.k[:, int(table[b, i // self.c.page_size]), 0, i % self.c.page_size, 0] = self.next
                self.has[s].append(self.next)
                self.next += 1

    def check(self):
        held = set()
        for s, want in self.has.items():
            pages, P = self.c._pages[s], self.c.page_size
            assert self.c.length(s) == len(want) and len(pages) == -(-len(want) // P)
            held.update(pages)
            for layer in range(2):
                got = [int(self.c.k[layer, pages[i // P], 0, i % P, 0]) for i in range(len(want))]
                assert got == want
        # every page free or held, and counted as often as it is held
        assert held.isdisjoint(self.c._free) and len(held) + len(self.c._free) == self.c.n_pages
        for p in held:
            times = sum(pages.count(p) for pages in self.c._pages.values())
            assert times == 1 + self.c._more.get(p, 0)
        assert set(self.c._more) <= held


@pytest.mark.parametrize("seed", range(6))
def test_shared_pages_hold_what_each_sequence_wrote(pkg, monkeypatch, seed):
    """Random forks, writes, frees, moves and sizes."""
    from dawn_srw_amd import kv
    monkeypatch.setattr(kv, "kv_copy", _copied())
    rng = random.Random(seed)
    c = pkg.PagedKvCache(2, 40, 1, 64, page_size=16, dtype=torch.float8_e4m3fn if seed % 2 else torch.bfloat16,
                         device="cpu", indexed=seed % 3 == 0)
    c.k = torch.zeros(2, 40, 1, 16, 64, dtype=torch.int64)     # (whole numbers of any size, in place of keys)
    new = c._new
    c._new = lambda n: [torch.zeros(2, n, 1, 16, 64, dtype=torch.int64)] + new(n)[1:]
    m = Model(c)
    for _ in range(150):
        what = rng.random()
        seqs = list(m.has)
        if what < 0.15 or not seqs:
            s = c.add()
            m.has[s] = []
        elif what < 0.35:
            s = rng.choice(seqs)
            m.has[c.fork(s)] = list(m.has[s])
        elif what < 0.75:
            some = rng.sample(seqs, rng.randint(1, min(4, len(seqs))))
            counts = [rng.choice([0, 1, 1, 5, 16, 23]) for _ in some]
            before = (dict(c._lens), {s: list(p) for s, p in c._pages.items()}, list(c._free), dict(c._more))
            try:
                m.write(some, counts)
            except MemoryError:
                assert before == (c._lens, c._pages, c._free, c._more)
        elif what < 0.9:
            s = rng.choice(seqs)
            c.free(s)
            del m.has[s]
        elif what < 0.95:
            c.compact()
            held = c._held()
            assert held == list(range(len(held)))
        else:
            n = rng.randint(1, 60)
            if n < len(c._held()):
                with pytest.raises(MemoryError):
                    c.resize(n)
            else:
                c.resize(n)
                assert c.n_pages == n and c.k.shape[1] == n
        m.check()
    for s in list(m.has):
        c.free(s)
    assert c.free_pages == c.n_pages and not c._more


def test_a_partial_page_is_copied_for_the_first_writer_alone(pkg, monkeypatch):
    from dawn_srw_amd import kv
    log = []
    monkeypatch.setattr(kv, "kv_copy", _copied(log))
    c = pkg.PagedKvCache(2, 10, 1, 64, page_size=16, device="cpu")
    a = c.add()
    c.extend([a], [20])
    b = c.fork(a)
    assert c.free_pages == 8 and c.length(b) == 20
    c.extend([a, b], [1, 1])         # one copy, the other keeps the page
    assert len(log) == 1 and len(log[0][0]) == 1 and c.free_pages == 7 and not set(c._pages[a][1:]) & set(c._pages[b][1:])
    c.extend([a, b], [1, 1])
    assert len(log) == 1
    d = c.fork(a)
    c.extend([d], [0])               # nothing new, no copy
    assert len(log) == 1
    c.free(a)
    c.extend([d], [1])               # its last holder writes in place
    assert len(log) == 1
    e = c.add()
    c.extend([e], [32])
    f = c.fork(e)
    c.extend([f], [1])               # full pages are only read
    assert len(log) == 1 and c._pages[f][:2] == c._pages[e]


def test_a_failed_extend_of_shared_pages_changes_nothing(pkg, monkeypatch):
    from dawn_srw_amd import kv
    monkeypatch.setattr(kv, "kv_copy", _copied())
    c = pkg.PagedKvCache(1, 8, 1, 64, page_size=16, device="cpu")
    a = c.add()
    c.extend([a], [20])
    b, d = c.fork(a), c.fork(a)

    def state():
        return dict(c._lens), {s: list(p) for s, p in c._pages.items()}, list(c._free), dict(c._more)

    before = state()
    with monkeypatch.context() as m:
        m.setattr(torch, "tensor", lambda *x, **kw: (_ for _ in ()).throw(RuntimeError("no memory")))
        with pytest.raises(RuntimeError):
            c.extend([a, b, d], [13, 40, 1])
    assert before == state()
    with monkeypatch.context() as m:
        m.setattr(kv, "kv_copy", lambda *x, **kw: (_ for _ in ()).throw(RuntimeError("no launch")))
        for call in (lambda: c.extend([a, b], [1, 1]), c.compact, lambda: c.resize(20)):
            with pytest.raises(RuntimeError):
                call()
    assert before == state() and c.n_pages == 8
    with pytest.raises(MemoryError):
        c.extend([a, b, d], [13, 70, 40])
    assert before == state()
    c.extend([a, b, d], [1, 1, 1])
    assert c.free_pages == 4


def test_forks_and_evicted_pages(pkg):
    c = pkg.PagedKvCache(1, 12, 1, 64, page_size=16, device="cpu")
    a = c.add()
    c.extend([a], [64])
    b = c.fork(a)
    assert c.evict(a, 16, 0) == 3 and c.free_pages == 8     # b holds them still
    assert c._pages[b] == [p for p in c._pages[b] if p >= 0]
    assert c.evict(b, 32) == 2 and c.free_pages == 10
    d = c.fork(a)                                           # with its gaps
    c.free(a)
    c.free(b)
    assert c.free_pages == 11
    c.free(d)
    assert c.free_pages == 12
    with pytest.raises(KeyError):
        c.fork(a)
    with pytest.raises(ValueError):
        c.resize(0)


@pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc")
def test_entry_points_clean_under_sanitizers():
    """Address and undefined-behaviour sanitizers over the host code up to the ends of the
    fields (tests/serving/serving_sanitize.c)."""
    folder = os.path.join(os.path.dirname(os.path.abspath(__file__)), "serving")
    build = subprocess.run(["make", "-C", folder, "-j4"], capture_output=True, text=True)
    assert build.returncode == 0, build.stdout[-2000:] + build.stderr[-2000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:abort_on_error=1:verify_asan_link_order=0",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    run = subprocess.run([os.path.join(folder, "_build", "serving_sanitize")], capture_output=True, text=True, env=env,
                         timeout=300)
    out = run.stdout + run.stderr
    assert run.returncode == 0 and " 0 failures" in out, out[-4000:]
    assert "runtime error" not in out and "AddressSanitizer" not in out
