"""CPU: the paged cache's host side -- the C descriptions, the argument checks
that return before any launch, and the pages' bookkeeping."""

from __future__ import annotations

import ctypes
import os
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
    from dawn_srw_amd import kv
    structs = {"srw_kv_t": C.SrwKv, "srw_kv_rows_t": C.SrwKvRows, "srw_attention_t": C.SrwAttention}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "srw_amd.h"', "int main(void){"]
    for name, cls in structs.items():
        lines.append(f'printf("{name} - %zu\\n", sizeof({name}));')
        for f, *_ in cls._fields_:
            lines.append(f'printf("{name} {f} %zu\\n", offsetof({name}, {f}));')
    lines.append("return 0;}")
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.dirname(HEADER), str(src), "-o", str(exe)],
                   check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n"):
        if line:
            name, f, n = line.split()
            cls = structs[name]
            assert int(n) == (ctypes.sizeof(cls) if f == "-" else getattr(cls, f).offset), line
    # the packed forms are the same bytes
    at = tuple(range(1, 17))
    assert kv._KV.pack(*at) == bytes(C.SrwKv(*at))
    assert kv._ROWS.pack(*at[:6]) == bytes(C.SrwKvRows(*at[:6]))
    rest = (17, 18, 19, 20, 21, 22, 23, 24, 0.5)
    assert kv._ATTENTION.pack(*at, *rest) == bytes(C.SrwAttention(C.SrwKv(*at), *rest))


def _kv(C, **kw):
    f = dict(k=4096, v=4096, k_scale=4096, v_scale=4096, table=4096, lens=4096, cu=4096, B=2, T=5, n_pages=8,
             table_width=3, table_stride=3, n_kv_heads=2, head_dim=64, page_size=16, kind=C.SRW_KV_INT8)
    f.update(kw)
    return C.SrwKv(**f)


BAD = [dict(B=-1), dict(T=-1), dict(n_pages=-1), dict(table_width=-1), dict(n_kv_heads=0), dict(kind=7),
       dict(head_dim=0), dict(page_size=0), dict(B=0), dict(cu=None), dict(table=None), dict(table_stride=2),
       dict(lens=None), dict(lens=4098), dict(cu=4098), dict(k=None), dict(v=4104), dict(k_scale=None),
       dict(v_scale=4100)]
UNSUPPORTED = [dict(head_dim=96), dict(head_dim=32), dict(page_size=24), dict(page_size=8), dict(page_size=512),
               dict(table_width=1 << 28, table_stride=1 << 28), dict(T=1 << 31), dict(n_pages=1 << 31),
               dict(B=1 << 25), dict(n_kv_heads=70000)]


@pytest.mark.parametrize("change", BAD + UNSUPPORTED, ids=str)
def test_descriptions_are_checked(C, change):
    want = C.SRW_EINVAL if change in BAD else C.SRW_EUNSUPPORTED
    lib, c = C.load_library(), _kv(C, **change)
    rows = C.SrwKvRows(4096, 4096, 128, 64, 128, 64)
    assert lib.srw_kv_write(ctypes.byref(c), ctypes.byref(rows), C.SRW_BF16, None) == want
    assert lib.srw_kv_read(ctypes.byref(c), ctypes.byref(rows), C.SRW_F32, None) == want
    a = C.SrwAttention(c, 4096, 4096, 256, 64, 4, 0, 0, 0, 1.0)
    n = ctypes.c_size_t(7)
    assert lib.srw_attention_workspace_size(ctypes.byref(a), ctypes.byref(n)) == want and n.value == 7
    assert lib.srw_attention(ctypes.byref(a), None, 0, None) == want


def test_rows_and_queries_are_checked(C):
    lib, c = C.load_library(), _kv(C)
    for rows, dtype in [((None, 4096, 128, 64, 128, 64), C.SRW_BF16), ((4096, 4100, 128, 64, 128, 64), C.SRW_BF16),
                        ((4096, 4104, 128, 64, 128, 64), C.SRW_F32), ((4096, 4096, 126, 64, 128, 64), C.SRW_BF16),
                        ((4096, 4096, 128, 64, -128, 64), C.SRW_BF16), ((4096, 4096, 128, 64, 128, 64), 5)]:
        r = C.SrwKvRows(*rows)
        for f in (lib.srw_kv_write, lib.srw_kv_read):
            assert f(ctypes.byref(c), ctypes.byref(r), dtype, None) == C.SRW_EINVAL
    assert lib.srw_kv_write(ctypes.byref(c), None, C.SRW_BF16, None) == C.SRW_EINVAL
    assert lib.srw_kv_write(None, None, C.SRW_BF16, None) == C.SRW_EINVAL
    ok = dict(q=4096, out=4096, q_token_stride=256, q_head_stride=64, n_heads=4, max_new=0, window=0, sinks=0, scale=1.0)
    for change in (dict(q=None), dict(out=4104), dict(q_token_stride=252), dict(q_head_stride=-64), dict(n_heads=3),
                   dict(n_heads=0), dict(max_new=-1), dict(window=-1), dict(sinks=4), dict(window=5, sinks=-1),
                   dict(scale=float("nan"))):
        a = C.SrwAttention(kv=c, **{**ok, **change})
        assert lib.srw_attention(ctypes.byref(a), None, 0, None) == C.SRW_EINVAL, change
    a = C.SrwAttention(kv=_kv(C, T=1 << 30), **{**ok, "n_heads": 8})
    n = ctypes.c_size_t(0)
    assert lib.srw_attention_workspace_size(ctypes.byref(a), ctypes.byref(n)) == C.SRW_EUNSUPPORTED
    # no tokens: nothing to do, nothing looked at
    a = C.SrwAttention(kv=_kv(C, T=0, lens=None, table=None), **{**ok, "q": None})
    assert lib.srw_attention(ctypes.byref(a), None, 0, None) == C.SRW_OK
    assert lib.srw_attention_workspace_size(ctypes.byref(a), ctypes.byref(n)) == C.SRW_OK and n.value == 0


def test_workspace_of_splits(C):
    """Few rows over a long table: partial results of every split, a float2 and
    head_dim floats for each row; many rows: none."""
    lib, n = C.load_library(), ctypes.c_size_t(0)
    long = dict(kind=C.SRW_KV_BF16, page_size=64, table_width=1000, table_stride=1000, T=1, B=1, cu=None)
    a = C.SrwAttention(kv=_kv(C, **long), q=4096, out=4096, q_token_stride=128, q_head_stride=64, n_heads=2, scale=1.0)
    assert lib.srw_attention_workspace_size(ctypes.byref(a), ctypes.byref(n)) == C.SRW_OK
    S = 250   # four of the 1000 tiles each
    al = lambda b: (b + 255) // 256 * 256  # noqa: E731
    assert n.value == al(S * 2 * 8) + al(S * 2 * 64 * 4)
    a.kv.table_width = a.kv.table_stride = 8
    assert lib.srw_attention_workspace_size(ctypes.byref(a), ctypes.byref(n)) == C.SRW_OK and n.value == 0


# -- bookkeeping -----------------------------------------------------------------

def test_pages_are_handed_out_and_back(pkg):
    c = pkg.PagedKvCache(2, 6, 3, 64, page_size=16, dtype=torch.int8, device="cpu")
    assert c.k.shape == (2, 6, 3, 16, 64) and c.v.shape == (2, 6, 3, 64, 16) and c.k_scale.shape == (2, 6, 3, 16)
    a, b = c.add(), c.add()
    table, lens, cu, most = c.extend([a, b], [17, 16])
    assert table.shape == (2, 2) and lens.tolist() == [17, 16] and cu.tolist() == [0, 17, 33] and most == 17
    used = [p for p in table.flatten().tolist() if p >= 0]
    assert len(set(used)) == 3 and table[1, 1] == -1 and c.free_pages == 3
    table2, lens, cu, most = c.extend([b, a], [1, 1])
    assert cu is None and most == 1 and lens.tolist() == [17, 18]
    assert table2[1].tolist() == table[0].tolist() and table2[0, 0] == table[1, 0] and c.free_pages == 2
    before = (c.length(a), c.length(b), c.free_pages)
    with pytest.raises(MemoryError):
        c.extend([a, b], [16, 64])
    with pytest.raises(ValueError):
        c.extend([a, a], [1, 1])
    with pytest.raises(ValueError):
        c.extend([a], [-1])
    with pytest.raises(KeyError):
        c.extend([a, 99], [1, 1])
    assert before == (c.length(a), c.length(b), c.free_pages)
    c.free(a)
    assert c.free_pages == 4 and c.length(b) == 17
    with pytest.raises(KeyError):
        c.length(a)
    d = c.add()
    assert d not in (a, b)
    _, lens, cu, most = c.extend([b, d], [0, 3])
    assert lens.tolist() == [17, 3] and cu.tolist() == [0, 0, 3]


def test_evict_keeps_what_a_later_token_sees(pkg):
    for n in (1, 16, 31, 32, 33, 100, 160):
        for window in (1, 15, 16, 17, 40, 200):
            for sinks in (0, 1, 16, 17):
                c = pkg.PagedKvCache(1, 12, 1, 64, page_size=16, device="cpu")
                a = c.add()
                c.extend([a], [n])
                gone = c.evict(a, window, sinks)
                table = c.extend([a], [1])[0][0].tolist()
                lost = [p for p in range(n) if table[p // 16] < 0]
                # a token at position n or later
                assert all(p <= n - window and p >= sinks for p in lost)
                assert len(lost) == 16 * gone
                rest = [i for i in range(-(-n // 16)) if table[i] >= 0]
                assert all((i + 1) * 16 > n - window + 1 or i * 16 < sinks for i in rest)
                c.free(a)
                assert c.free_pages == 12


def test_cache_refusals(pkg):
    for kw in (dict(head_dim=96), dict(page_size=24), dict(n_pages=0)):
        args = dict(n_layers=1, n_pages=4, n_heads=1, head_dim=64, page_size=16)
        args.update(kw)
        with pytest.raises(ValueError):
            pkg.PagedKvCache(args["n_layers"], args["n_pages"], args["n_heads"], args["head_dim"],
                             page_size=args["page_size"], device="cpu")
    with pytest.raises(TypeError):
        pkg.PagedKvCache(1, 4, 1, 64, dtype=torch.float16, device="cpu")
    c = pkg.PagedKvCache(1, 4, 1, 64, page_size=16, device="cpu")
    with pytest.raises(ValueError):
        c.layer(0)                     # the calls run on a HIP device
    with pytest.raises(ValueError):
        c.evict(c.add(), 0)


def test_a_failed_extend_changes_nothing(pkg, monkeypatch):
    """A copy to the device that fails (no memory) after pages were handed out."""
    c = pkg.PagedKvCache(1, 8, 1, 64, page_size=16, device="cpu")
    a, b = c.add(), c.add()
    c.extend([a], [20])
    before = (dict(c._lens), {s: list(p) for s, p in c._pages.items()}, list(c._free))
    with monkeypatch.context() as m:
        m.setattr(torch, "tensor", lambda *x, **kw: (_ for _ in ()).throw(RuntimeError("no memory")))
        with pytest.raises(RuntimeError):
            c.extend([a, b], [13, 40])
    assert before == (c._lens, c._pages, c._free)
    table, lens, _, _ = c.extend([a, b], [13, 40])
    assert lens.tolist() == [33, 40] and len({p for p in table.flatten().tolist() if p >= 0}) == 6


def test_plans_of_calls(C):
    """Rows a workgroup and splits: single tokens, short and long chunks."""
    lib = C.load_library()

    def plan(max_new, window=0, sinks=0, **kw):
        f = dict(kind=C.SRW_KV_BF16, page_size=64, B=1)
        f.update(kw)
        f["table_stride"] = f["table_width"]
        a = C.SrwAttention(_kv(C, **f), 4096, 4096, 256, 64, 4, max_new, window, sinks, 1.0)
        rows, splits = ctypes.c_int32(-1), ctypes.c_int32(-1)
        assert lib.srw_attention_plan(ctypes.byref(a), ctypes.byref(rows), ctypes.byref(splits)) == C.SRW_OK
        return rows.value, splits.value

    assert plan(0, T=0, table_width=8) == (0, 0)
    assert plan(1, T=1, cu=None, table_width=8) == (16, 1)
    assert plan(1, T=1, cu=None, table_width=1000)[0] == 16 and plan(1, T=1, cu=None, table_width=1000)[1] > 1
    assert plan(16, T=16, table_width=8) == (32, 1)
    assert plan(300, T=300, table_width=8) == (32, 1)              # 1 200 rows of 8 tiles: too few for 128 each
    assert plan(4000, T=4000, table_width=12) == (128, 1)
    assert plan(300, T=300, table_width=1000)[0] == 128 and plan(300, T=300, table_width=1000)[1] > 1
    assert plan(300, T=300, table_width=1000, window=100) == (32, 1)
    a = C.SrwAttention(_kv(C), 4096, 4096, 256, 64, 4, 0, 0, 0, 1.0)
    n = ctypes.c_int32(0)
    assert lib.srw_attention_plan(ctypes.byref(a), ctypes.byref(n), None) == C.SRW_EINVAL
    assert lib.srw_attention_plan(None, ctypes.byref(n), ctypes.byref(n)) == C.SRW_EINVAL


def test_counts_are_whole_numbers(pkg):
    """A count of another type is refused before any sequence has its pages."""
    import numpy as np
    c = pkg.PagedKvCache(1, 8, 1, 64, page_size=16, device="cpu")
    a, b = c.add(), c.add()
    before = (dict(c._lens), {s: list(p) for s, p in c._pages.items()}, list(c._free))
    for bad in (1.0, "1", None):
        with pytest.raises(TypeError):
            c.extend([a, b], [20, bad])
        assert before == (c._lens, c._pages, c._free)
    assert c.extend([a, b], [np.int64(20), 1])[1].tolist() == [20, 1]
