"""GPU: kv_index where sequences hold more tokens than their tables have places for, with
and without the number of new tokens, and where few of many places are new."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_kv import I32, KINDS, Cache, _cu, _fill
from tests.test_gpu_kv_select import _empty_index, _index_of

pytestmark = pytest.mark.gpu


def _check(index, want, touched, pages):
    codes, scale = index.codes.cpu(), index.scale.cpu()
    for page in range(pages):
        if page in touched:
            assert torch.equal(codes[page], want[page][0]) and torch.equal(scale[page], want[page][1]), page
        else:
            assert (codes[page] == 3).all() and (scale[page] == 3).all(), page


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("total", [True, False], ids=["total", "any"])
def test_tokens_behind_the_table(pkg, dev, kind, total):
    print(f"[gpu] kv_index behind the table {kind} {total}", flush=True)
    P, lens = 16, [40, 40, 9, 75]
    c = Cache(pkg, dev, kind, 2, 64, P, lens, seed=5)
    _fill(pkg, dev, c, torch.Generator().manual_seed(5))
    want = _index_of(c)
    for width, counts in ((2, lens), (1, lens), (2, [40, 30, 0, 75]), (3, [1, 40, 9, 50])):
        index = _empty_index(pkg, dev, c)
        pkg.kv_index(c.pages, index, c.table[:, :width], c.len_t, _cu(dev, counts), total=sum(counts) if total else None)
        touched = {c.rows[b][j] for b, n in enumerate(counts) if n
                   for j in range((lens[b] - n) // P, min(width, -(-lens[b] // P)))}
        _check(index, want, touched, c.pages.n_pages)


@pytest.mark.parametrize("total", [True, False], ids=["total", "any"])
def test_few_new_tokens_of_wide_tables(pkg, dev, total):
    """More places than tokens: units by the tokens; fewer: by the places."""
    print(f"[gpu] kv_index wide {total}", flush=True)
    P, lens = 32, [1000, 31, 32, 33, 640]
    c = Cache(pkg, dev, "int8", 3, 128, P, lens, seed=6)
    _fill(pkg, dev, c, torch.Generator().manual_seed(6))
    want = _index_of(c)
    wide = torch.full((5, 200), -1, dtype=I32, device=dev)
    wide[:, :c.table.shape[1]] = c.table
    for counts in ([3, 0, 2, 33, 64], [1, 1, 1, 1, 1], [1000, 31, 0, 1, 640], [0, 0, 0, 0, 0]):
        for table in (c.table, wide):
            index = _empty_index(pkg, dev, c)
            pkg.kv_index(c.pages, index, table, c.len_t, _cu(dev, counts), total=sum(counts) if total else None)
            touched = {c.rows[b][j] for b, n in enumerate(counts) if n for j in range((lens[b] - n) // P, (lens[b] - 1) // P + 1)}
            _check(index, want, touched, c.pages.n_pages)
    pkg.kv_index(c.pages, index, c.table[:, :0], c.len_t, _cu(dev, lens), total=sum(lens) if total else None)
