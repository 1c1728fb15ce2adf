"""GPU: what DawnModel.extend leaves of a cache when a call is refused or fails."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_model_paged import _prompts, model  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


def _state(cache):
    return dict(cache._lens), {s: list(p) for s, p in cache._pages.items()}, list(cache._free)


@pytest.mark.parametrize("why", ["window", "sinks", "windows type", "layer"])
def test_a_call_that_fails_leaves_the_cache_as_it_was(model, monkeypatch, why):  # noqa: F811
    """Refused arguments and failures in the layers: lengths and pages as before,
    and the same call made right gives what it gives on a cache that saw no
    failure."""
    cfg, m = model
    print(f"[gpu] extend fails: {why}", flush=True)
    ids = _prompts([50, 20], 41)
    outs = []
    for fail in (False, True):
        cache = m.new_cache(12, page_size=16)
        a, b = cache.add(), cache.add()
        m.extend(ids[0][:30], cache, [a], [30])
        if fail:
            before = _state(cache)
            rest = torch.cat([ids[0][30:], ids[1]])
            kw, kind = {"window": (dict(window=-1), ValueError), "sinks": (dict(sinks=4), ValueError),
                        "windows type": (dict(window=2.5), TypeError), "layer": ({}, RuntimeError)}[why]
            with monkeypatch.context() as mp:
                if why == "layer":
                    know, n = m._know, []

                    def broken(*args):
                        n.append(1)
                        if len(n) == 2:
                            raise RuntimeError("no memory")
                        return know(*args)
                    mp.setattr(m, "_know", broken)
                with pytest.raises(kind):
                    m.extend(rest, cache, [a, b], [20, 20], **kw)
            assert _state(cache) == before
        outs.append(m.extend(torch.cat([ids[0][30:], ids[1]]), cache, [a, b], [20, 20]))
    assert torch.equal(*outs)
