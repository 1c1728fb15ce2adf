"""CPU: what DawnModel.generate refuses before it reads a prompt or asks the cache for a
sequence."""

from __future__ import annotations

import types

import pytest
import torch

NAN = float("nan")
Z = torch.zeros
BAD = [(ValueError, dict(keep=4)), (ValueError, dict(keep=4, n=1)), (ValueError, dict(keep=1, indexed=True)),
       (ValueError, dict(keep=4, first=-1, indexed=True)), (ValueError, dict(keep=4, last=0, indexed=True)),
       (ValueError, dict(keep=4, first=3, last=2, indexed=True)), (ValueError, dict(keep=-2, indexed=True)),
       (ValueError, dict(keep=4, window=8, indexed=True)), (TypeError, dict(keep=2.5, indexed=True)),
       (TypeError, dict(keep=4, first=0.5, indexed=True)), (ValueError, dict(window=-1)), (ValueError, dict(sinks=2)),
       (ValueError, dict(temperature=-1.0)), (ValueError, dict(temperature=NAN)), (ValueError, dict(temperature=Z(3))),
       (TypeError, dict(temperature=Z(4).double())), (TypeError, dict(top_k=Z(4))), (ValueError, dict(top_k=-1)),
       (TypeError, dict(top_k=1.5)), (ValueError, dict(top_p=1.5)), (ValueError, dict(top_p=Z(4, 1))),
       (ValueError, dict(min_p=2)), (ValueError, dict(min_p=Z(4, device="meta"))), (ValueError, dict(u=Z(4, 3))),
       (ValueError, dict(u=[0.5] * 12)), (TypeError, dict(u=Z(3, 4).double())), (TypeError, dict(u=Z(3, 4, device="meta"))),
       (ValueError, dict(samples=0)), (ValueError, dict(n=0)), (ValueError, dict(n=20)), (ValueError, dict(prompts=[[1], []])),
       (ValueError, dict(prompts=[[1], [50]]))]


def call(pkg, n=3, indexed=False, prompts=([1, 2], [3]), samples=2, **kw):
    def reads(*a, **k):
        raise AssertionError("a prompt was read")

    model = types.SimpleNamespace(cfg=pkg.DawnConfig(vocab_size=50, max_seq_len=16), device=torch.device("cpu"), extend=reads)
    cache = types.SimpleNamespace(indexed=indexed, add=reads)
    return pkg.DawnModel.generate(model, list(prompts), cache, n, samples=samples, **kw)


@pytest.mark.parametrize("err,kw", BAD, ids=str)
def test_refused_before_prompts_are_read(pkg, err, kw):
    with pytest.raises(err):
        call(pkg, **kw)


@pytest.mark.parametrize("kw", [dict(), dict(keep=4, indexed=True), dict(window=8, sinks=2), dict(u=Z(4, 3).T),
                                dict(temperature=Z(1).expand(4), top_k=torch.ones(8, dtype=torch.int32)[::2])], ids=str)
def test_others_are_read(pkg, kw):
    with pytest.raises(AssertionError, match="was read"):
        call(pkg, **kw)
