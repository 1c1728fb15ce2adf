"""GPU: DawnModel.extend (sequences of different lengths over the paged cache)
against the model's own prefill and decode_step.

With a bf16 cache the two differ where the pools' bf16 outputs are the same and
the attention rounds its weights and its output to bf16 (2^-8 each); behind the
first layer that goes through the steep gates of further calls: the models' bar
of 2e-2.  int8 pages hold values to 1/254 of a row's largest, about as bf16 does
its own to 2^-8: the same bar.  fp8 pages hold them to 2^-4 of each (2.6% rms),
averaged by the attention: 0.1."""

from __future__ import annotations

import pytest
import torch

from tests.parity import rel_fro

pytestmark = pytest.mark.gpu
BARS = {torch.bfloat16: 2e-2, torch.int8: 2e-2, torch.float8_e4m3fn: 0.1}


@pytest.fixture(scope="module")
def model(pkg, dev):
    cfg = pkg.DawnConfig(vocab_size=300, d_model=128, n_layers=2, n_heads=2, max_seq_len=300, d_route=64,
                         n_qk=300, n_v=500, n_know=1000, max_chunk_size=600)
    params = pkg.init_params(cfg, seed=5)
    g = torch.Generator().manual_seed(6)
    params["router"]["tau_attn"]["kernel"] = 0.05 * torch.randn(128, 3, generator=g)
    params["router"]["tau_know"]["kernel"] = 0.05 * torch.randn(128, 1, generator=g)
    params["norm"]["bias"] = 0.1 * torch.randn(128, generator=g)
    return cfg, pkg.DawnModel(params, cfg, dev)


def _prompts(lens, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 300, (n,), generator=g) for n in lens]


@pytest.mark.parametrize("dtype", BARS, ids=lambda d: str(d).split(".")[1])
def test_prompts_chunks_and_tokens(model, dev, dtype):
    """Ragged prompts, the rest of one together with single tokens of the
    others, a few generated tokens: every logit against the whole sequence's
    prefill."""
    cfg, m = model
    print(f"[gpu] extend {dtype}", flush=True)
    lens = [150, 37, 1, 90]
    ids = _prompts(lens, 11)
    cache = m.new_cache(40, page_size=16, dtype=dtype)
    seqs = [cache.add() for _ in lens]
    steps = [[70, 30, 0, 90], [77, 1, 1, 0], [1, 1, 0, 0], [1, 1, 0, 0], [1, 4, 0, 0]]
    got = [[] for _ in lens]
    at = [0] * len(lens)
    for counts in steps:
        take = torch.cat([ids[i][at[i]:at[i] + n] for i, n in enumerate(counts)])
        out = m.extend(take, cache, seqs, counts)
        for i, piece in enumerate(torch.split(out, counts)):
            got[i].append(piece)
            at[i] += counts[i]
    assert at == lens and [cache.length(q) for q in seqs] == lens
    for i, t in enumerate(ids):
        want, *_ = m.prefill(t[None])
        err = rel_fro(torch.cat(got[i]).cpu(), want[0].cpu())
        print(f"  sequence of {lens[i]}: {err:.2e}", flush=True)
        assert err <= BARS[dtype]


def test_matches_decode_step_and_last_only(model, dev):
    """The next token of sequences of different lengths, in one call, as the
    model's own one-sequence steps give it."""
    cfg, m = model
    lens = [40, 3, 129]
    ids = _prompts(lens, 21)
    cache = m.new_cache(12, page_size=64)
    seqs = [cache.add() for _ in lens]
    print("[gpu] extend, decode steps", flush=True)
    last = m.extend(torch.cat(ids), cache, seqs, lens, last_only=True)
    token = torch.tensor([5, 7, 9])
    nxt = m.extend(token, cache, seqs, [1, 1, 1], last_only=True)
    assert last.shape == nxt.shape == (3, cfg.vocab_size)
    for i, t in enumerate(ids):
        want, k, v, n = m.prefill(t[None])
        assert rel_fro(last[i].cpu(), want[0, -1].cpu()) <= 2e-2
        step, *_ = m.decode_step(token[i:i + 1], k, v, n)
        assert rel_fro(nxt[i].cpu(), step[0].cpu()) <= 2e-2


def test_window_and_evicted_pages(model, dev):
    """With a window, giving back the pages that it has left changes nothing,
    bit for bit, and another sequence may write into them."""
    cfg, m = model
    ids = _prompts([200, 120], 31)
    outs = []
    print("[gpu] extend, window", flush=True)
    for evict in (False, True):
        cache = m.new_cache(30, page_size=16)
        a = cache.add()
        m.extend(ids[0][:150], cache, [a], [150], window=40, sinks=4)
        if evict:
            free = cache.free_pages
            assert cache.evict(a, 40, 4) == (150 - 40 + 1) // 16 - 1   # all but the sinks' page
            assert cache.free_pages == free + (150 - 40 + 1) // 16 - 1
            b = cache.add()
            m.extend(ids[1], cache, [b], [120])
        outs.append(m.extend(ids[0][150:], cache, [a], [50], window=40, sinks=4))
    assert torch.equal(outs[0], outs[1])


def test_refusals(model, dev):
    cfg, m = model
    cache = m.new_cache(3, page_size=16)
    a, b = cache.add(), cache.add()
    ids = torch.zeros(60, dtype=torch.long)
    for bad in (lambda: m.extend(ids[:3], cache, [a, b], [1, 1]), lambda: m.extend(ids[:0], cache, [a], [0]),
                lambda: m.extend(ids[:1], cache, [a, b], [1, 0], last_only=True),
                lambda: m.extend(torch.zeros(301, dtype=torch.long), cache, [a], [301])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(MemoryError):
        m.extend(ids, cache, [a], [60])
    assert cache.length(a) == 0 and cache.free_pages == 3
    print("[gpu] extend refusals", flush=True)
    assert m.extend(ids[:40], cache, [a], [40]).shape == (40, cfg.vocab_size)
    cache.free(a)
    assert cache.free_pages == 3
