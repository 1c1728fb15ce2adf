"""GPU: DawnModel.generate and extend over chosen pages: the cache, its forks and its
index, the attention to kept pages and the sampling together, as a program uses them.

Logits of the same model by other calls agree within its bar for bf16 caches
(2e-2 relative to all, as for extend against prefill).  Calls of the same shapes on
the same pages agree bit for bit."""

from __future__ import annotations

import pytest
import torch

from tests.parity import rel_fro

pytestmark = pytest.mark.gpu
BAR = 2e-2


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


def _draw(logits, u, t, k, p):
    """The rule in float64, and whether u or the nucleus' edge lie too close to a border
    to tell: weights are exact to 2^-50, float64 sums of 300 of them to 2^-44."""
    l = logits.double().cpu()
    w = torch.exp((l - l.max()) / t)
    order = torch.sort(l, descending=True, stable=True).indices[:k or None]
    run = w[order].cumsum(0)
    edge = p * run[-1]
    n = min(int((run < edge).sum()) + 1, len(order)) if p < 1 else len(order)
    near = p < 1 and float((run - edge).abs().min() / run[-1]) < 1e-12
    kept = torch.zeros_like(w)
    kept[order[:n]] = w[order[:n]]
    run = kept.cumsum(0)
    at = float(u) * run[-1]
    near = near or float((run[kept > 0] - at).abs().min() / run[-1]) < 1e-12
    token = int((run > at).nonzero()[0])
    return token, float(torch.log(kept[token] / run[-1])), near


@pytest.mark.parametrize("samples,keep", [(1, 0), (3, 0), (3, 4)])
def test_generated_tokens_follow_their_logits(pkg, model, dev, monkeypatch, samples, keep):
    """Each token is the one that the rule gives of the step's logits and the caller's
    number; the logits of the steps are those of the finished sequences, read whole."""
    cfg, m = model
    print(f"[gpu] generate {samples} {keep}", flush=True)
    lens, n = [50, 3, 64], 21
    prompts = _prompts(lens, 31)
    B = len(lens) * samples
    u = torch.rand(n, B, generator=torch.Generator().manual_seed(3))
    cache = m.new_cache(60, page_size=16, indexed=keep > 0)
    seen = []
    step = m.extend

    def extend(ids, cache, seqs, *rest, **named):
        out = step(ids, cache, seqs, *rest, **named)
        seen.append(out.clone())
        return out

    monkeypatch.setattr(m, "extend", extend)
    tokens, logprobs = m.generate(prompts, cache, n, samples=samples, u=u.to(dev), temperature=1.5, top_k=40, top_p=0.9,
                                  keep=keep)
    monkeypatch.undo()
    assert tokens.shape == logprobs.shape == (B, n) and cache.free_pages == 60
    seen[0] = seen[0].repeat_interleave(samples, 0)
    for i in range(n):
        for b in range(B):
            token, share, near = _draw(seen[i][b], u[i, b], 1.5, 40, 0.9)
            assert near or (int(tokens[b, i]) == token and abs(float(logprobs[b, i]) - share) < 1e-5)
    if samples > 1:  # (numbers of their own: the samples of a prompt part)
        assert any(not torch.equal(tokens[samples * i], tokens[samples * i + 1]) for i in range(len(lens)))
    if keep:
        return
    for b in range(B):
        whole = torch.cat([prompts[b // samples].to(dev), tokens[b, :-1]])
        want, *_ = m.prefill(whole[None])
        got = torch.stack([seen[i][b] for i in range(n)])
        assert rel_fro(got.cpu(), want[0, lens[b // samples] - 1:].cpu()) <= BAR


def test_parameters_of_each_row_and_an_end(model, dev):
    """Rows with parameters of their own; a row stops at the end's token and the others
    go on."""
    cfg, m = model
    print("[gpu] generate, end", flush=True)
    prompts = _prompts([20, 33], 41)
    t = torch.tensor([0.0, 0.0, 2.0, 2.0], device=dev)
    u = torch.rand(12, 4, generator=torch.Generator().manual_seed(8)).to(dev)
    free, _ = m.generate(prompts, m.new_cache(20, page_size=16), 12, samples=2, u=u, temperature=t)
    assert torch.equal(free[0], free[1])  # greedy: samples agree
    end = int(free[2, 4])
    cache = m.new_cache(20, page_size=16)
    tokens, logprobs = m.generate(prompts, cache, 12, samples=2, u=u, temperature=t, end=end)
    assert cache.free_pages == 20
    for b in range(4):
        hit = (tokens[b] == end).nonzero()
        stop = int(hit[0]) + 1 if len(hit) else 12
        assert (tokens[b, stop:] == end).all() and (logprobs[b, stop:] == 0).all()
    stop = int((tokens[2] == end).nonzero()[0])
    assert stop <= 4


def test_all_pages_kept_is_attention_to_all(model, dev):
    """A list as long as the table keeps every page: the logits of a step agree with the
    step over all pages."""
    cfg, m = model
    print("[gpu] extend, all pages kept", flush=True)
    lens = [150, 37, 1]
    ids = torch.cat(_prompts(lens, 51))
    out = []
    for keep in (0, 19):
        cache = m.new_cache(40, page_size=16, indexed=True)
        seqs = [cache.add() for _ in lens]
        m.extend(ids, cache, seqs, lens)
        step = [m.extend(torch.tensor([7, 8, 9]), cache, seqs, [1, 1, 1], keep=keep),
                m.extend(torch.arange(12), cache, seqs, [3, 9, 0], keep=keep)]
        out.append(torch.cat(step).cpu())
    assert rel_fro(out[1], out[0]) <= BAR


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8], ids=["bf16", "int8"])
def test_ends_alone_kept_is_a_window_with_sinks(model, dev, dtype):
    """At a page's last position the first and the last two pages are what a window of
    two pages with a page of sinks sees."""
    cfg, m = model
    print("[gpu] extend, ends kept", flush=True)
    ids = _prompts([207], 61)[0]
    out = []
    for call in (dict(keep=3, first=1, last=2), dict(window=32, sinks=16)):
        cache = m.new_cache(20, page_size=16, indexed=True, dtype=dtype)
        a = cache.add()
        m.extend(ids, cache, [a], [207])
        out.append(m.extend(torch.tensor([3]), cache, [a], [1], **call).cpu())
        assert cache.length(a) == 208
    assert rel_fro(out[0], out[1]) <= BAR


def test_a_fork_and_a_moved_cache_go_on(model, dev):
    """A sequence read once and forked, one fork extended, the cache compacted and
    resized: each goes on bit for bit as one that never shared or moved a page."""
    cfg, m = model
    print("[gpu] forks, moves", flush=True)
    ids = _prompts([70], 71)[0]

    def step(cache, seq, token, keep):
        return m.extend(torch.tensor([token]), cache, [seq], [1], keep=keep).cpu()

    alone = m.new_cache(30, page_size=16, indexed=True)
    x, y = alone.add(), alone.add()
    m.extend(ids, alone, [x], [70])
    m.extend(ids, alone, [y], [70])
    cache = m.new_cache(30, page_size=16, indexed=True)
    gone, a = cache.add(), cache.add()
    m.extend(ids[:33], cache, [gone], [33])
    m.extend(ids, cache, [a], [70])
    b = cache.fork(a)
    assert torch.equal(step(cache, a, 1, 3), step(alone, x, 1, 3))
    cache.free(gone)
    assert cache.compact() > 0
    assert torch.equal(step(cache, b, 2, 0), step(alone, y, 2, 0))
    cache.resize(13)
    for t in range(3, 14):
        assert torch.equal(step(cache, a, t, 3), step(alone, x, t, 3))
        assert torch.equal(step(cache, b, t, 3), step(alone, y, t, 3))


def test_refusals_leave_the_cache(model, dev):
    cfg, m = model
    print("[gpu] generate, refusals", flush=True)
    prompts = _prompts([20, 33], 81)
    plain, indexed = m.new_cache(12, page_size=16), m.new_cache(12, page_size=16, indexed=True)
    for cache, call in ((plain, dict(keep=4)), (indexed, dict(keep=4, window=8)), (indexed, dict(keep=2, first=1, last=2)),
                        (indexed, dict(keep=4, last=0)), (plain, dict(u=torch.zeros(4, 3, device=dev))),
                        (plain, dict(samples=0)), (plain, dict(temperature=-1.0)), (plain, dict(top_k=-1))):
        with pytest.raises(ValueError):
            m.generate(prompts, cache, 4, **call)
        assert cache.free_pages == 12 and not cache._lens
    with pytest.raises(ValueError):
        m.generate(prompts, plain, 269)
    with pytest.raises(ValueError):
        m.generate([], plain, 2)
    with pytest.raises(ValueError):
        m.generate([torch.tensor([300])], plain, 2)
    with pytest.raises(MemoryError):
        m.generate(prompts, plain, 60, samples=3)
    assert plain.free_pages == 12 and not plain._lens
