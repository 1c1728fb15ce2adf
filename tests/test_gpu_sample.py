"""GPU: sample (one token of every row of logits from given random numbers) against
the definition in float64 on the CPU.

Tokens are equal.  The kernel sums weights in units of 2^-q (q at least 38), the
definition in float64: a draw or a border would have to lie within V 2^-q of the sum
to differ, which at these sizes is under 1e-8 of it, and the inputs are fixed.
Logprobs are float32 roundings (2^-24 of the value) of a double that is within V 2^-q of
the logarithm: |error| <= 2^-23 |logprob| + 1e-7."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
INF, NAN = math.inf, math.nan


def definition(logits, u, temperature, top_k, top_p, min_p):
    """(token, logprob) of one row."""
    l = torch.nan_to_num(logits.to(F64), nan=-INF, posinf=INF, neginf=-INF)
    V, top = l.shape[0], l.max().item()
    if top == -INF:
        return -1, -INF
    if not temperature > 0:
        return int(torch.nonzero(l == top)[0]), 0.0
    if top == INF:
        z = torch.where(l == INF, 0.0, -INF).to(F64)
    else:
        z = torch.where(l == -INF, torch.full_like(l, -INF), (l - top) / temperature)
    order = sorted(range(V), key=lambda i: (-l[i].item(), i)) if V < 300 else torch.sort(l, descending=True, stable=True).indices.tolist()
    w = torch.exp(z)[torch.tensor(order)]
    n = min(V, top_k) if top_k > 0 else V
    if top_p < 1:
        run = torch.cumsum(w[:n], 0)
        reach = torch.nonzero(run >= top_p * run[-1])
        n = int(reach[0]) + 1
    if min_p > 0:
        n = min(n, int((w >= min(min_p, 1.0)).sum()))
    kept = torch.zeros(V, dtype=F64)
    kept[torch.tensor(order[:n])] = w[:n]
    run = torch.cumsum(kept, 0)
    x = 0.0 if not u > 0 else min(float(u), 1 - 2.0 ** -53)
    token = int((run <= x * run[-1]).sum())
    while token >= V or kept[token] == 0:
        token -= 1
    return token, float(torch.log(kept[token] / run[-1]))


def f32(x):
    return float(torch.tensor(x, dtype=F32))


def check(pkg, dev, logits, u, **p):
    p = {**dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **p}
    at = lambda t: t.to(dev) if isinstance(t, torch.Tensor) else t  # noqa: E731
    token, logprob = pkg.sample(logits if logits.is_cuda else logits.to(dev), u.to(dev), **{k: at(v) for k, v in p.items()})
    assert token.dtype == torch.int64 and logprob.dtype == F32 and token.shape == logprob.shape == u.shape
    token, logprob, logits = token.tolist(), logprob.tolist(), logits.cpu()
    for b in range(len(token)):
        row = {k: (v[b].item() if isinstance(v, torch.Tensor) else v if k == "top_k" else f32(v)) for k, v in p.items()}
        want, log = definition(logits[b], u[b].item(), **row)
        assert token[b] == want, (b, row, token[b], want)
        if math.isinf(log):
            assert logprob[b] == log
        else:
            assert abs(logprob[b] - log) <= 2.0 ** -23 * abs(log) + 1e-7, (b, row, logprob[b], log)


RULES = {
    "whole": {},
    "k": dict(top_k=40),
    "k1": dict(top_k=1),
    "p": dict(top_p=0.9),
    "p0": dict(top_p=0.0),
    "min_p": dict(min_p=0.05),
    "all": dict(temperature=0.7, top_k=100, top_p=0.95, min_p=0.01),
    "k_p": dict(temperature=1.3, top_k=20, top_p=0.5),
    "greedy": dict(temperature=0.0, top_k=5),
    "hot": dict(temperature=50.0, top_p=0.99),
    "hot_k": dict(temperature=50.0, top_k=6000, top_p=0.98, min_p=0.8),
    "cold": dict(temperature=0.01, top_p=0.9),
}


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 63, 64, 257, 1000, 4099, 32000, 131073])
@pytest.mark.parametrize("rule", RULES)
def test_rules_and_sizes(pkg, dev, rule, V, dtype):
    print(f"[gpu] sample {rule} {V} {dtype}", flush=True)
    g = torch.Generator().manual_seed(V + len(rule))
    B = 3 if V > 30000 else 7
    logits = (3 * torch.randn(B, V, generator=g)).to(dtype)
    check(pkg, dev, logits, torch.rand(B, generator=g), **RULES[rule])


@pytest.mark.parametrize("V", [50, 5003, 40000])
def test_parameters_of_each_row(pkg, dev, V):
    print(f"[gpu] sample rows {V}", flush=True)
    g = torch.Generator().manual_seed(V)
    B = 24
    logits = 2 * torch.randn(B, V, generator=g)
    t = 0.2 + 1.5 * torch.rand(B, generator=g)
    t[::5] = 0
    k = torch.randint(0, 60, (B,), generator=g, dtype=I32)
    k[1::4] = 0
    p = 0.3 + 0.9 * torch.rand(B, generator=g)
    m = 0.1 * torch.rand(B, generator=g) * (torch.arange(B) % 3 == 0)
    check(pkg, dev, logits, torch.rand(B, generator=g), temperature=t, top_k=k, top_p=p.clamp_max(1), min_p=m)


def test_entries_that_mean_off(pkg, dev):
    """What a number could not be: each entry as the documentation says."""
    print("[gpu] sample entries", flush=True)
    g = torch.Generator().manual_seed(5)
    logits = torch.randn(9, 300, generator=g)
    u = torch.rand(9, generator=g)
    f = lambda *x: torch.tensor(x, dtype=F32)  # noqa: E731
    check(pkg, dev, logits, u, temperature=f(-1, NAN, -INF, INF, 1, 1e-40, 3e38, 1, 1),
          top_k=torch.tensor([0, 0, 0, 0, -5, 0, 0, 2 ** 31 - 1, -2 ** 31], dtype=I32))
    ones = torch.ones(9)
    got = pkg.sample(logits.to(dev), u.to(dev), top_p=f(1, 2, NAN, INF, 1, 1, 1, 1, 1).to(dev),
                     min_p=f(0, -1, NAN, -INF, 0, 0, 0, 0, 0).to(dev), temperature=ones.to(dev))
    want = pkg.sample(logits.to(dev), u.to(dev))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    token, logprob = pkg.sample(logits.to(dev), u.to(dev), min_p=torch.full((9,), 7.0, device=dev))
    assert torch.equal(token.cpu(), logits.argmax(1)) and (logprob == 0).all()


def test_random_numbers_at_the_ends(pkg, dev):
    print("[gpu] sample ends", flush=True)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 5.0, -1.0, INF, -INF, NAN, 0.5])
    for V in (7, 6000):
        logits = torch.zeros(9, V)
        token, logprob = pkg.sample(logits.to(dev), u.to(dev))
        last = V - 1
        assert token.tolist() == [0, last, last, last, 0, last, 0, 0, V // 2]
        assert (logprob.cpu() + math.log(V)).abs().max() < 1e-6


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("V", [100, 9001, 70000])
def test_equal_logits(pkg, dev, V, dtype):
    """Borders of top-k and top-p inside runs of equal logits: the first by index."""
    print(f"[gpu] sample equal {V} {dtype}", flush=True)
    g = torch.Generator().manual_seed(V)
    few = torch.randint(0, 4, (6, V), generator=g).to(dtype)
    few[2] = 1.5
    few[3, ::2], few[3, 1::2] = 0.0, -0.0     # equal too
    u = torch.rand(6, generator=g)
    for rule in (dict(top_k=max(1, V // 3)), dict(top_p=0.55), dict(top_k=V // 2, top_p=0.7), dict(top_k=5),
                 dict(temperature=1e-3, top_p=0.3), dict(min_p=1.0), dict(top_k=V), dict(top_k=V - 1)):
        check(pkg, dev, few, u, **rule)


@pytest.mark.parametrize("V", [65, 20001])
def test_masked_infinite_and_nan(pkg, dev, V):
    print(f"[gpu] sample masks {V}", flush=True)
    g = torch.Generator().manual_seed(V)
    l = 3 * torch.randn(10, V, generator=g)
    l[0, torch.rand(V, generator=g) < 0.9] = -INF
    l[1] = -INF
    l[2] = -INF
    l[2, V // 2] = -1e30                       # one token left
    l[3, 7:] = torch.finfo(F32).min            # masks of the type's lowest value
    l[4] = torch.finfo(F32).min                # all of them: all alike
    l[5, ::3] = NAN
    l[6] = NAN
    l[7, [3, V - 2]] = INF
    l[8, 5], l[8, 6] = INF, NAN
    l[9, 0], l[9, 1:] = torch.finfo(F32).max, torch.finfo(F32).min
    u = torch.rand(10, generator=g)
    for rule in ({}, dict(top_k=10), dict(top_p=0.8), dict(top_k=50, top_p=0.9, min_p=0.1), dict(temperature=0.0),
                 dict(temperature=3e38, top_p=0.9)):
        check(pkg, dev, l, u, **rule)
    token, logprob = pkg.sample(l.to(dev), u.to(dev), temperature=0.0)
    assert token[[1, 6]].tolist() == [-1, -1] and (logprob[[1, 6]] == -INF).all()


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
def test_strides_and_alignments(pkg, dev, dtype):
    """Rows that begin anywhere, repeat or lie apart."""
    print(f"[gpu] sample strides {dtype}", flush=True)
    g = torch.Generator().manual_seed(3)
    wide = (3 * torch.randn(6, 2111, generator=g)).to(dtype).to(dev)
    u = torch.rand(6, generator=g)
    for first in range(9):
        check(pkg, dev, wide[:, first:first + 2000], u, top_p=0.9)
    check(pkg, dev, wide.T[:6], u, top_k=3)                        # columns: copied
    check(pkg, dev, wide[:1].expand(6, -1), u, top_k=30)
    check(pkg, dev, wide[::2], u[:3], temperature=0.0)
    one = pkg.sample(wide[2:3, 5:], u[2:3].to(dev), top_p=0.8)
    all_ = pkg.sample(wide[:, 5:], u.to(dev), top_p=0.8)
    assert one[0][0] == all_[0][2] and one[1][0] == all_[1][2]     # not by the batch
    empty = pkg.sample(wide[:0], u[:0].to(dev))
    assert empty[0].shape == empty[1].shape == (0,)


def test_draws_follow_the_weights(pkg, dev):
    """u over a fine even grid: every token's share of the draws is its weight, within
    one step of the grid at either end."""
    print("[gpu] sample shares", flush=True)
    n = 4096
    for V, rule in ((11, {}), (11, dict(top_k=4)), (6000, {}), (6000, dict(top_p=0.5))):
        logits = torch.randn(V, generator=torch.Generator().manual_seed(V))
        token, logprob = pkg.sample(logits.to(dev).expand(n, -1), ((torch.arange(n) + 0.5) / n).to(dev), **rule)
        count = torch.bincount(token.cpu(), minlength=V).to(F64) / n
        assert (torch.diff(token.cpu()) >= 0).all()
        share = torch.zeros(V, dtype=F64).scatter_(0, token.cpu(), logprob.cpu().to(F64).exp())
        assert ((count - share).abs() <= 2.0 / n).all()


def test_streams_and_capture(pkg, dev):
    print("[gpu] sample streams, capture", flush=True)
    g = torch.Generator().manual_seed(8)
    logits = torch.randn(5, 33000, generator=g).to(dev)
    u = torch.rand(5, generator=g).to(dev)
    k = torch.full((5,), 9, dtype=I32, device=dev)
    want = pkg.sample(logits, u, top_k=k, top_p=0.9)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = pkg.sample(logits, u, top_k=k, top_p=0.9)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = pkg.sample(logits, u, top_k=k, top_p=0.9)
    for seed in range(3):
        logits.copy_(torch.randn(5, 33000, generator=torch.Generator().manual_seed(seed)))
        k.fill_(seed * 7)
        graph.replay()
        torch.cuda.synchronize()
        want = pkg.sample(logits, u, top_k=k, top_p=0.9)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(pkg, dev):
    x, u = torch.zeros(3, 10, device=dev), torch.zeros(3, device=dev)
    bad = [(ValueError, (x[0], u), {}), (ValueError, (x.cpu(), u), {}), (TypeError, (x.half(), u), {}),
           (ValueError, (x, u[:2]), {}), (TypeError, (x, u.double()), {}), (TypeError, (x, 0.5), {}),
           (ValueError, (x, u.cpu()), {}), (ValueError, (x[:, :0], u), {}),
           (ValueError, (x, u), dict(temperature=-0.1)), (ValueError, (x, u), dict(temperature=NAN)),
           (ValueError, (x, u), dict(top_k=-1)), (TypeError, (x, u), dict(top_k=1.5)),
           (ValueError, (x, u), dict(top_p=1.1)), (ValueError, (x, u), dict(top_p=NAN)),
           (ValueError, (x, u), dict(min_p=-0.1)), (TypeError, (x, u), dict(top_k=u)),
           (ValueError, (x, u), dict(top_p=u[:2])), (TypeError, (x, u), dict(temperature=u.double())),
           (NotImplementedError, (x.clone().requires_grad_(), u), {})]
    for err, args, kw in bad:
        with pytest.raises(err):
            pkg.sample(*args, **kw)
    with torch.no_grad():
        pkg.sample(x.clone().requires_grad_(), u)


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("V,size", [(4500, 450), (20000, 2000), (30001, 1500)])
def test_top_k_at_the_ends_of_equal_runs(pkg, dev, V, size, dtype):
    """Runs of equal logits, and k one before, at and one behind each run's end."""
    print(f"[gpu] sample runs {V} {size} {dtype}", flush=True)
    g = torch.Generator().manual_seed(V)
    level = (torch.randperm(V, generator=g) // size).to(F32)
    k = torch.tensor([size * i + d for i in range(1, V // size + 1) for d in (-1, 0, 1)], dtype=I32)
    B = len(k)
    logits = (-0.25 * level)[None].repeat(B, 1).to(dtype)
    u = torch.rand(B, generator=g)
    check(pkg, dev, logits, u, top_k=k)
    check(pkg, dev, logits, u, top_k=k, top_p=0.97)
    check(pkg, dev, logits, u, top_k=k, top_p=0.9, min_p=0.2, temperature=0.8)


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("V", [90, 700, 1025, 2047, 2049, 4097, 4466, 12000, 40001])
def test_any_parameters(pkg, dev, V, dtype):
    """Rows with a k of any size, half of them with top-p, some with min-p."""
    print(f"[gpu] sample any {V} {dtype}", flush=True)
    g = torch.Generator().manual_seed(V + 1)
    B = 160
    logits = (2.5 * torch.randn(B, V, generator=g)).to(dtype)
    rand = lambda: torch.rand(B, generator=g)  # noqa: E731
    k = torch.exp(rand() * math.log(V + 1)).to(I32)
    k[::7] = 0
    p = torch.where(rand() < 0.5, torch.ones(B), 1 - 10 ** (-3 * rand()))
    least = torch.where(rand() < 0.7, torch.zeros(B), 10 ** (-4 * rand()))
    check(pkg, dev, logits, rand(), temperature=0.3 + 1.5 * rand(), top_k=k, top_p=p, min_p=least)


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("V,B", [(9000, 12), (32001, 40)])
def test_min_p_above_the_border_of_top_p(pkg, dev, V, B, dtype):
    """min-p that leaves less than top-p does, far less, about as much and more."""
    print(f"[gpu] sample p and min_p {V} {dtype}", flush=True)
    g = torch.Generator().manual_seed(V + 3)
    logits = (3 * torch.randn(B, V, generator=g)).to(dtype)
    least = 10 ** (-torch.arange(B, dtype=F32) / 8)
    for p in (0.999, 0.9, 0.3):
        check(pkg, dev, logits, torch.rand(B, generator=g), top_p=p, min_p=least)
    check(pkg, dev, logits, torch.rand(B, generator=g), top_p=0.98, min_p=least, temperature=3.0)
