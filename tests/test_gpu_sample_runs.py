"""GPU: sample over rows of several runs of 8 192 logits whose largest lie far apart, at
random numbers that fall on and next to a run's border.

Tokens are those of the whole numbers (sample_numbers.py), logprobs within float32's
rounding of a double that is within 2^-37 of them: 2^-23 |logprob| + 1e-7."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from tests.sample_numbers import draw_top_p, draw_whole
from tests.test_gpu_sample import definition, f32

pytestmark = pytest.mark.gpu
BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32
INF = math.inf
OUT = 0x5a5a5a


def aligned(rows, dtype, dev):
    """Rows that begin at 16-byte borders."""
    V = len(rows[0])
    held = torch.zeros(len(rows), (V + 7) // 8 * 8, dtype=dtype, device=dev)
    held[:, :V] = torch.tensor(np.stack(rows)).to(dtype).to(dev)
    return held[:, :V]


def both(pkg, logits, u, t=1.0):
    """From numbers and from tensors as parameters: each a kernel of its own, one result."""
    B, dev = logits.shape[0], logits.device
    held = [torch.full((B,), OUT, dtype=torch.int64, device=dev) for _ in range(16)]
    del held             # (what an output without a result would hold)
    got = pkg.sample(logits, u, temperature=t)
    rows = pkg.sample(logits, u, temperature=torch.full((B,), t, device=dev))
    assert torch.equal(got[0], rows[0]) and torch.equal(got[1], rows[1])
    return got[0].tolist(), got[1].tolist()


def far_runs(V, dtype):
    """Rows with runs 40 to 60 octaves under the rest: the first, a middle one, the last;
    behind tokens that weigh as much as those before (u = 1/2 falls into the run)."""
    cast = lambda x: float(torch.tensor(x).to(dtype))  # noqa: E731
    rows = []
    for octaves in (40, 44.5, 46.3, 47.6, 50, 52, 57.7, 60):
        low = cast(-octaves * math.log(2))
        for run in (0, 1, V // 8192):
            l = np.zeros(V, np.float32)
            l[8192 * run:8192 * run + 8192] = low
            rows.append(l)
        l = np.full(V, -60.0, np.float32)
        l[0] = l[16384] = 0.0
        l[8192:16384] = low
        rows.append(l)
    return rows


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("V", [20000, 100003])
def test_draws_inside_runs_that_weigh_little(pkg, dev, V, dtype):
    print(f"[gpu] sample far runs {V} {dtype}", flush=True)
    rows = far_runs(V, dtype)
    for u in (0.0, 2.0 ** -24, 0.5, 1 - 2.0 ** -24):
        tokens, logs = both(pkg, aligned(rows, dtype, dev), torch.full((len(rows),), u, device=dev))
        for b, l in enumerate(rows):
            want, log = draw_whole(l, u)
            assert tokens[b] == want, (b, u, tokens[b], want)
            assert abs(logs[b] - log) <= 2.0 ** -23 * abs(log) + 1e-7, (b, u, logs[b], log)


@pytest.mark.parametrize("V,octaves,p", [(1 << 20, 43.2, 1 - 2.0 ** -24), (1 << 20, 43.6, 1 - 2.0 ** -24),
                                         (1 << 20, 34, 0.99999), (1 << 20, 31.9, 0.99999), (1 << 20, 32.1, 0.9999),
                                         (1 << 24, 39.4, 1 - 2.0 ** -16), (1 << 24, 36, 1 - 2.0 ** -13)])
def test_top_p_whose_border_lies_in_the_far_tail(pkg, dev, V, octaves, p):
    """A token that weighs nearly all, and a tail that weighs together as much as top-p
    leaves out: each of its tokens nothing in the row's units, or a few."""
    print(f"[gpu] sample far tail {V} {octaves} {p}", flush=True)
    rows = []
    for at in (0, V // 2 + 3, V - 1):
        l = np.full(V, -octaves * math.log(2), np.float32)
        l[at] = 0.0
        rows.append(l)
    logits = aligned(rows, F32, dev)
    for u in (0.0, 0.5, 1 - 2.0 ** -24):
        token, log = pkg.sample(logits, torch.full((3,), u, device=dev), top_p=p)
        for b, l in enumerate(rows):
            want, share = draw_top_p(l, u, p)
            assert token[b].item() == want, (b, u, token[b].item(), want)
            assert abs(log[b].item() - share) <= 2.0 ** -23 * abs(share) + 1e-7, (b, u, log[b].item(), share)


RULES = [{}, dict(top_p=0.5), dict(top_p=0.93), dict(top_p=0.9995), dict(top_p=0.9, min_p=0.03), dict(min_p=1e-3),
         dict(top_k=7), dict(top_k=900), dict(top_k=3000), dict(top_k=200, top_p=0.8), dict(temperature=0.0),
         dict(temperature=0.31), dict(temperature=2.5, top_p=0.99)]


def anywhere(l, dtype, dev, B=9):
    """B rows that all hold l and begin at every place of a 16-byte vector."""
    V = len(l)
    stride = V + 3 if V % 2 == 0 else V + 2
    held = torch.full((B * stride + 8,), 50.0, dtype=dtype, device=dev)      # (larger than what the rows hold)
    logits = held[:B * stride].as_strided((B, V), (stride, 1))
    logits.copy_(torch.as_tensor(l).to(dtype).to(dev).expand(B, -1))
    return logits, logits[4:5]


def same_anywhere(pkg, dev, l, dtype, rules, us):
    one = aligned([np.asarray(l, np.float32)], dtype, dev)
    many, other = anywhere(l, dtype, dev)
    for rule in rules:
        for u in us:
            token, log = pkg.sample(one, torch.full((1,), u, device=dev), **rule)
            for logits in (many, other):
                got = pkg.sample(logits, torch.full((logits.shape[0],), u, device=dev), **rule)
                assert (got[0] == token).all(), (rule, u, token.tolist(), got[0].tolist())
                assert (got[1] == log).all(), (rule, u, log.tolist(), got[1].tolist())


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("V", [1500, 2047, 2100, 8192, 8193, 16385, 40001])
def test_rows_give_the_same_wherever_they_lie(pkg, dev, V, dtype):
    """Bit for bit, in other batches and from every address."""
    print(f"[gpu] sample anywhere {V} {dtype}", flush=True)
    g = torch.Generator().manual_seed(V)
    l = (3 * torch.randn(V, generator=g)).numpy()
    us = torch.rand(3, generator=g).tolist() + [0.0, 1 - 2.0 ** -24]
    same_anywhere(pkg, dev, l, dtype, RULES, us)
    same_anywhere(pkg, dev, np.sort(l), dtype, RULES[:6], us)


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("V", [16385, 40001])
@pytest.mark.parametrize("at", [8187, 8191, 8192, 8195, 16383, 16384])
def test_a_large_logit_at_a_runs_border(pkg, dev, V, at, dtype):
    """Over tails whose tokens weigh nothing beside it, and something in a run without it;
    the last logits of runs drawn too."""
    print(f"[gpu] sample border {V} {at} {dtype}", flush=True)
    for octaves in (47.3, 49, 52):
        l = np.full(V, float(torch.tensor(-octaves * math.log(2)).to(dtype)), np.float32)
        l[at] = 0.0
        for u in (0.0, 0.5, 1 - 2.0 ** -24):
            want, log = draw_whole(l, u)
            logits, _ = anywhere(l, dtype, dev)
            token, share = pkg.sample(logits, torch.full((logits.shape[0],), u, device=dev))
            assert (token == want).all(), (u, want, token.tolist())
            assert ((share - log).abs() <= 2.0 ** -23 * abs(log) + 1e-7).all()
        same_anywhere(pkg, dev, l, dtype, [{}, dict(top_p=0.9), dict(top_k=2), dict(min_p=0.5)], [0.0, 0.7])


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("V", [24576, 24583])
def test_draws_of_a_runs_last_logits(pkg, dev, V, dtype):
    """Every token alike, u at each of the last and first ones of the runs."""
    print(f"[gpu] sample last of runs {V} {dtype}", flush=True)
    logits, _ = anywhere(np.zeros(V, np.float32), dtype, dev)
    for i in [*range(8182, 8196), *range(16380, 16388), *range(24570, V), V - 1]:
        u = float(np.float32((i + 0.5) / V))
        token, log = pkg.sample(logits, torch.full((logits.shape[0],), u, device=dev))
        assert (token == draw_whole(np.zeros(V, np.float32), u)[0]).all(), (i, token.tolist())
        assert ((log + math.log(V)).abs() < 1e-6).all()


@pytest.mark.parametrize("dtype", [F32, BF], ids=["f32", "bf16"])
def test_whether_top_p_lists_tokens_goes_by_their_number(pkg, dev, dtype):
    """512 equal logits, 257 of them a wave's where the row begins inside of a vector, over a run that adds
    a few units to the sum: top-p of a half keeps one more than a half of them."""
    print(f"[gpu] sample lists {dtype}", flush=True)
    E = 4 if dtype == F32 else 8
    V, q = 70001, 45
    l = np.full(V, -200.0, np.float32)
    wave = 64 * E                                    # a wave's next logits, every 16 waves
    places = [16 * wave * j + i for j in range(2) for i in range(128)] + [wave]
    rest = iter(range(2 * wave, 16 * wave, 7))
    while len(places) < 512:
        places.append(next(rest))
    l[places] = 0.0
    low = float(torch.tensor(-50 * math.log(2)).to(dtype))
    l[65536:65536 + 4000] = low                      # nothing each in the row's units, some 120 together
    same_anywhere(pkg, dev, l, dtype, [dict(top_p=0.5), dict(top_p=0.25)], [0.0, 0.3, 0.75, 1 - 2.0 ** -24])
    token, _ = pkg.sample(torch.tensor(l).to(dtype).to(dev)[None], torch.full((1,), 1 - 2.0 ** -24, device=dev), top_p=0.5)
    assert token.item() == sorted(places)[256]


def test_sums_of_more_than_53_bits(pkg, dev):
    """u and p of a half over sums of 2^61 and a few units: the border lies among tokens of
    a unit each, or in a run of some hundred units."""
    print("[gpu] sample halves", flush=True)
    u = lambda x: torch.full((1,), x, device=dev)  # noqa: E731
    l = np.zeros(1027, np.float32)
    l[512:515] = -51 * math.log(2)                    # one unit each, behind 2^60 and before 2^60
    row = torch.tensor(l, device=dev)[None]
    # 2^60 + 1 of 2^61 + 3 units: the second of them
    assert draw_whole(l, 0.5)[0] == 513
    assert pkg.sample(row, u(0.5))[0].item() == 513
    # top-p reaches 2^60 + 1.5: 513 of the large ones
    assert draw_top_p(l, 1 - 2.0 ** -24, 0.5)[0] == 515
    assert pkg.sample(row, u(1 - 2.0 ** -24), top_p=0.5)[0].item() == 515
    assert pkg.sample(row, u(1 - 2.0 ** -24), top_p=0.5, top_k=1026)[0].item() == 515
    for V, far in ((24576, 53.0), (24576, 55.5), (24577, 54.0)):
        l = np.zeros(V, np.float32)
        l[8192:16384] = -far * math.log(2)
        for dtype in (F32, BF):
            l = torch.tensor(l).to(dtype).float().numpy()
            for x in (0.5, 0.25, 0.75, 0.3):
                want, log = draw_whole(l, x)
                token, share = both(pkg, aligned([l], dtype, dev), u(x))
                assert token == [want] and abs(share[0] - log) <= 2.0 ** -23 * abs(log) + 1e-7, (V, far, x, token, want)


@pytest.mark.parametrize("t", [1e-5, 1e-6, 1e-7, 2e-8, 1e-8])
@pytest.mark.parametrize("V", [60, 1000, 3000, 20001])
def test_very_low_temperatures(pkg, dev, V, t):
    """Logits a few roundings apart, up to 2^30 octaves over 0 and under it.  A token's
    octaves are a product of 53 bits, off by 2^-24 at most: so are weights, sums and the
    logarithm of a share, 2^-23 ln 2 in all, beside what other rows' logprobs are off."""
    print(f"[gpu] sample cold {V} {t}", flush=True)
    g = torch.Generator().manual_seed(V)
    near = torch.randint(0, 40, (6, V), generator=g).float()
    base = torch.tensor([12.0, -12.0, 10.25, -9.5, 0.75, -0.03])[:, None]
    logits = base + near * torch.tensor([2.0 ** -20, 2.0 ** -20, 2.0 ** -20, 2.0 ** -20, 2.0 ** -23, 2.0 ** -28])[:, None]
    u = torch.rand(6, generator=g)
    for rule in ({}, dict(top_k=V // 3), dict(top_p=0.8), dict(top_k=30, top_p=0.6), dict(min_p=0.2)):
        token, log = pkg.sample(logits.to(dev), u.to(dev), temperature=t, **rule)
        for b in range(6):
            p = {**dict(top_k=0, top_p=1.0, min_p=0.0), **rule}
            want, share = definition(logits[b], u[b].item(), f32(t), p["top_k"], f32(p["top_p"]), f32(p["min_p"]))
            assert token[b].item() == want, (rule, b, token[b].item(), want)
            assert abs(log[b].item() - share) <= 2.0 ** -23 * abs(share) + 1e-7 + 2.0 ** -23 * math.log(2), (rule, b)


@pytest.mark.parametrize("V", [2, 3000])
def test_min_p_between_zero_and_the_smallest_number(pkg, dev, V):
    """min-p's border lies between the logits 0 and 2^-149: 0 weighs less than it asks."""
    print(f"[gpu] sample smallest {V}", flush=True)
    tiny = 2.0 ** -149
    l = torch.zeros(1, V)
    l[0, V // 3] = tiny
    for least, u in ((0.6, 0.99), (0.6, 0.0), (0.3, 0.99), (0.3, 0.0)):
        want, share = definition(l[0], u, tiny, 0, 1.0, f32(least))
        token, log = pkg.sample(l.to(dev), torch.full((1,), u, device=dev), temperature=tiny, min_p=least)
        assert token.item() == want and abs(log.item() - share) <= 2.0 ** -23 * abs(share) + 1e-7, (least, u, token, want)


@pytest.mark.parametrize("V", [900, 1500, 2049, 8192, 9001, 40001])
def test_arrays_give_what_numbers_do(pkg, dev, V):
    """Other kernels and other parameters beside a row's own, entries that mean off: the
    same bits."""
    print(f"[gpu] sample arrays {V}", flush=True)
    g = torch.Generator().manual_seed(V)
    B = 6
    logits = (3 * torch.randn(B, V, generator=g)).to(dev)
    logits[1, ::2] = logits[1, 1::2][:1]            # many alike
    logits[2, V // 3:] -= 30.0                      # later runs far under the first
    u = torch.rand(B, generator=g).to(dev)
    off = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    array = lambda k, x: torch.full((B,), x, device=dev, dtype=I32 if k == "top_k" else F32)  # noqa: E731
    for rule in RULES:
        want = pkg.sample(logits, u, **rule)
        whole = {**off, **rule}
        for names in (["top_k"], ["top_p"], ["min_p"], ["temperature", "top_p"], list(off)):
            got = pkg.sample(logits, u, **{**rule, **{k: array(k, whole[k]) for k in names}})
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (rule, names)
        mixed = {k: array(k, x) for k, x in whole.items()}
        mixed["top_k"][0], mixed["top_p"][1], mixed["min_p"][2], mixed["temperature"][3] = 3, 0.4, 0.2, 0.0
        got = pkg.sample(logits, u, **mixed)
        assert torch.equal(got[0][4:], want[0][4:]) and torch.equal(got[1][4:], want[1][4:]), rule


@pytest.mark.parametrize("rule", [{}, dict(top_p=0.9), dict(top_p=0.99, min_p=0.01)], ids=str)
def test_captured_calls_with_workspaces(pkg, dev, rule):
    """Two graphs of one pool, replayed in turn with eager calls between."""
    print(f"[gpu] sample captured {rule}", flush=True)
    draw = lambda seed: 3 * torch.randn(4, 30011, generator=torch.Generator().manual_seed(seed))  # noqa: E731
    logits, u = [draw(s).to(dev) for s in (1, 2)], torch.rand(4, generator=torch.Generator().manual_seed(3)).to(dev)
    pkg.sample(logits[0], u, **rule)
    torch.cuda.synchronize()
    graphs, got = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph, l in zip(graphs, logits):
        with torch.cuda.graph(graph, pool=graphs[0].pool() if got else None):
            got.append(pkg.sample(l, u, **rule))
    for seed in range(4):
        for i in (seed % 2, 1 - seed % 2):
            logits[i].copy_(draw(10 * seed + i))
            graphs[i].replay()
            want = pkg.sample(logits[i], u, **rule)
            torch.cuda.synchronize()
            assert torch.equal(got[i][0], want[0]) and torch.equal(got[i][1], want[1]), (seed, i)
