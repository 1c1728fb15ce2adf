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
