"""The whole numbers that srw_sample sums, on the CPU: a logit's weight bit for bit
(exact rationals, rounded where the kernel rounds), and the draw from a row's whole
distribution by runs of 8 192 logits.

The kernel's table of 2^(j / 128) is the device's; numbers here agree with it wherever a
logit lies at a whole octave (j = 0) and else within a unit, which decides a draw only
where it falls on a border."""

from __future__ import annotations

import math
from fractions import Fraction

import numpy as np

RUN = 8192


def f32(x):
    return float(np.float32(x))


def _fma(a, b, c):
    return float(Fraction(a) * Fraction(b) + Fraction(c))


class Numbers:
    """Weights of a row of V logits at temperature t (a float32 number)."""

    def __init__(self, t, V):
        self.q = min(51, 62 - (V - 1).bit_length())
        self.c, self.per = 1.4426950408889634 / t, t * 0.6931471805599453

    def top(self, m):
        """The octave R of a largest logit m."""
        return math.ceil(float(m) * self.c)

    def lowest(self, R):
        return f32(max((R - self.q - 1.0) * self.per, -3.4028234663852886e38))

    def weight(self, l, R):
        if not l >= self.lowest(R):
            return 0
        y = l * self.c
        n = round(y * 128)
        r = y - n / 128
        p = _fma(float.fromhex("0x1.c6b095a17a14dp-5"), r, float.fromhex("0x1.ebfbeebe2d1a2p-3"))
        p = _fma(p, r, float.fromhex("0x1.62e42fefa39efp-1"))
        p = _fma(p, r, 1.0) * 2.0 ** ((n & 127) / 128)
        return round(Fraction(math.ldexp(p, (n >> 7) - R)) * 2 ** self.q)

    def weights(self, l, R):
        values, place = np.unique(np.asarray(l, np.float32), return_inverse=True)
        return np.array([self.weight(float(x), R) for x in values], dtype=np.int64)[place]


def place(u, total):
    """The whole number under u times total."""
    return min(int(Fraction(f32(u)) * total), total - 1)


def first_past(weights, at):
    """The first index at which the running sum passes at."""
    return int(np.nonzero(np.cumsum(weights) > at)[0][0])


def draw_whole(logits, u, t=1.0):
    """(token, logprob) of a row of finite logits from its whole distribution: a run's
    weights are in units of its own largest, its sum is taken down to the row's."""
    l = np.asarray(logits, np.float32)
    w = Numbers(f32(t), len(l))
    R = w.top(l.max())
    runs = [l[a:a + RUN] for a in range(0, len(l), RUN)]
    own = [w.weights(x, w.top(x.max())) for x in runs]
    under = [min(R - w.top(x.max()), 63) for x in runs]
    sums = [int(x.sum()) >> d for x, d in zip(own, under)]
    total = sum(sums)
    at = place(u, total)
    for i, s in enumerate(sums):
        if at < s:
            break
        at -= s
    token = i * RUN + first_past(own[i], at << under[i])
    return token, _log_share(w, l[token], R, int(own[i][token - i * RUN]) == total << under[i], total)


def _log_share(w, l, R, alone, total):
    return 0.0 if alone else (float(l) * w.c - R - math.log2(total / 2 ** w.q)) * math.log(2)


def draw_top_p(logits, u, p, t=1.0):
    """(token, logprob) by top-p, every weight in the units of the row's largest."""
    l = np.asarray(logits, np.float32)
    w = Numbers(f32(t), len(l))
    R = w.top(l.max())
    own = w.weights(l, R)
    order = np.argsort(-l, kind="stable")
    total = int(own.sum())
    goal = min(max(1, math.ceil(Fraction(f32(p)) * total)), total)
    n = int(np.nonzero(np.cumsum(own[order]) >= goal)[0][0]) + 1
    kept = np.zeros_like(own)
    kept[order[:n]] = own[order[:n]]
    total = int(kept.sum())
    token = first_past(kept, place(u, total))
    return token, _log_share(w, l[token], R, int(kept[token]) == total, total)
