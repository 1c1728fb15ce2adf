"""Performance cases of what a program that generates text does around the paged
cache's attention: choosing tokens from logits, copying pages when sequences
branch or move, and attending to a few pages that a cheap score selects.

A case is a dict of plain values; ``kind`` names the pass:

* ``sample``  ``sample`` draws one token of every row of logits from given
              random numbers, with temperature, top-k, top-p and min-p, and
              gives the logarithm of its probability;
* ``copy``    ``kv_copy`` copies pages of all layers of a cache onto other
              pages;
* ``index``   ``kv_index`` brings the pages' index (the mean of a page's keys
              for each head, in 8 bits) up to date with new tokens;
* ``attend``  ``kv_select`` chooses pages for each new token and key head by
              the index, ``paged_attention`` attends to these alone.

Sampling, for a row of logits l with temperature t, largest logit M and weights
w_i = exp((l_i - M) / t): tokens in the order of their logits, the largest
first, equal ones by index; top-k keeps the first k; top-p keeps the shortest
run of those whose weights reach p times the sum of theirs; min-p keeps what
weighs min_p or more.  The token is the first, by index, at which the kept
weights' running sum passes u times their sum.  t = 0: the first in the order.

Pages: k [pages, H, P, dh], v [pages, H, dh, P]; with 8 bits one float32 scale
for each token and head, [pages, H, P].  Position p of sequence b lies in page
``table[b, p // P]`` at slot ``p % P``.  The index of a page and head: m the
largest magnitude of the mean of its keys, codes round(mean * (127 / m)), scale
m / 127.  A new token at position i of a sequence sees the pages 0 ... i // P
of its table; always selected are the first ``first`` and the last ``last`` of
them, and of the others those with the largest scores, equal ones from the
front, until there are ``n``.  The score of a page is scale * (c . codes), c the
codes of the sum of the queries of the key head's group, as the index holds
means.
"""

import math
import random

import torch

own = False

DEV = "cuda:0"
BF16, F32, F64, I32, U8 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.uint8
FP8 = torch.float8_e4m3fn
TYPES = {"bf16": BF16, "f32": F32, "int8": torch.int8, "fp8": FP8}
TINY = 2.0 ** -100  # a mean whose largest magnitude is at most this is held as zeros


def _sample(B, V, dtype, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, rows=False, **rest):
    """``rows``: every row has parameters of its own around these."""
    return dict(rest, kind="sample", B=B, V=V, dtype=dtype, temperature=temperature, top_k=top_k, top_p=top_p,
                min_p=min_p, rows=rows)


def _copy(L, pages, pairs, H, dh, P, cache, **rest):
    return dict(rest, kind="copy", L=L, pages=pages, pairs=pairs, H=H, dh=dh, P=P, cache=cache)


def _seqs(kind, B, new, past, H, dh, P, cache, **rest):
    """B sequences with new[0] to new[1] new tokens behind past[0] to past[1]."""
    return dict(rest, kind=kind, B=B, new_lo=new[0], new_hi=new[1], past_lo=past[0], past_hi=past[1], H=H, dh=dh, P=P,
                cache=cache)


def listed():
    return [
        # one user's next token from the model's vocabulary, every rule on: the smallest call
        _sample(name="sample_one", B=1, V=30000, dtype="f32", temperature=0.8, top_k=50, top_p=0.95, min_p=0.02),
        # 64 sequences of a batch, each request with parameters of its own, some greedy
        _sample(name="sample_batch", B=64, V=32000, dtype="f32", temperature=0.9, top_k=100, top_p=0.9, min_p=0.05,
                rows=True),
        # a large vocabulary of odd size, bf16 logits (many equal ones), nucleus sampling
        _sample(name="sample_nucleus", B=192, V=131073, dtype="bf16", temperature=1.0, top_p=0.92),
        # many samples for scoring or training, from the whole distribution
        _sample(name="sample_whole", B=512, V=100003, dtype="f32", temperature=1.0),
        # a sequence of the 40M model branches: its last, partial page gets a copy for each of three others
        _copy(name="copy_branch", L=12, pages=64, pairs=3, H=6, dh=64, P=64, cache="bf16"),
        # compacting a larger cache: 200 pages move
        _copy(name="copy_compact", L=24, pages=500, pairs=200, H=8, dh=128, P=64, cache="fp8"),
        # the prompts of 8 sequences of the model's full length enter the index
        _seqs("index", name="index_prompts", B=8, new=(512, 512), past=(0, 0), H=6, dh=64, P=64, cache="bf16"),
        # a long document, wide heads, 8 bits
        _seqs("index", name="index_long", B=1, new=(65521, 65521), past=(9, 9), H=8, dh=128, P=64, cache="int8"),
        # generating for one sequence, small pages
        _seqs("attend", name="attend_one", B=1, new=(1, 1), past=(4000, 4000), H=6, dh=64, P=16, cache="bf16", G=1, n=24,
              first=1, last=2),
        # generating for 32 long sequences, four query heads to a key head: an eighth of the positions
        _seqs("attend", name="attend_long", B=32, new=(1, 1), past=(4000, 32000), H=8, dh=128, P=64, cache="fp8", G=4,
              n=32, first=1, last=2),
        # generating at the end of one very long sequence
        _seqs("attend", name="attend_deep", B=1, new=(1, 1), past=(200002, 200002), H=2, dh=128, P=128, cache="bf16",
              G=8, n=64, first=1, last=1),
        # drafted tokens of several sequences checked together
        _seqs("attend", name="attend_drafts", B=12, new=(3, 17), past=(900, 6000), H=4, dh=64, P=32, cache="int8", G=2,
              n=20, first=1, last=2),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """Another case of the listed ranges: other batches, vocabularies, rules,
    lengths, head layouts, pages and types."""
    kind = rng.choice(["sample", "sample", "sample", "copy", "index", "attend", "attend", "attend"])
    if kind == "sample":
        V = _log_int(rng, 64, 262144)
        B = _log_int(rng, 1, max(1, min(512, 50000000 // V)))
        return _sample(B=B, V=V, dtype=rng.choice(["f32", "bf16"]), temperature=round(rng.uniform(0.3, 1.8), 3),
                       top_k=rng.choice([0, 0, 1, _log_int(rng, 2, 2000)]),
                       top_p=rng.choice([1.0, 1.0, round(rng.uniform(0.05, 0.999), 4)]),
                       min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.3), 4)]), rows=rng.random() < 0.5)
    dh = rng.choice([64, 64, 128])
    cache = rng.choice(["bf16", "int8", "fp8"])
    P = rng.choice([16, 32, 64, 128, 256])
    H = rng.choice([1, 2, 4, 6, 8])
    if kind == "copy":
        L = _log_int(rng, 1, 24)
        pages = _log_int(rng, 8, max(8, min(2000, 800000000 // (L * H * P * dh * 4))))
        return _copy(L=L, pages=pages, pairs=_log_int(rng, 1, max(1, pages * 2 // 5)), H=H, dh=dh, P=P, cache=cache)
    if kind == "index":
        n = _log_int(rng, 1, 16000)
        B = _log_int(rng, 1, max(1, min(128, 60000 // n)))
        return _seqs("index", B=B, new=(max(1, n // 2), n), past=(0, _log_int(rng, 1, 4000)), H=H, dh=dh, P=P,
                     cache=cache)
    G = rng.choice([1, 2, 4, 8])
    n = _log_int(rng, 4, 64)
    new = rng.choice([1, 1, 1, _log_int(rng, 2, 24)])
    past = _log_int(rng, 20, 60000)
    # at most the positions of attend_long and selected values that the plain form can hold
    B = _log_int(rng, 1, max(1, min(64, int(4e8 / (past * H * dh)), int(1.2e8 / (new * H * n * P * dh)))))
    last = rng.choice([1, 2, 3])
    return _seqs("attend", B=B, new=(max(1, new // 2), new), past=(past // 4, past), H=H, dh=dh, P=P, cache=cache, G=G,
                 n=n, first=min(rng.choice([0, 1, 1, 2]), n - last), last=last)


def _lengths(case):
    """(new, total) positions of each sequence: the case's own, whatever the
    seed."""
    rng = random.Random(" ".join("%s=%s" % (k, case[k]) for k in sorted(case) if k != "name"))
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["B"])]
    return new, [n + rng.randint(case["past_lo"], case["past_hi"]) for n in new]


def work(case):
    if case["kind"] == "sample":
        B, V = case["B"], case["V"]
        # a comparison, a difference, an exponential and a sum of each logit
        return {"bytes": B * V * (2 if case["dtype"] == "bf16" else 4) + B * 16, "flops": 4 * B * V}
    H, dh, P = case["H"], case["dh"], case["P"]
    key = dh * 2 if case["cache"] == "bf16" else dh + 4
    if case["kind"] == "copy":
        return {"bytes": 2 * case["pairs"] * case["L"] * H * P * 2 * key, "flops": 0}
    new, total = _lengths(case)
    if case["kind"] == "index":
        pages = [((t - n) // P, (t - 1) // P) for n, t in zip(new, total)]
        keys = sum(t - a * P for (a, _), t in zip(pages, total))
        return {"bytes": keys * H * key + sum(b - a + 1 for a, b in pages) * H * (dh + 4), "flops": keys * H * dh}
    n, G = case["n"], case["G"]
    byts = flops = 0
    for m, t in zip(new, total):
        pages = -(-t // P)
        # the index's entries, and pages that its tokens select (each could be another's too), read once
        byts += H * (pages * (dh + 4) + 2 * key * min(t, m * n * P)) + m * H * (4 * G * dh + 4 * n)
        flops += H * m * (2 * pages * dh + 4 * G * dh * min(t, n * P))
    return {"bytes": byts, "flops": flops}


# -- inputs ------------------------------------------------------------------------

def _prepare_sample(case, g):
    B, V = case["B"], case["V"]
    rand = lambda *shape: torch.rand(*shape, generator=g, device=DEV)  # noqa: E731
    logits = torch.randn(B, V, generator=g, device=DEV).mul_(3.0).to(TYPES[case["dtype"]])
    s = dict(case, logits=logits, u=rand(B))
    if case["rows"]:
        greedy = rand(B) < 0.1
        s["temperature"] = torch.where(greedy, torch.zeros(B, device=DEV), case["temperature"] * (0.5 + rand(B)))
        some = rand(B) < 0.7
        s["top_k"] = torch.where(some, (case["top_k"] * (0.2 + 2 * rand(B))).to(I32), torch.zeros(B, dtype=I32, device=DEV))
        s["top_p"] = (case["top_p"] + 0.15 * (rand(B) - 0.5)).clamp_(0.01, 1.0)
        s["min_p"] = case["min_p"] * 2 * rand(B)
    return s


def _held(case, shape, g, offset=None):
    """Random pages, around ``offset``."""
    kind = case["cache"]
    x = torch.randn(shape, generator=g, device=DEV, dtype=BF16)
    if offset is not None:
        x = x.mul_(0.8).add_(offset)
    if kind == "int8":
        return x.mul_(40.0).clamp_(-127.0, 127.0).round_().to(torch.int8)
    return x.mul_(100.0).clamp_(-448.0, 448.0).to(FP8) if kind == "fp8" else x


def _scales(case, shape, g):
    # tokens of different sizes
    if case["cache"] == "bf16":
        return None
    return torch.exp(0.3 * torch.randn(shape, generator=g, device=DEV)) / (40.0 if case["cache"] == "int8" else 100.0)


def _prepare_copy(case, g):
    L, N, H, dh, P = (case[k] for k in ("L", "pages", "H", "dh", "P"))
    t = [_held(case, (L, N, H, P, dh), g), _held(case, (L, N, H, dh, P), g)]
    if case["cache"] != "bf16":
        t += [_scales(case, (L, N, H, P), g) for _ in range(2)]
    # what the planner on the host holds: pages that are copied, some of them several times, and others for them
    order = torch.randperm(N, generator=g, device=DEV).tolist()
    to = order[:case["pairs"]]
    left = order[case["pairs"]:]
    return dict(case, tensors=t, src=[left[i // 2 % len(left)] for i in range(len(to))], dst=to)


def _bits(t):
    """fp8 pages are indexed as bytes."""
    return t.view(U8) if t.dtype == FP8 else t


def _mean_codes(mean):
    """(codes, scales) of means [..., dh], float32 or rounded to it."""
    mean = mean.to(F32)
    most = mean.abs().amax(-1)
    fine = most > TINY
    zero, top = torch.zeros_like(most), torch.full_like(most, 127.0)   # (a number / a tensor is two roundings)
    y = torch.round(mean * torch.where(fine, top / most, zero)[..., None])
    return y.to(torch.int8), torch.where(fine, most / top, zero)


def _prepare_seqs(case, g):
    new, total = _lengths(case)
    P, B, H, dh = (case[k] for k in ("P", "B", "H", "dh"))
    need = [-(-t // P) for t in total]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(I32)
    at = torch.arange(max(need), device=DEV)[None]
    count = torch.tensor(need, device=DEV)[:, None]
    begin = torch.cumsum(count, 0) - count
    table = torch.where(at < count, order[(begin + at).clamp_max(pages - 1)], torch.full((), -1, dtype=I32, device=DEV))
    cu = None if max(new) == 1 else torch.tensor([sum(new[:i]) for i in range(B + 1)], dtype=I32, device=DEV)
    T = sum(new)
    s = dict(case, table=table.contiguous(), lens=torch.tensor(total, dtype=I32, device=DEV), cu=cu, T=T, most=max(new))
    # what a page is about, and tokens around it
    topic = torch.randn(pages, H, 1, dh, generator=g, device=DEV, dtype=BF16).mul_(0.6)
    s["pages"] = [_held(case, (pages, H, P, dh), g, topic), _held(case, (pages, H, dh, P), g)]
    s["scales"] = [_scales(case, (pages, H, P), g) for _ in range(2)]
    if case["kind"] == "index":
        s["index"] = [torch.zeros(pages, H, dh, dtype=torch.int8, device=DEV), torch.zeros(pages, H, device=DEV)]
        return s
    # the index as it stands: the program has kept it up to date
    codes, scale = [], []
    for part in range(0, pages, 512):
        k = s["pages"][0][part:part + 512].to(F32)
        if s["scales"][0] is not None:
            k = k * s["scales"][0][part:part + 512][..., None]
        c, sc = _mean_codes(k.mean(2))
        codes.append(c)
        scale.append(sc)
    s["index"] = [torch.cat(codes), torch.cat(scale)]
    s["q"] = torch.randn(T, H * case["G"], dh, generator=g, device=DEV).to(BF16)
    return s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    return {"sample": _prepare_sample, "copy": _prepare_copy}.get(case["kind"], _prepare_seqs)(case, g)


# -- the plain forms ---------------------------------------------------------------

def _column(x, B, dtype):
    return (x if isinstance(x, torch.Tensor) else torch.full((B,), x, device=DEV)).to(dtype)[:, None]


def _plain_sample(s):
    B, V = s["B"], s["V"]
    # 64 bits: the running sums decide between neighbours
    l = s["logits"].to(F64)
    # (a number's value is that of the float32 that a tensor would hold)
    t, p, least = (_column(s[n], B, F32).to(F64) for n in ("temperature", "top_p", "min_p"))
    k = _column(s["top_k"], B, torch.int64)
    l, order = torch.sort(l, dim=-1, descending=True, stable=True)
    w = ((l - l[:, :1]) / torch.where(t > 0, t, torch.ones_like(t))).exp_()
    del l
    rank = torch.arange(V, device=DEV)[None]
    keep = (rank < k) | (k <= 0)
    of_k = w * keep
    run = torch.cumsum(of_k, -1)
    keep &= (run - of_k < p * run[:, -1:]) | (p >= 1) | (rank == 0)
    del of_k, run
    keep &= w >= least
    keep = torch.where(t > 0, keep, rank == 0)
    kept = torch.zeros_like(w).scatter_(1, order, w * keep)
    run = torch.cumsum(kept, -1)
    total = run[:, -1:]
    token = (run <= s["u"].to(F64)[:, None] * total).sum(-1, keepdim=True).clamp_max(V - 1)
    return token[:, 0], torch.log(kept.gather(1, token) / total)[:, 0].to(F32)


def _plain_copy(s):
    src, dst = (torch.tensor(s[n], device=DEV) for n in ("src", "dst"))
    for t in s["tensors"]:
        t = _bits(t)
        t[:, dst] = t[:, src]
    return s["tensors"]


def _plain_index(s):
    P, lens = s["P"], s["lens"].long()
    B = s["B"]
    cu = torch.arange(B + 1, device=DEV) if s["cu"] is None else s["cu"].long()
    at = torch.arange(s["table"].shape[1], device=DEV)[None]
    first = (lens - (cu[1:] - cu[:-1]))[:, None] // P
    seq, at = torch.nonzero((at >= first) & (at * P < lens[:, None]), as_tuple=True)
    page = s["table"].long()[seq, at]
    k = _bits(s["pages"][0])[page].view(s["pages"][0].dtype).to(F32)
    # 64 bits: a code next to a border
    k = k.to(F64)
    if s["cache"] != "bf16":
        k = k * s["scales"][0][page][..., None].to(F64)
    have = (at * P)[:, None] + torch.arange(P, device=DEV) < lens[seq][:, None]
    mean = (k * have[:, None, :, None]).sum(2) / have.sum(1)[:, None, None]
    s["index"][0][page], s["index"][1][page] = _mean_codes(mean)
    return _values(s)


def _values(s):
    """The values that the index's codes stand for."""
    return s["index"][0].to(F32) * s["index"][1][..., None]


def _plain_select(s):
    B, H, G, dh, P, T, n = (s[k] for k in ("B", "H", "G", "dh", "P", "T", "n"))
    cu = torch.arange(B + 1, device=DEV) if s["cu"] is None else s["cu"].long()
    at = torch.arange(T, device=DEV)
    seq = torch.searchsorted(cu, at, right=True) - 1
    pos = s["lens"].long()[seq] - cu[seq + 1] + at
    own_page = (pos // P)[:, None, None]
    c, _ = _mean_codes(s["q"].to(F64).reshape(T, H, G, dh).sum(2))
    table = s["table"].long().clamp_min(0)
    W, most = table.shape[1], s["most"]
    row = (cu[:-1, None] + torch.arange(most, device=DEV)).clamp_max(T - 1)               # [B, most]: the packed rows, padded
    codes = s["index"][0][table].to(F32).permute(0, 2, 3, 1).contiguous()                 # [B, H, dh, W]
    # (whole numbers under 2^24: exact in any order)
    dots = torch.matmul(c[row].to(F32).transpose(1, 2).contiguous(), codes)               # [B, H, most, W]
    score = (dots * s["index"][1][table].transpose(1, 2)[:, :, None])[seq, :, at - cu[seq]]  # [T, H, W]
    j = torch.arange(W, device=DEV)
    sees = j <= own_page
    always = sees & ((j < s["first"]) | (j > own_page - s["last"]))
    score = score.masked_fill_(always, float("inf")).masked_fill_(~sees, float("-inf"))
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :n]
    keep = torch.where(order <= own_page, order, W)
    keep = torch.sort(keep, dim=-1).values
    keep = torch.where(keep < W, keep, -1)
    if W < n:
        keep = torch.cat([keep, torch.full((T, H, n - W), -1, device=DEV)], -1)
    return keep.to(I32), seq, pos


def _plain_attend(s):
    H, G, dh, P, T, n = (s[k] for k in ("H", "G", "dh", "P", "T", "n"))
    keep, seq, pos = _plain_select(s)
    at = keep.long().clamp_min(0)
    page = s["table"].long().clamp_min(0)[seq[:, None, None], at]                         # [T, H, n]
    head = torch.arange(H, device=DEV)[None, :, None]
    get = lambda t: _bits(t)[page, head].view(t.dtype).to(F32)  # noqa: E731
    k, v = (get(t) for t in s["pages"])                                                   # [T, H, n, P, dh], [.., dh, P]
    if s["cache"] != "bf16":
        k = k * s["scales"][0][page, head][..., None]
        v = v * s["scales"][1][page, head][..., None, :]
    k = k.reshape(T * H, n * P, dh).transpose(1, 2).contiguous()
    v = v.transpose(3, 4).reshape(T * H, n * P, dh)
    x = torch.matmul(s["q"].to(F32).reshape(T * H, G, dh), k).mul_(1.0 / math.sqrt(dh))
    see = (keep >= 0)[..., None] & (at[..., None] * P + torch.arange(P, device=DEV) <= pos[:, None, None, None])
    x = x.masked_fill_(~see.reshape(T * H, 1, n * P), float("-inf"))
    x = x.sub_(x.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    o = torch.matmul(x, v) / x.sum(-1, keepdim=True).clamp_min(1e-30)
    return o.reshape(T, H * G, dh).to(BF16), keep


# -- one pass ------------------------------------------------------------------------

def _package():
    import __graft_entry__
    return __graft_entry__.load_package()


def run(state):
    s = state
    if not own:
        return {"sample": _plain_sample, "copy": _plain_copy, "index": _plain_index, "attend": _plain_attend}[s["kind"]](s)
    srw = _package()
    if s["kind"] == "sample":
        return srw.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                          min_p=s["min_p"])
    if s["kind"] == "copy":
        srw.kv_copy(s["tensors"], s["src"], s["dst"])
        return s["tensors"]
    pages, index = srw.KvPages(*s["pages"], *s["scales"]), srw.KvIndex(*s["index"])
    if s["kind"] == "index":
        srw.kv_index(pages, index, s["table"], s["lens"], s["cu"])
        return _values(s)
    keep = srw.kv_select(s["q"], pages, index, s["table"], s["lens"], s["cu"], n=s["n"], first=s["first"], last=s["last"])
    return srw.paged_attention(s["q"], pages, s["table"], s["lens"], s["cu"], max_new=s["most"], keep=keep), keep


# -- the same in 64 bits -------------------------------------------------------------

def _exact_sample(case, s):
    B, V = case["B"], case["V"]
    row = lambda x, b: float(x[b]) if isinstance(x, torch.Tensor) else x  # noqa: E731
    f32 = lambda x: float(torch.tensor(x, dtype=F32))  # noqa: E731
    tokens, logs = [], []
    for b in range(B):
        l = s["logits"][b].to(F64)
        t, k, p, least = (f32(row(s[n], b)) for n in ("temperature", "top_k", "top_p", "min_p"))
        if t <= 0:
            tokens.append(int(torch.nonzero(l == l.max())[0]))
            logs.append(0.0)
            continue
        z, order = torch.sort((l - l.max()) / t, descending=True, stable=True)
        count = V if k <= 0 else min(V, int(k))
        mass = torch.softmax(z[:count], 0)
        if p < 1:
            # the first place at which the mass reaches p
            reach = torch.nonzero(torch.cumsum(mass, 0) >= p)
            count = min(count, int(reach[0]) + 1) if len(reach) else count
        if least > 0:
            count = min(count, int((z >= math.log(least)).sum()))
        kept, back = torch.sort(order[:count])
        mass = torch.softmax(z[:count], 0)[back]
        i = min(int(torch.searchsorted(torch.cumsum(mass, 0), s["u"][b].to(F64), right=True)), count - 1)
        tokens.append(int(kept[i]))
        logs.append(float(torch.log(mass[i])))
    return torch.tensor(tokens), torch.tensor(logs, dtype=F64)


def _codes64(x):
    """What the index holds of float32 numbers x: whole numbers and the number
    each stands for."""
    x = x.to(F32)
    m = x.abs().max(-1, keepdim=True).values
    inverse = (127.0 / m.to(F64)).to(F32)                         # rounded once, as the definition does
    return torch.round(x * inverse).to(F64), (m.to(F64) / 127.0).to(F32).to(F64)


def _keys64(case, s, page):
    k = _bits(s["pages"][0])[page].view(s["pages"][0].dtype).to(F32).to(F64)
    return k if case["cache"] == "bf16" else k * s["scales"][0][page].to(F64)[..., None]


def _exact_index(case, s):
    new, total = _lengths(case)
    P = case["P"]
    out = torch.zeros(s["index"][0].shape, dtype=F64, device=DEV)
    for b, (n, t) in enumerate(zip(new, total)):
        ids = s["table"][b].tolist()
        for j in range((t - n) // P, (t - 1) // P + 1):
            have = min(P, t - j * P)
            c, unit = _codes64(_keys64(case, s, ids[j])[:, :have].sum(1) / have)
            out[ids[j]] = c * unit
    return out


def _exact_attend(case, s):
    new, total = _lengths(case)
    H, G, dh, P, n = (case[k] for k in ("H", "G", "dh", "P", "n"))
    out, at = [], 0
    for b, (m, t) in enumerate(zip(new, total)):
        ids = s["table"][b, :-(-t // P)].long()
        codes, unit = (x[ids] for x in s["index"])
        k = _keys64(case, s, ids)                                 # [pages, H, P, dh]
        v = _bits(s["pages"][1])[ids].view(s["pages"][1].dtype).to(F32).to(F64).transpose(2, 3)
        if case["cache"] != "bf16":
            v = v * s["scales"][1][ids].to(F64)[..., None]
        for i in range(m):
            pos = t - m + i
            q = s["q"][at + i].to(F64).reshape(H, G, dh)
            mine = pos // P
            c, _ = _codes64(q.sum(1))
            row = torch.empty(H, G, dh, dtype=F64, device=DEV)
            for h in range(H):
                # (scores as the definition rounds them: one product in 32 bits)
                score = ((codes[:mine + 1, h].to(F64) @ c[h]).to(F32) * unit[:mine + 1, h]).tolist()
                ends = set(range(min(case["first"], mine + 1))) | set(range(max(0, mine - case["last"] + 1), mine + 1))
                rest = sorted((j for j in range(mine + 1) if j not in ends), key=lambda j: (-score[j], j))
                take = sorted(ends | set(rest[:max(0, n - len(ends))]))
                take = torch.tensor(take, device=DEV)
                place = (take[:, None] * P + torch.arange(P, device=DEV)).reshape(-1)
                fine = place <= pos
                kk, vv = (x[take, h].reshape(-1, dh)[fine] for x in (k, v))
                row[h] = torch.softmax(q[h] @ kk.T / math.sqrt(dh), -1) @ vv
            out.append(row.reshape(H * G, dh))
        at += m
    return torch.stack(out), None


def _exact_copy(s):
    for t in s["tensors"]:
        for a, b in zip(s["src"], s["dst"]):
            t.select(1, b).copy_(t.select(1, a))
    return s["tensors"]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "copy":
        return _exact_copy(s)
    if case["kind"] == "attend":
        new, _ = _lengths(case)
        if sum(new) * case["H"] > 6000:  # (about 3 ms each)
            return None
    return {"sample": _exact_sample, "index": _exact_index, "attend": _exact_attend}[case["kind"]](case, s)
