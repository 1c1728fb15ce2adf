"""Performance cases of the paged key/value cache and the attention over it:
the calls that a program serving many sequences of different lengths makes.

A case is a dict of plain values; ``kind`` names the pass:

* ``store``   ``kv_write`` puts the new tokens' keys and values into the pages
              (quantised as they are written where the pages hold 8 bits), and
              ``kv_read`` reads them back;
* ``attend``  ``paged_attention`` of every sequence's new tokens over its
              pages: single tokens, chunks of a prompt, mixed batches, with or
              without a sliding window and first tokens that stay visible.

A sequence b has ``lens[b]`` positions, the last ``cu[b + 1] - cu[b]`` of them
new (one where ``cu`` is None); position p lies in page ``table[b, p // P]`` at
slot ``p % P``.  Pages: k [pages, Hkv, P, dh], v [pages, Hkv, dh, P]; with 8
bits one float32 scale for each token and head, [pages, Hkv, P].
"""

import math
import random

import torch

own = False

DEV = "cuda:0"
BF16, F32, F64, I32, U8 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.uint8
FP8 = torch.float8_e4m3fn
TYPES = {"bf16": BF16, "f32": F32, "int8": torch.int8, "fp8": FP8}
TOP = {"int8": 127.0, "fp8": 448.0}      # the largest code's value
TINY = 2.0 ** -100                       # a row whose largest magnitude is at most this is held as zeros


def _case(new, past, **rest):
    """A case whose sequences have new[0] to new[1] new tokens behind past[0]
    to past[1] positions."""
    return dict(rest, new_lo=new[0], new_hi=new[1], past_lo=past[0], past_hi=past[1])


def listed():
    return [
        # one generated token of each of 64 sequences goes into the cache of one layer of the 40M model
        _case(name="store_step", kind="store", B=64, new=(1, 1), past=(255, 511), Hkv=6, dh=64, P=64, cache="int8",
              src="bf16", out="bf16"),
        # the prompts of 8 sequences of the model's full length
        _case(name="store_prompts", kind="store", B=8, new=(512, 512), past=(0, 0), Hkv=6, dh=64, P=32, cache="fp8",
              src="bf16", out="bf16"),
        # one long document, float32 projections, wide heads
        _case(name="store_long", kind="store", B=1, new=(65521, 65521), past=(9, 9), Hkv=8, dh=128, P=64, cache="int8",
              src="f32", out="f32"),
        # generating for one sequence: the smallest call
        _case(name="step_one", kind="attend", B=1, new=(1, 1), past=(300, 300), Hq=6, Hkv=6, dh=64, P=16, cache="bf16",
              window=0, sinks=0),
        # generating for 64 sequences of the 40M model at different positions
        _case(name="step_batch", kind="attend", B=64, new=(1, 1), past=(130, 511), Hq=6, Hkv=6, dh=64, P=64,
              cache="int8", window=0, sinks=0),
        # generating for 32 long sequences, four query heads to a key head
        _case(name="step_long", kind="attend", B=32, new=(1, 1), past=(4000, 32000), Hq=32, Hkv=8, dh=128, P=64,
              cache="fp8", window=0, sinks=0),
        # generating at the end of one very long sequence
        _case(name="step_deep", kind="attend", B=1, new=(1, 1), past=(200002, 200002), Hq=16, Hkv=2, dh=128, P=128,
              cache="bf16", window=0, sinks=0),
        # the prompts of 8 sequences of the model's full length, nothing cached yet
        _case(name="prompts", kind="attend", B=8, new=(512, 512), past=(0, 0), Hq=6, Hkv=6, dh=64, P=64, cache="bf16",
              window=0, sinks=0),
        # a chunk of a long prompt behind what is cached of it: the largest call
        _case(name="chunk_long", kind="attend", B=1, new=(2048, 2048), past=(30011, 30011), Hq=32, Hkv=8, dh=128, P=64,
              cache="int8", window=0, sinks=0),
        # a batch of generated tokens and pieces of prompts, ragged, small pages
        _case(name="mixed", kind="attend", B=24, new=(1, 300), past=(1, 2000), Hq=8, Hkv=4, dh=64, P=16, cache="fp8",
              window=0, sinks=0),
        # a long prompt with a sliding window, four first tokens visible throughout
        _case(name="window_prompt", kind="attend", B=2, new=(7001, 8003), past=(100, 777), Hq=8, Hkv=2, dh=64, P=64,
              cache="bf16", window=1024, sinks=4),
        # generating without an end: 48 sequences with a sliding window
        _case(name="window_step", kind="attend", B=48, new=(1, 1), past=(500, 20000), Hq=16, Hkv=4, dh=64, P=32,
              cache="int8", window=1000, sinks=4),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """Another case of the listed ranges: other batches, lengths, head
    layouts, pages and types."""
    dh = rng.choice([64, 64, 128])
    cache = rng.choice(["bf16", "int8", "fp8"])
    P = rng.choice([16, 32, 64, 128])
    kind = rng.choice(["store", "step", "step", "chunk", "chunk", "window_step", "window_chunk"])
    if kind == "store":
        n = _log_int(rng, 1, 8000)
        B = _log_int(rng, 1, min(128, max(1, 60000 // n)))
        return _case(kind="store", B=B, new=(max(1, n // 2), n), past=(0, _log_int(rng, 1, 4000)),
                     Hkv=rng.choice([1, 2, 6, 8]), dh=dh, P=P, cache=cache, src=rng.choice(["bf16", "f32"]),
                     out="f32" if cache != "bf16" and rng.random() < 0.5 else "bf16")
    Hkv = rng.choice([1, 2, 4, 6, 8])
    G = rng.choice([1, 2, 4, 8])
    window = _log_int(rng, 100, 4000) if kind.startswith("window") else 0
    sinks = rng.choice([0, 1, 4, 16]) if window else 0
    if kind.endswith("step"):
        past = _log_int(rng, 20, 100000)
        # at most the bytes of step_long and scores that the plain form can hold
        B = _log_int(rng, 1, max(1, min(200, int(4e8 / (past * Hkv * dh)))))
        new = (1, 1)
    else:
        n = _log_int(rng, 2, 4000)
        past = _log_int(rng, 1, 12000)
        B = _log_int(rng, 1, max(1, min(32, int(1e9 / (n * (n + past) * Hkv * G)))))
        new = (max(1, n // 8), n)
    return _case(kind="attend", B=B, new=new, past=(past // 4, past), Hq=Hkv * G, Hkv=Hkv, dh=dh, P=P, cache=cache,
                 window=window, sinks=sinks)


def _lengths(case):
    """(new, total) positions of each sequence: the case's own, whatever the
    seed."""
    rng = random.Random(" ".join("%s=%s" % (k, case[k]) for k in sorted(case) if k != "name"))
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["B"])]
    return new, [n + rng.randint(case["past_lo"], case["past_hi"]) for n in new]


def _visible(case, first, last):
    """How many positions the queries at first..last see together."""
    if not case["window"]:
        return last + 1
    lo = max(0, first - case["window"] + 1)
    return last + 1 - lo + min(case["sinks"], lo)


def _seen(case, p):
    return _visible(case, p, p)


def work(case):
    new, total = _lengths(case)
    T, Hkv, dh = sum(new), case["Hkv"], case["dh"]
    held = 2 * dh * (2 if case["cache"] == "bf16" else 1) + (0 if case["cache"] == "bf16" else 8)
    if case["kind"] == "store":
        size = {"bf16": 2, "f32": 4}
        return {"bytes": T * Hkv * (2 * dh * (size[case["src"]] + size[case["out"]]) + 2 * held),
                "flops": T * Hkv * dh * (2 if case["cache"] == "bf16" else 8)}
    keys = sum(_visible(case, t - n, t - 1) for n, t in zip(new, total))
    if not case["window"]:
        rows = sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, total))
    else:
        rows = sum(_seen(case, p) for n, t in zip(new, total) for p in range(t - n, t))
    return {"bytes": keys * Hkv * held + 2 * T * case["Hq"] * dh * 2, "flops": 4 * rows * case["Hq"] * dh}


# -- inputs ------------------------------------------------------------------------

def _addresses(case, g):
    new, total = _lengths(case)
    P, B = case["P"], case["B"]
    need = [-(-t // P) for t in total]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(I32)
    width = max(need)
    at = torch.arange(width, device=DEV)[None]
    count = torch.tensor(need, device=DEV)[:, None]
    first = torch.cumsum(count, 0) - count
    table = torch.where(at < count, order[(first + at).clamp_max(pages - 1)], torch.full((), -1, dtype=I32, device=DEV))
    lens = torch.tensor(total, dtype=I32, device=DEV)
    cu = None if max(new) == 1 else torch.tensor([sum(new[:i]) for i in range(B + 1)], dtype=I32, device=DEV)
    return pages, table.contiguous(), lens, cu, sum(new), max(new)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    pages, table, lens, cu, T, most = _addresses(case, g)
    Hkv, dh, P, kind = case["Hkv"], case["dh"], case["P"], case["cache"]
    s = dict(case, table=table, lens=lens, cu=cu, T=T, most=most)

    def held(shape):
        x = torch.randn(shape, generator=g, device=DEV, dtype=BF16)
        if kind == "int8":
            return (x * 42.0).clamp_(-127.0, 127.0).round_().to(torch.int8)
        return (x * 150.0).clamp_(-448.0, 448.0).to(FP8) if kind == "fp8" else x

    def scales():
        # tokens of different sizes
        size = torch.exp(0.3 * torch.randn(pages, Hkv, P, generator=g, device=DEV))
        return size / (42.0 if kind == "int8" else 150.0)

    s["pages"] = [held((pages, Hkv, P, dh)), held((pages, Hkv, dh, P))]
    s["scales"] = [None, None] if kind == "bf16" else [scales(), scales()]
    if case["kind"] == "store":
        size = torch.exp(0.3 * torch.randn(T, Hkv, 1, generator=g, device=DEV))
        s["new"] = [(torch.randn(T, Hkv, dh, generator=g, device=DEV) * size).to(TYPES[case["src"]]) for _ in range(2)]
    else:
        s["q"] = torch.randn(T, case["Hq"], dh, generator=g, device=DEV).to(BF16)
    return s


# -- the plain forms ---------------------------------------------------------------

def _places(s):
    """(page, slot) of each new token."""
    at = torch.arange(s["T"], device=DEV)
    if s["cu"] is None:
        seq, pos = at, s["lens"].long() - 1
    else:
        cu = s["cu"].long()
        seq = torch.searchsorted(cu, at, right=True) - 1
        pos = s["lens"].long()[seq] - cu[seq + 1] + at
    return s["table"].long()[seq, pos // s["P"]], pos % s["P"]


def _codes(x, kind):
    """(codes, scales) of rows of 8 bits: the largest magnitude is the
    largest code."""
    x = x.to(F32)
    most = x.abs().amax(-1)
    fine = most > TINY
    zero, top = torch.zeros_like(most), torch.full_like(most, TOP[kind])   # (a number / a tensor is two roundings)
    y = x * torch.where(fine, top / most, zero)[..., None]
    return (torch.round(y) if kind == "int8" else y).to(TYPES[kind]), torch.where(fine, most / top, zero)


def _bits(t):
    """fp8 pages are indexed as bytes."""
    return t.view(U8) if t.dtype == FP8 else t


def _plain_store(s):
    page, slot = _places(s)
    head = torch.arange(s["Hkv"], device=DEV)[None]
    at = (page[:, None], head, slot[:, None])
    d = torch.arange(s["dh"], device=DEV)
    at_v = (page[:, None, None], head[..., None], d, slot[:, None, None])
    got = []
    for x, pages, scales, i in ((s["new"][0], s["pages"][0], s["scales"][0], at),
                                (s["new"][1], s["pages"][1], s["scales"][1], at_v)):
        if s["cache"] == "bf16":
            pages[i] = x.to(BF16)
            got.append(pages[i])
            continue
        c, sc = _codes(x, s["cache"])
        _bits(pages)[i] = _bits(c)
        scales[at] = sc
        got.append((_bits(pages)[i].view(pages.dtype).to(F32) * scales[at][..., None]).to(TYPES[s["out"]]))
    return got


def _plain_attend(s):
    B, Hq, Hkv, dh, P, T, most = (s[k] for k in ("B", "Hq", "Hkv", "dh", "P", "T", "most"))
    G, L = Hq // Hkv, s["table"].shape[1] * P
    page = s["table"].long().clamp_min(0)                                  # [B, pages of the longest]
    k, v = (_bits(t)[page].view(t.dtype).to(F32) for t in s["pages"])      # [B, W, Hkv, P, dh], [B, W, Hkv, dh, P]
    if s["cache"] != "bf16":
        k = k * s["scales"][0][page][..., None]
        v = v * s["scales"][1][page][..., None, :]
    k = k.permute(0, 2, 4, 1, 3).reshape(B, Hkv, dh, L)
    v = v.permute(0, 2, 1, 4, 3).reshape(B, Hkv, L, dh)
    lens = s["lens"].long()
    cu = torch.arange(B + 1, device=DEV) if s["cu"] is None else s["cu"].long()
    n = cu[1:] - cu[:-1]
    i = torch.arange(most, device=DEV)[None]
    row = (cu[:-1, None] + i).clamp_max(T - 1)                             # [B, most]: the packed rows, padded
    q = s["q"][row].to(F32).reshape(B, most, Hkv, G, dh).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * most, dh)
    pos = (lens - n)[:, None] + i
    key = torch.arange(L, device=DEV)
    see = (key <= pos[..., None]) & (i < n[:, None])[..., None]
    if s["window"]:
        see = see & ((key > pos[..., None] - s["window"]) | (key < s["sinks"]))
    x = torch.matmul(q, k).mul_(1.0 / math.sqrt(dh)).reshape(B, Hkv, G, most, L)
    x = x.masked_fill_(~see[:, None, None], float("-inf"))
    x = x.sub_(x.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    den = x.sum(-1, keepdim=True)
    o = torch.matmul(x.reshape(B, Hkv, G * most, L), v).reshape(B, Hkv, G, most, dh) / den.clamp_min(1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(B * most, Hq, dh)
    at = torch.arange(T, device=DEV)
    seq = torch.searchsorted(cu, at, right=True) - 1
    return o[seq * most + at - cu[seq]].to(BF16)


# -- one pass ------------------------------------------------------------------------

def _package():
    import __graft_entry__
    return __graft_entry__.load_package()


def run(state):
    s = state
    if not own:
        return _plain_store(s) if s["kind"] == "store" else _plain_attend(s)
    srw = _package()
    pages = srw.KvPages(*s["pages"], *s["scales"])
    if s["kind"] == "store":
        srw.kv_write(pages, *s["new"], s["table"], s["lens"], s["cu"])
        return list(srw.kv_read(pages, s["table"], s["lens"], s["cu"], total=s["T"], dtype=TYPES[s["out"]]))
    return srw.paged_attention(s["q"], pages, s["table"], s["lens"], s["cu"], max_new=s["most"], window=s["window"],
                               sinks=s["sinks"])


# -- the same in 64 bits -------------------------------------------------------------

def _held64(x, kind):
    """What 8 bits hold of x, from the formats' definitions."""
    x = x.to(F64)
    if kind == "bf16":
        return x.to(BF16).to(F64)
    unit = x.abs().amax(-1, keepdim=True) / TOP[kind]
    y = x / unit
    if kind == "int8":
        return torch.round(y) * unit
    # 3 bits behind the leading one down to 2^-6, steps of 2^-9 below
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / step) * step * unit


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "store":
        return [_held64(x, case["cache"]) for x in s["new"]]
    new, total = _lengths(case)
    Hkv, dh = case["Hkv"], case["dh"]
    G = case["Hq"] // Hkv
    out, at = [], 0
    for b, (n, t) in enumerate(zip(new, total)):
        ids = s["table"][b, :-(-t // case["P"])].long()
        got = torch.empty(n, Hkv, G, dh, dtype=F64, device=DEV)
        for h in range(Hkv):
            k, v = (_bits(x)[ids, h].view(x.dtype).to(F32).to(F64) for x in s["pages"])
            v = v.transpose(1, 2)
            if case["cache"] != "bf16":
                k = k * s["scales"][0][ids, h].to(F64)[..., None]
                v = v * s["scales"][1][ids, h].to(F64)[..., None]
            k, v = (x.reshape(-1, dh)[:t].contiguous() for x in (k, v))
            step = max(1, int(1e8 // (t * G)))
            for a in range(0, n, step):
                e = min(n, a + step)
                # the keys that these rows can see: all, or the first ones and the window's
                lo = max(0, t - n + a - case["window"] + 1) if case["window"] else 0
                first = min(case["sinks"], lo)
                keys = torch.cat([torch.arange(first, device=DEV), torch.arange(lo, t - n + e, device=DEV)])
                q = s["q"][at + a:at + e, h * G:(h + 1) * G].to(F64).reshape((e - a) * G, dh)
                z = (q @ k[keys].T / math.sqrt(dh)).reshape(e - a, G, -1)
                p = torch.arange(t - n + a, t - n + e, device=DEV)[:, None]
                hide = keys > p
                if case["window"]:
                    hide |= (keys <= p - case["window"]) & (keys >= case["sinks"])
                z = torch.softmax(z.masked_fill(hide[:, None], float("-inf")), -1)
                got[a:e, h] = (z.reshape((e - a) * G, -1) @ v[keys]).reshape(e - a, G, dh)
        out.append(got.reshape(n, case["Hq"], dh))
        at += n
    return torch.cat(out)
