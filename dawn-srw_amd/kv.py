"""The paged key/value cache and the attention over it: torch tensors in,
torch tensors out, every computation in libsrw_amd.so's HIP kernels.

A layer's pages (:class:`KvPages`) hold ``page_size`` positions of every
key/value head, in bf16 or in 8 bits with a float32 scale for each token and
head.  Sequences of any lengths share them: a call describes its sequences by

* ``table`` [B, width] int32: the page of each run of ``page_size`` positions
  (an entry that names no page, -1 say, holds nothing and is not seen);
* ``lens`` [B] int32: the sequences' lengths, the call's new tokens included;
* ``cu`` [B + 1] int32: sequence b's new tokens are the packed rows
  [cu[b], cu[b + 1]) of T and lie at its last positions; None: one each.
  cu[0] is 0 and cu[B] is T: rows of an output that no sequence names are not
  written.

All three are device tensors that only the kernels read: the functions wait for
nothing on the GPU.  :func:`kv_write` stores new tokens, :func:`kv_read` reads
tokens back, :func:`paged_attention` attends from new tokens to everything
before them.  :class:`PagedKvCache` keeps the pages of all layers of a model and
hands them out to sequences; its ``extend`` copies a call's table to the device,
which waits.
"""

from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import operator
import os
import struct

import torch
from torch.autograd import forward_ad

from . import _capi as C

__all__ = ["KvPages", "PagedKvCache", "kv_write", "kv_read", "paged_attention"]

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
_KINDS = {torch.bfloat16: C.SRW_KV_BF16, torch.int8: C.SRW_KV_INT8, torch.float8_e4m3fn: C.SRW_KV_FP8}
_DTYPES = {torch.float32: C.SRW_F32, torch.bfloat16: C.SRW_BF16}

# srw_kv_t, srw_kv_rows_t and srw_attention_t as bytes (packed in a fraction of the
# time that a ctypes structure takes to fill)
_KV = struct.Struct("@7P5q4i")
_ROWS = struct.Struct("@2P4q")
_ATTENTION = struct.Struct("@7P5q4i2P2q4if4x")


_host = None
_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _native():
    """The calls' native host side (csrc/srw_host.cpp), which takes calls whose
    tensors are as the C entry points take them and answers None for any other:
    those go through the checks and copies here.  (64 single tokens of 6 heads:
    the kernel takes 10 us, the call from Python took 12, through this 5.)"""
    global _host
    if _host is None:
        C.load_library()
        path = os.path.join(os.path.dirname(C.LIB_PATH), "_srw_host.so")
        if not os.path.exists(path):
            raise C.SrwLibraryError(f"{path} is not built; run __graft_entry__.build() first")
        spec = importlib.util.spec_from_file_location(
            "_srw_host", path, loader=importlib.machinery.ExtensionFileLoader("_srw_host", path))
        _host = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(_host)
    return _host


def _tensor(name, t, dev, dtype, shape):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype is dtype and t.shape == shape and t.device == dev and t.is_contiguous():
        return t.data_ptr()
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, expected {dev}")
    if t.dtype != dtype:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    raise ValueError(f"{name} must be contiguous")


class KvPages:
    """One layer's pages: ``k`` [n_pages, H, page_size, head_dim], ``v``
    [n_pages, H, head_dim, page_size] (dimension by dimension, as the
    attention's matrix products read it), both bfloat16, int8 or
    float8_e4m3fn; 8-bit pages with ``k_scale`` and ``v_scale`` [n_pages, H,
    page_size] float32.  Holds the tensors, which the calls read and write in
    place."""

    __slots__ = ("_t", "n_pages", "heads", "page_size", "head_dim", "kind", "device")

    def __init__(self, k, v, k_scale=None, v_scale=None):
        self._t = (k, v, k_scale, v_scale)
        at = (_host or _native()).pages(self._t)
        if at is None:
            at = self._at[4:]
        self.n_pages, self.heads, self.page_size, self.head_dim, self.kind, _ = at
        self._t += tuple(at)  # as they were taken
        self.device = k.device

    k = property(lambda self: self._t[0])
    v = property(lambda self: self._t[1])
    k_scale = property(lambda self: self._t[2])
    v_scale = property(lambda self: self._t[3])

    @property
    def _at(self):
        """(k, v, k_scale, v_scale addresses, n_pages, heads, page_size, head_dim,
        kind, device) of the tensors as they are now."""
        k, v, k_scale, v_scale = self._t[:4]
        if not isinstance(k, torch.Tensor) or k.dim() != 4:
            raise ValueError("k must be a tensor [n_pages, heads, page_size, head_dim]")
        n, h, p, d = k.shape
        dev = k.device
        if dev.type != "cuda":
            raise ValueError(f"the cache lives on a HIP device; got {dev}")
        if k.dtype not in _KINDS:
            raise TypeError(f"pages hold bfloat16, int8 or float8_e4m3fn; got {k.dtype}")
        if not k.is_contiguous():
            raise ValueError("k must be contiguous")
        kind, v_at, scales = _KINDS[k.dtype], _tensor("v", v, dev, k.dtype, (n, h, d, p)), (0, 0)
        if kind != C.SRW_KV_BF16:
            scales = (_tensor("k_scale", k_scale, dev, F32, (n, h, p)), _tensor("v_scale", v_scale, dev, F32, (n, h, p)))
        elif k_scale is not None or v_scale is not None:
            raise ValueError("bfloat16 pages have no scales")
        return (k.data_ptr(), v_at, *scales, n, h, p, d, kind, dev.index)


def _no_grad(name, t):
    # (tangents are of a level: outside of one there are none to look for)
    if (t.requires_grad and torch.is_grad_enabled()
            or forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None):
        raise NotImplementedError(f"{name} requires a gradient; the paged cache's calls have none (torch.no_grad())")


def _written(*tensors):
    """Counts the tensors as changed in place."""
    for t in tensors:
        if t is not None and not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _address(pages, table, lens, cu, T):
    """The fields of srw_kv_t: a call's sequences over these pages."""
    dev = pages.device
    if not isinstance(lens, torch.Tensor) or lens.dim() != 1:
        raise ValueError("lens must be a tensor [B]")
    B = lens.shape[0]
    lens_at = _tensor("lens", lens, dev, I32, (B,))
    if not isinstance(table, torch.Tensor) or table.dim() != 2 or table.shape[0] != B:
        raise ValueError(f"table must be a tensor [{B}, width]")
    if table.dtype is not I32 or table.device != dev:
        raise TypeError(f"table must be int32 on {dev}; got {table.dtype} on {table.device}")
    width = table.shape[1]
    stride, step = table.stride()
    if step != 1 and width > 1 or stride < width and B > 1:
        raise ValueError("rows of table must be consecutive")
    if cu is not None:
        cu_at = _tensor("cu", cu, dev, I32, (B + 1,))
    elif T == B:
        cu_at = 0
    else:
        raise ValueError(f"{T} tokens of {B} sequences need cu")
    at = pages._at
    if at[4:] != pages._t[4:]:
        raise ValueError("the pages' tensors have changed since KvPages took them")
    for name, t in zip(("k", "v", "k_scale", "v_scale"), pages._t):
        if t is not None:
            _no_grad("the pages' " + name, t)
    return (*at[:4], table.data_ptr(), lens_at, cu_at, B, T, pages.n_pages, width,
            stride if stride > width else width, pages.heads, pages.head_dim, pages.page_size, pages.kind)


def _rows(name, t, pages, T, dtypes, unit):
    """(t, token stride, head stride) of t [T, heads, head_dim] with consecutive
    dims; rows that the kernels cannot take as they lie (other strides or
    alignment) are copied.  (The stride of a single token or head is never used,
    and may be anything.)"""
    if not isinstance(t, torch.Tensor) or t.dim() != 3 or t.shape[2] != pages.head_dim or t.shape[0] != T:
        got = tuple(t.shape) if isinstance(t, torch.Tensor) else type(t)
        raise ValueError(f"{name} must be [{T}, heads, {pages.head_dim}]; got {got}")
    if t.device != pages.device:
        raise ValueError(f"{name} is on {t.device}, expected {pages.device}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {' or '.join(str(d) for d in dtypes)}")
    _no_grad(name, t)
    H, d = t.shape[1:]
    s0, s1, s2 = t.stride()
    s0, s1 = H * d if T == 1 else s0, d if H == 1 else s1
    if s2 != 1 or s0 % unit or s1 % unit or t.data_ptr() % (unit * t.element_size()):
        t, s0, s1 = t.clone(memory_format=torch.contiguous_format), H * d, d
    return t, s0, s1


def _check_window(window, sinks):
    if not (type(window) is int is type(sinks) or hasattr(window, "__index__") and hasattr(sinks, "__index__")):
        raise TypeError(f"window and sinks are whole numbers; got {window!r} and {sinks!r}")
    if window < 0 or sinks < 0 or (sinks and not window):
        raise ValueError("window and sinks are not negative, and sinks need a window")


def _call(f, dev, *args):
    """f's status with the current stream of dev as its last argument (launches
    go to the current device's streams)."""
    stream = _raw_stream(dev.index)
    if _current_device() == dev.index:
        return f(*args, stream)
    with torch.cuda.device(dev):
        return f(*args, stream)


def kv_write(pages: KvPages, k, v, table, lens, cu=None) -> None:
    """Store the new tokens' keys and values (``k``, ``v`` [T, heads,
    head_dim], bfloat16 or float32, any token and head strides) into the pages,
    rounded to bfloat16 or quantised: a row x of one token and head as codes of
    x * (127 / m) (int8) or x * (448 / m) (fp8) with scale m / 127 or m / 448,
    m its largest magnitude.  Rows of at most 2^-100 are held as zeros; a row
    with an infinity or NaN reads back as NaN.  Tokens whose position has no
    page are left out; all other slots keep what they hold."""
    if _current_device() == pages.device.index:
        status = (_host or _native()).write(pages._t, k, v, table, lens, cu, _raw_stream(pages.device.index))
        if status is not None:
            return C.check(status)
    T = k.shape[0] if isinstance(k, torch.Tensor) and k.dim() else -1
    a = _address(pages, table, lens, cu, T)
    k, *ks = _rows("k", k, pages, T, _DTYPES, 4)
    v, *vs = _rows("v", v, pages, T, (k.dtype,), 4)
    if k.shape[1] != pages.heads or v.shape[1] != pages.heads:
        raise ValueError(f"k and v have {k.shape[1]} and {v.shape[1]} heads, the pages {pages.heads}")
    r = _ROWS.pack(k.data_ptr(), v.data_ptr(), *ks, *vs)
    C.check(_call(C.load_library().srw_kv_write, pages.device, _KV.pack(*a), r, _DTYPES[k.dtype]))
    _written(*pages._t[:4])


def kv_read(pages: KvPages, table, lens, cu=None, *, total=None, dtype=BF16):
    """(k, v) [T, heads, head_dim] in ``dtype`` (bfloat16 or float32) of the
    tokens that (lens, cu) describe -- with cu from cumulated lens, whole
    sequences.  ``total`` is T, which lies on the device (cu's last entry);
    None where cu is None.  Positions without a page give zeros."""
    if dtype not in _DTYPES:
        raise TypeError(f"kv_read gives float32 or bfloat16, not {dtype}")
    if cu is not None and total is None:
        raise ValueError("total, the number of tokens, is needed with cu")
    T = int(total) if total is not None else lens.shape[0]
    if _current_device() == pages.device.index:
        got = (_host or _native()).read(pages._t, table, lens, cu, T, dtype is F32, _raw_stream(pages.device.index))
        if got is not None:
            return got
    a = _address(pages, table, lens, cu, T)
    H, d = pages.heads, pages.head_dim
    k = torch.empty((T, H, d), dtype=dtype, device=pages.device)
    v = torch.empty_like(k)
    r = _ROWS.pack(k.data_ptr(), v.data_ptr(), H * d, d, H * d, d)
    C.check(_call(C.load_library().srw_kv_read, pages.device, _KV.pack(*a), r, _DTYPES[dtype]))
    return k, v


def paged_attention(q, pages: KvPages, table, lens, cu=None, *, max_new: int = 0, scale=None, window: int = 0,
                    sinks: int = 0, out=None):
    """Attention of the new tokens ``q`` [T, n_heads, head_dim] (bfloat16, any
    token and head strides; n_heads a multiple of the pages' heads) over their
    sequences' pages, which must hold the new tokens already: a token at
    position i sees the positions j <= i, with ``window`` > 0 those with j > i
    - window or j < ``sinks``.  ``scale`` multiplies the scores (default 1 /
    sqrt(head_dim)).  ``max_new``: the most new tokens of one sequence, where
    the caller knows it.  Returns ``out`` [T, n_heads, head_dim] bfloat16; a
    token that sees nothing gets zeros.

    Sums and statistics are float32.  The softmax weights enter the second
    product as one bfloat16 in calls of many rows, as two (16 bits) in calls of
    few.  Which kernel and how many splits a call gets goes by ``max_new``, its
    rows, heads and the table's width: a sequence's outputs are the same bit for
    bit in calls that agree in these, and within these roundings in any."""
    scale = pages.head_dim ** -0.5 if scale is None else float(scale)
    if out is None and _current_device() == pages.device.index:
        got = (_host or _native()).attention(pages._t, q, table, lens, cu, max_new, scale, window, sinks,
                                             _raw_stream(pages.device.index))
        if got is not None:
            return got
    T = q.shape[0] if isinstance(q, torch.Tensor) and q.dim() else -1
    kv = _address(pages, table, lens, cu, T)
    q, *qs = _rows("q", q, pages, T, (BF16,), 8)
    Hq = q.shape[1]
    if Hq < 1 or Hq % pages.heads:
        raise ValueError(f"{Hq} query heads are no multiple of the pages' {pages.heads}")
    _check_window(window, sinks)
    if max_new < 0:
        raise ValueError("max_new is not negative")
    dev = pages.device
    given = out is not None
    if given:
        _tensor("out", out, dev, BF16, (T, Hq, pages.head_dim))
        _no_grad("out", out)
    else:
        out = torch.empty((T, Hq, pages.head_dim), dtype=BF16, device=dev)
    a = _ATTENTION.pack(*kv, q.data_ptr(), out.data_ptr(), *qs, Hq, max_new, window, sinks, scale)
    lib = C.load_library()
    status = _call(lib.srw_attention, dev, a, None, 0)
    if status == C.SRW_EWORKSPACE:  # splits to join, nothing launched yet
        need = ctypes.c_size_t(0)
        C.check(lib.srw_attention_workspace_size(a, ctypes.byref(need)))
        ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
        status = _call(lib.srw_attention, dev, a, ws.data_ptr(), need.value)
    C.check(status)
    if given:
        _written(out)
    return out


class PagedKvCache:
    """Pages of all layers of a model and the sequences that hold them.

    ``layer(i)`` is layer i's :class:`KvPages`; a page id names the same page
    of every layer.  ``add()`` opens a sequence, ``extend(seqs, counts)``
    makes room for that many new tokens of each and returns the call's
    (table, lens, cu, max_new) on the device, ``free(seq)`` gives its pages
    back.  With a sliding window, ``evict(seq, window, sinks)`` gives back
    the pages that no later token sees."""

    def __init__(self, n_layers: int, n_pages: int, n_heads: int, head_dim: int, *, page_size: int = 64, dtype=BF16,
                 device="cuda:0"):
        dev = torch.device(device)
        if dtype not in _KINDS:
            raise TypeError(f"pages hold bfloat16, int8 or float8_e4m3fn; got {dtype}")
        if head_dim not in (64, 128) or page_size not in (16, 32, 64, 128, 256):
            raise ValueError("head_dim is 64 or 128 and page_size 16, 32, 64, 128 or 256")
        if min(n_layers, n_pages, n_heads) < 1:
            raise ValueError("n_layers, n_pages and n_heads are at least 1")
        if dev.type == "cuda" and dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.page_size, self.n_pages, self.device, self.dtype = page_size, n_pages, dev, dtype
        shape = (n_layers, n_pages, n_heads)
        self.k = torch.empty(*shape, page_size, head_dim, dtype=dtype, device=dev)
        self.v = torch.empty(*shape, head_dim, page_size, dtype=dtype, device=dev)
        self.k_scale = self.v_scale = None
        if dtype != BF16:
            self.k_scale, self.v_scale = (torch.empty(*shape, page_size, device=dev) for _ in range(2))
        self._free = list(range(n_pages - 1, -1, -1))
        self._pages, self._lens, self._next = {}, {}, 0

    def layer(self, i: int) -> KvPages:
        if self.dtype == BF16:
            return KvPages(self.k[i], self.v[i])
        return KvPages(self.k[i], self.v[i], self.k_scale[i], self.v_scale[i])

    def add(self) -> int:
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._lens[seq] = [], 0
        return seq

    def length(self, seq: int) -> int:
        return self._lens[seq]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def extend(self, seqs, counts):
        """Room for counts[i] (0 or more) further tokens of seqs[i]; (table, lens, cu,
        max_new) of the call that writes and attends to them, copied to the device
        (which waits for it).  Raises MemoryError where the free pages do not do;
        whatever it raises, nothing has changed."""
        if len(seqs) != len(counts) or len(set(seqs)) != len(seqs):
            raise ValueError("one count for each of different sequences")
        counts = [operator.index(n) for n in counts]
        need = {}
        for s, n in zip(seqs, counts):
            if s not in self._lens:
                raise KeyError(f"no sequence {s}")
            if n < 0:
                raise ValueError("counts are not negative")
            need[s] = -(-(self._lens[s] + n) // self.page_size) - len(self._pages[s])
        if sum(need.values()) > len(self._free):
            raise MemoryError(f"{sum(need.values())} pages are needed, {len(self._free)} are free")
        for s, n in zip(seqs, counts):
            self._pages[s].extend(self._free.pop() for _ in range(need[s]))
            self._lens[s] += n
        try:
            return self._call_of(seqs, counts)
        except BaseException:
            self._take_back(seqs, counts)
            raise

    def _call_of(self, seqs, counts):
        width = max((len(self._pages[s]) for s in seqs), default=0)
        # one copy to the device: the table's rows, then lens, then cu
        host, at = [], 0
        for s in seqs:
            host += self._pages[s] + [-1] * (width - len(self._pages[s]))
        host += [self._lens[s] for s in seqs] + [0]
        for n in counts:
            at += n
            host.append(at)
        B = len(seqs)
        t = torch.tensor(host, dtype=I32).to(self.device)
        table, lens, cu = t[:B * width].view(B, width), t[B * width:B * width + B], t[B * width + B:]
        most = max(counts, default=0)
        return table, lens, None if most == 1 and min(counts) == 1 else cu, most

    def _take_back(self, seqs, counts):
        """What extend did, undone for a call that failed after it."""
        for s, n in reversed(list(zip(seqs, counts))):
            self._lens[s] -= n
            pages = self._pages[s]
            while len(pages) > -(-self._lens[s] // self.page_size):
                self._free.append(pages.pop())

    def evict(self, seq: int, window: int, sinks: int = 0) -> int:
        """Give back the pages that hold only positions which a token at
        position length(seq) or later does not see under this window; returns
        their number."""
        if window < 1 or sinks < 0:
            raise ValueError("evict needs a window, and sinks are not negative")
        P, pages, n = self.page_size, self._pages[seq], 0
        for i in range(-(-sinks // P), len(pages)):
            if (i + 1) * P > self._lens[seq] - window + 1:
                break
            if pages[i] >= 0:
                self._free.append(pages[i])
                pages[i] = -1
                n += 1
        return n

    def free(self, seq: int) -> None:
        self._free.extend(p for p in reversed(self._pages.pop(seq)) if p >= 0)
        del self._lens[seq]
