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
before them, or to a few pages of it: :func:`kv_index` keeps an index of what the
pages' keys are about (:class:`KvIndex`), :func:`kv_select` chooses pages by it.
:func:`kv_copy` copies pages.  :class:`PagedKvCache` keeps the pages of all layers
of a model and hands them out to sequences, which can branch (``fork``); its
``extend`` copies a call's table to the device, which waits.
"""

from __future__ import annotations

import array
import ctypes
import importlib.machinery
import importlib.util
import operator
import os
import struct

import torch
from torch.autograd import forward_ad

from . import _capi as C

__all__ = ["KvPages", "KvIndex", "PagedKvCache", "kv_write", "kv_read", "kv_copy", "kv_index", "kv_select",
           "paged_attention"]

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
_KINDS = {torch.bfloat16: C.SRW_KV_BF16, torch.int8: C.SRW_KV_INT8, torch.float8_e4m3fn: C.SRW_KV_FP8}
_DTYPES = {torch.float32: C.SRW_F32, torch.bfloat16: C.SRW_BF16}

# srw_kv_t, srw_kv_rows_t, srw_attention_t, srw_kv_index_t, srw_kv_select_t and
# srw_kv_copy_t as bytes (packed in a fraction of the time that a ctypes structure
# takes to fill)
_KV = struct.Struct("@7P5q4i")
_ROWS = struct.Struct("@2P4q")
_ATTENTION = struct.Struct("@7P5q4i2P2q4if4x")
_INDEX = struct.Struct("@2P")
_SELECT = struct.Struct("@7P5q4i4P2q4i")
_COPY = struct.Struct("@16P24q4q2P2i")


_ANY_TOKENS = 1 << 29  # kv_index: more than a call has new tokens, as many as it takes

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


class KvIndex:
    """The index of one layer's pages: ``codes`` [n_pages, H, head_dim] int8 and
    ``scale`` [n_pages, H] float32, the mean of a page's keys of each head in 8 bits
    (:func:`kv_index`).  Holds the tensors, which the calls read and write in
    place."""

    __slots__ = ("_t",)

    def __init__(self, codes, scale):
        self._t = (codes, scale)
        if not (_host or _native()).index_pair(self._t):
            self._at(None)

    codes = property(lambda self: self._t[0])
    scale = property(lambda self: self._t[1])

    def _at(self, pages):
        """(codes, scale addresses) of the tensors as they are now, of these pages."""
        codes, scale = self._t
        if not isinstance(codes, torch.Tensor) or codes.dim() != 3:
            raise ValueError("codes must be a tensor [n_pages, heads, head_dim]")
        dev, shape = codes.device, codes.shape
        if pages is not None:
            dev, shape = pages.device, (pages.n_pages, pages.heads, pages.head_dim)
        elif dev.type != "cuda":
            raise ValueError(f"the cache lives on a HIP device; got {dev}")
        at = _tensor("codes", codes, dev, torch.int8, shape), _tensor("scale", scale, dev, F32, shape[:2])
        _no_grad("the index's scale", scale)
        return at


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


def _page_tensors(tensors):
    if isinstance(tensors, KvPages):
        return [t[None] for t in tensors._t[:4] if t is not None]
    return list(tensors)


def kv_copy(tensors, src, dst, *, to=None) -> None:
    """Copy pages: page ``dst[i]`` of every tensor and layer gets what page ``src[i]``
    holds.  ``tensors``: a :class:`KvPages`, or up to eight tensors [layers, n_pages,
    ...] of any types, each layer contiguous (tensors' layers may lie between each
    other's) -- a cache's keys, values, scales and index; ``to``: tensors of the same layouts, with a number of pages of their own, that
    get the pages (None: the same ones).  ``src`` and ``dst`` are sequences of whole
    numbers on the host, of one length; the call waits for nothing, and one captured in
    a graph copies these pages in every replay.  A page may be read several times; one
    that is written twice, or both read and written, is refused."""
    a = _page_tensors(tensors)
    b = a if to is None else _page_tensors(to)
    if not a or len(a) != len(b) or len(a) > C.COPY_TENSORS:
        raise ValueError(f"1 to {C.COPY_TENSORS} tensors, and as many to copy to; got {len(a)} and {len(b)}")
    if isinstance(src, torch.Tensor) or isinstance(dst, torch.Tensor):
        raise TypeError("src and dst are sequences of whole numbers on the host")
    try:
        src, dst = array.array("i", src), array.array("i", dst)
    except OverflowError:
        raise ValueError("src and dst name pages") from None
    if len(src) != len(dst):
        raise ValueError(f"{len(src)} pages to read and {len(dst)} to write")
    if to is None and isinstance(a[0], torch.Tensor) and a[0].is_cuda:
        at = _current_device()
        if (_host or _native()).copy(a, src, dst, at, _raw_stream(at)) is not None:
            return
    shape = None
    at, size, strides = ([], []), [], ([], [])
    for x, y in zip(a, b):
        for which, t in enumerate((x, y)):
            if not isinstance(t, torch.Tensor) or t.dim() < 2:
                raise ValueError("tensors must be [layers, n_pages, ...]")
            if shape is None:
                other = b[0].shape[1] if isinstance(b[0], torch.Tensor) and b[0].dim() > 1 else -1
                dev, shape = t.device, (t.shape[0], [t.shape[1], other])
                if dev.type != "cuda":
                    raise ValueError(f"the cache lives on a HIP device; got {dev}")
            if t.device != dev:
                raise ValueError(f"a tensor is on {t.device}, expected {dev}")
            if t.shape[0] != shape[0] or t.shape[1] != shape[1][which]:
                raise ValueError(f"tensors of {shape[0]} layers and {shape[1][which]} pages; got one of shape {tuple(t.shape)}")
            _no_grad("a tensor", t)
            if t.numel() and not t[0].is_contiguous():
                raise ValueError("a layer's pages must be contiguous")
            at[which].append(t.data_ptr())
            strides[which].append(t.stride(0) * t.element_size())
        if x.dtype != y.dtype or x.shape[2:] != y.shape[2:]:
            raise ValueError(f"pages of {x.dtype} {tuple(x.shape[2:])} cannot be copied to {y.dtype} {tuple(y.shape[2:])}")
        n = x.element_size()
        for d in x.shape[2:]:
            n *= d
        if n % 4 or n == 0:
            raise ValueError(f"pages of {n} bytes, no multiple of 4")
        size.append(n)
    if not len(src) or not shape[0]:
        return
    z = [0] * (C.COPY_TENSORS - len(a))
    c = _COPY.pack(*at[0], *z, *at[1], *z, *size, *z, *strides[0], *z, *strides[1], *z, shape[0], *shape[1], len(src),
                   src.buffer_info()[0], dst.buffer_info()[0], len(a), 0)
    status = _call(C.load_library().srw_kv_copy, dev, c)
    if status == C.SRW_EINVAL:
        raise ValueError("src and dst must name pages, none of them written twice or both read and written, of tensors "
                         "that do not overlap")
    C.check(status)
    _written(*b)


def kv_index(pages: KvPages, index: KvIndex, table, lens, cu=None, *, total=None) -> None:
    """Bring the index's entries of the pages that hold the call's new tokens up to
    date with what the pages hold of them (:func:`kv_write` before): of every page and
    head the mean of its keys at positions before ``lens``, m its largest magnitude,
    as codes round(mean * (127 / m)) with scale m / 127.  Means of at most 2^-100 are
    held as zeros; the scale of a page with an infinite or NaN key is NaN.  Other
    entries keep what they hold.  ``total``: the number of new tokens, where the caller
    knows it (cu's last entry, which lies on the device; without it the launch looks at
    every place of the table)."""
    if total is not None:
        T = operator.index(total)
    else:
        T = lens.shape[0] if isinstance(lens, torch.Tensor) and lens.dim() else -1
        if cu is not None:
            T = _ANY_TOKENS
    if _current_device() == pages.device.index:
        status = (_host or _native()).index(pages._t, index._t, table, lens, cu, T, _raw_stream(pages.device.index))
        if status is not None:
            return C.check(status)
    at = index._at(pages)
    a = _address(pages, table, lens, cu, T)
    C.check(_call(C.load_library().srw_kv_index, pages.device, _KV.pack(*a), _INDEX.pack(*at)))
    _written(*index._t)


def kv_select(q, pages: KvPages, index: KvIndex, table, lens, cu=None, *, n: int, first: int = 1, last: int = 1):
    """The pages that each new token attends to, for each key head: ``keep`` [T, heads,
    n] int32, places in the sequence's row of ``table``, ascending, -1 behind the last.
    ``q`` [T, n_heads, head_dim] as in :func:`paged_attention`.  A token at position i
    sees the pages of positions up to i; of more than ``n`` it keeps the ``first`` and
    the ``last`` ones (its own among these) and, of the others, those with the largest
    scores, equal ones from the front.  A page's score is the product of its mean key
    and the sum of the queries of the heads that read the key head, both in 8 bits: a
    whole number times the page's scale.  Pages whose index is NaN come first."""
    if _current_device() == pages.device.index:
        got = (_host or _native()).select(pages._t, index._t, q, table, lens, cu, n, first, last,
                                          _raw_stream(pages.device.index))
        if got is not None:
            return got
    for name, x in (("n", n), ("first", first), ("last", last)):
        if not hasattr(x, "__index__"):
            raise TypeError(f"{name} is a whole number; got {x!r}")
    if not (first >= 0 and last >= 1 and first + last <= n <= 0x7fffffff):
        raise ValueError("first is not negative, last at least 1, and n holds both")
    T = q.shape[0] if isinstance(q, torch.Tensor) and q.dim() else -1
    kv = _address(pages, table, lens, cu, T)
    q, *qs = _rows("q", q, pages, T, (BF16,), 4)
    if q.shape[1] < 1 or q.shape[1] % pages.heads:
        raise ValueError(f"{q.shape[1]} query heads are no multiple of the pages' {pages.heads}")
    at = index._at(pages)
    keep = torch.empty((T, pages.heads, n), dtype=I32, device=pages.device)
    s = _SELECT.pack(*kv, *at, q.data_ptr(), keep.data_ptr(), *qs, q.shape[1], n, first, last)
    C.check(_call(C.load_library().srw_kv_select, pages.device, s))
    return keep


def paged_attention(q, pages: KvPages, table, lens, cu=None, *, max_new: int = 0, scale=None, window: int = 0,
                    sinks: int = 0, keep=None, out=None):
    """Attention of the new tokens ``q`` [T, n_heads, head_dim] (bfloat16, any
    token and head strides; n_heads a multiple of the pages' heads) over their
    sequences' pages, which must hold the new tokens already: a token at
    position i sees the positions j <= i, with ``window`` > 0 those with j > i
    - window or j < ``sinks``.  ``scale`` multiplies the scores (default 1 /
    sqrt(head_dim)).  ``max_new``: the most new tokens of one sequence, where
    the caller knows it.  With ``keep`` [T, heads, n] int32 (:func:`kv_select`, or
    any ascending places in the sequence's row of ``table``) a token sees, of these
    positions, those of the kept pages alone; it goes without a window.  Returns
    ``out`` [T, n_heads, head_dim] bfloat16; a token that sees nothing gets zeros.

    Sums and statistics are float32.  The softmax weights enter the second
    product as one bfloat16 in calls of many rows, as two (16 bits) in calls of
    few.  Which kernel and how many splits a call gets goes by ``max_new``, its
    rows, heads and the table's width: a sequence's outputs are the same bit for
    bit in calls that agree in these, and within these roundings in any."""
    scale = pages.head_dim ** -0.5 if scale is None else float(scale)
    if out is None and _current_device() == pages.device.index:
        stream = _raw_stream(pages.device.index)
        if keep is None:
            got = (_host or _native()).attention(pages._t, q, table, lens, cu, max_new, scale, window, sinks, stream)
        elif type(window) is int is type(sinks) and window == sinks == 0 and max_new >= 0:
            got = (_host or _native()).attention_kept(pages._t, q, table, lens, cu, scale, keep, stream)
        else:
            got = None
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
    if keep is not None:
        if window:
            raise ValueError("kept pages go without a window")
        if not isinstance(keep, torch.Tensor) or keep.dim() != 3 or keep.shape[2] < 1:
            raise ValueError(f"keep must be [{T}, {pages.heads}, n]")
        kept = _tensor("keep", keep, dev, I32, (T, pages.heads, keep.shape[2])), keep.shape[2]
    given = out is not None
    if given:
        _tensor("out", out, dev, BF16, (T, Hq, pages.head_dim))
        _no_grad("out", out)
    else:
        out = torch.empty((T, Hq, pages.head_dim), dtype=BF16, device=dev)
    a = _ATTENTION.pack(*kv, q.data_ptr(), out.data_ptr(), *qs, Hq, max_new, window, sinks, scale)
    lib = C.load_library()
    if keep is None:
        attend, size = (lib.srw_attention, a), (lib.srw_attention_workspace_size, a)
    else:
        attend, size = (lib.srw_attention_kept, a, *kept), (lib.srw_attention_kept_workspace_size, a, kept[1])
    status = _call(attend[0], dev, *attend[1:], None, 0)
    if status == C.SRW_EWORKSPACE:  # splits to join, nothing launched yet
        need = ctypes.c_size_t(0)
        C.check(size[0](*size[1:], ctypes.byref(need)))
        ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
        status = _call(attend[0], dev, *attend[1:], ws.data_ptr(), need.value)
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
    the pages that no later token sees.

    ``fork(seq)`` opens a sequence that holds what ``seq`` does, on the same
    pages: a page that several sequences hold is copied (:func:`kv_copy`) when
    ``extend`` makes room in it for one of them.  ``compact()`` moves the held
    pages to the lowest ids, ``resize(n_pages)`` changes how many there are.

    ``indexed``: with an index of the pages (``index(i)``, layer i's
    :class:`KvIndex`), which copies take along."""

    def __init__(self, n_layers: int, n_pages: int, n_heads: int, head_dim: int, *, page_size: int = 64, dtype=BF16,
                 device="cuda:0", indexed: bool = False):
        dev = torch.device(device)
        if dtype not in _KINDS:
            raise TypeError(f"pages hold bfloat16, int8 or float8_e4m3fn; got {dtype}")
        if head_dim not in (64, 128) or page_size not in (16, 32, 64, 128, 256):
            raise ValueError("head_dim is 64 or 128 and page_size 16, 32, 64, 128 or 256")
        if min(n_layers, n_pages, n_heads) < 1:
            raise ValueError("n_layers, n_pages and n_heads are at least 1")
        if dev.type == "cuda" and dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.page_size, self.n_pages, self.device, self.dtype, self.indexed = page_size, n_pages, dev, dtype, bool(indexed)
        self._shape = (n_layers, n_heads, head_dim)
        self._hold(self._new(n_pages))
        self._free = list(range(n_pages - 1, -1, -1))
        self._pages, self._lens, self._next = {}, {}, 0
        self._more = {}   # pages that several sequences hold: how many beside the first

    def _new(self, n_pages):
        """Tensors of n_pages pages: k, v, then scales and the index's codes and scales
        where there are any."""
        L, H, d = self._shape
        P, dev = self.page_size, self.device
        t = [torch.empty(L, n_pages, H, *s, dtype=self.dtype, device=dev) for s in ((P, d), (d, P))]
        t += [torch.empty(L, n_pages, H, P, device=dev) for _ in range(2)] if self.dtype != BF16 else [None, None]
        if self.indexed:
            return t + [torch.zeros(L, n_pages, H, d, dtype=torch.int8, device=dev), torch.zeros(L, n_pages, H, device=dev)]
        return t + [None, None]

    def _hold(self, t):
        self.k, self.v, self.k_scale, self.v_scale, self._codes, self._code_scale = t

    def _tensors(self):
        return [t for t in (self.k, self.v, self.k_scale, self.v_scale, self._codes, self._code_scale) if t is not None]

    def layer(self, i: int) -> KvPages:
        if self.dtype == BF16:
            return KvPages(self.k[i], self.v[i])
        return KvPages(self.k[i], self.v[i], self.k_scale[i], self.v_scale[i])

    def index(self, i: int) -> KvIndex:
        if not self.indexed:
            raise ValueError("this cache has no index (indexed=True)")
        return KvIndex(self._codes[i], self._code_scale[i])

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
        (which waits for it).  A partly filled page that other sequences hold too is
        copied for the sequence first, on the current stream.  Raises MemoryError where
        the free pages do not do; whatever it raises, nothing has changed."""
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
        # pages that get new tokens beside what other sequences read there
        more, split = dict(self._more), []
        for s, n in zip(seqs, counts):
            at, used = divmod(self._lens[s], self.page_size)
            if n and used and self._pages[s][at] in more:
                split.append((s, at))
                self._drop(self._pages[s][at], more)
        wanted = sum(need.values()) + len(split)
        if wanted > len(self._free):
            raise MemoryError(f"{wanted} pages are needed, {len(self._free)} are free")
        if split:
            old = [self._pages[s][at] for s, at in split]
            new = self._free[:-len(split) - 1:-1]
            kv_copy(self._tensors(), old, new)
            del self._free[-len(split):]
            for (s, at), page in zip(split, new):
                self._pages[s][at] = page
            was, self._more = self._more, more
        for s, n in zip(seqs, counts):
            self._pages[s].extend(self._free.pop() for _ in range(need[s]))
            self._lens[s] += n
        try:
            return self._call_of(seqs, counts)
        except BaseException:
            self._take_back(seqs, counts)
            if split:
                for (s, at), page in zip(split, old):
                    self._pages[s][at] = page
                self._free.extend(reversed(new))
                self._more = was
            raise

    @staticmethod
    def _drop(page, more):
        """One sequence less holds a page of several."""
        if more[page] == 1:
            del more[page]
        else:
            more[page] -= 1

    def _give_back(self, page):
        if page in self._more:
            self._drop(page, self._more)
        else:
            self._free.append(page)

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
        their number (of those that other sequences hold too, this one's hold)."""
        if window < 1 or sinks < 0:
            raise ValueError("evict needs a window, and sinks are not negative")
        P, pages, n = self.page_size, self._pages[seq], 0
        for i in range(-(-sinks // P), len(pages)):
            if (i + 1) * P > self._lens[seq] - window + 1:
                break
            if pages[i] >= 0:
                self._give_back(pages[i])
                pages[i] = -1
                n += 1
        return n

    def free(self, seq: int) -> None:
        for p in reversed(self._pages.pop(seq)):
            if p >= 0:
                self._give_back(p)
        del self._lens[seq]

    def fork(self, seq: int) -> int:
        """A sequence that holds what seq does; no page is copied yet."""
        pages, n = list(self._pages[seq]), self._lens[seq]
        new, self._next = self._next, self._next + 1
        self._pages[new], self._lens[new] = pages, n
        for p in pages:
            if p >= 0:
                self._more[p] = self._more.get(p, 0) + 1
        return new

    def _renamed(self, names):
        """The bookkeeping with pages under other ids."""
        for pages in self._pages.values():
            pages[:] = [names.get(p, p) for p in pages]
        self._more = {names.get(p, p): n for p, n in self._more.items()}

    def _held(self):
        return sorted({p for pages in self._pages.values() for p in pages if p >= 0})

    def compact(self) -> int:
        """Move the held pages to the ids 0, 1, ..., as few as that takes; returns their
        number.  A table that extend gave before names pages of then."""
        held = self._held()
        n = len(held)
        src = [p for p in held if p >= n]
        dst = sorted(set(range(n)).difference(held))
        kv_copy(self._tensors(), src, dst)
        self._renamed(dict(zip(src, dst)))
        self._free = list(range(self.n_pages - 1, n - 1, -1))
        return len(src)

    def resize(self, n_pages: int) -> None:
        """Tensors of n_pages pages in place of the present ones; held pages are copied
        to the lowest ids.  Raises MemoryError where they are more; whatever it raises,
        nothing has changed.  ``layer(i)`` and ``index(i)`` of before are of the old
        tensors."""
        n_pages, held = operator.index(n_pages), self._held()
        if n_pages < 1:
            raise ValueError("n_pages is at least 1")
        if len(held) > n_pages:
            raise MemoryError(f"{len(held)} pages are held")
        new, old = self._new(n_pages), self._tensors()
        kv_copy(old, held, range(len(held)), to=[t for t in new if t is not None])
        for t in old:
            if t.is_cuda:  # (allocated on another stream, maybe: not given out again before the copy has read it)
                t.record_stream(torch.cuda.current_stream(t.device))
        self._hold(new)
        self._renamed({p: i for i, p in enumerate(held)})
        self.n_pages = n_pages
        self._free = list(range(n_pages - 1, len(held) - 1, -1))
