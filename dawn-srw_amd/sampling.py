"""Choosing tokens from logits: HIP kernels (csrc/srw_sample.hip; one for short rows
and top-k, two where the sum of a long row is needed), torch tensors in and out.
:func:`sample` takes its random numbers from the caller, so a program
that keeps them can repeat a run; it waits for nothing and can be captured in a
graph."""

from __future__ import annotations

import ctypes
import math
import struct

import torch

from . import _capi as C
from . import kv
from .kv import _call, _current_device, _no_grad, _raw_stream, _tensor

__all__ = ["sample"]

F32, I32, I64 = torch.float32, torch.int32, torch.int64
_DTYPES = {torch.float32: C.SRW_F32, torch.bfloat16: C.SRW_BF16}
_MOST = torch.finfo(F32).max
_SAMPLE = struct.Struct("@P3q7P3f3i")


def _parameter(name, x, dev, dtype, B):
    """(address, 0) of a tensor [B], (None, number) of a number."""
    if isinstance(x, torch.Tensor):
        _no_grad(name, x)
        return _tensor(name, x, dev, dtype, (B,)), 0
    if dtype is I32:
        if not hasattr(x, "__index__"):
            raise TypeError(f"{name} is a whole number or a tensor; got {x!r}")
        if not 0 <= x <= 0x7fffffff:
            raise ValueError(f"{name} is not negative; got {x!r}")
        return 0, x
    x = float(x)
    if not (x >= 0 and (name == "temperature" or x <= 1)):
        raise ValueError(f"{name} is not negative{'' if name == 'temperature' else ' and at most 1'}; got {x!r}")
    return 0, x if x <= _MOST else math.inf  # (a temperature that float32 does not hold)


def _parameters(dev, B, temperature, top_k, top_p, min_p):
    return [_parameter(n, x, dev, t, B) for n, x, t in (("temperature", temperature, F32), ("top_p", top_p, F32),
                                                       ("min_p", min_p, F32), ("top_k", top_k, I32))]


def check_parameters(B, dev, temperature, top_k, top_p, min_p):
    """Raises what :func:`sample` would of its parameters for B rows on dev (tensors of any
    stride)."""
    _parameters(dev, B, *(x.contiguous() if isinstance(x, torch.Tensor) else x for x in (temperature, top_k, top_p, min_p)))


def sample(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(tokens [B] int64, logprobs [B] float32): one token of every row of ``logits``
    [B, vocab] (float32 or bfloat16, any row stride) from the random numbers ``u`` [B]
    float32 in [0, 1).

    A logit l of a row with largest M weighs exp((l - M) / temperature).  In the order
    of the logits, the largest first, equal ones by index, ``top_k`` (0: off) keeps the
    first k, ``top_p`` (1: off) of these the shortest run whose weights reach p times
    their sum, ``min_p`` (0: off) what weighs min_p or more.  The token is the first, by
    index, at which the kept weights' running sum passes u times their sum; its logprob
    is the logarithm of its share.  Temperature 0 takes the first in the order, with
    logprob 0.  NaN counts as -infinity, several infinite logits weigh the same; a row
    of -infinity gives token -1 and logprob -infinity.

    Each parameter is a number or a tensor [B] of the logits' device (float32; ``top_k``
    int32), whose entries are read on the device: there a temperature that is not above
    0 counts as 0, a top_k below 1, a top_p that is not below 1 and a min_p that is not
    above 0 as off, a min_p above 1 as 1.  u outside of [0, 1) counts as the nearest
    number inside (NaN as 0).

    Weights are summed as whole numbers, in units of 2^-51 to 2^-50 of the largest (of
    more than 2048 logits so that the sum stays below 2^62); of more than 8192, where the
    sum of all is needed, by runs of 8192 in units of each run's largest, rounded down to
    the row's.  What weighs nothing in these is not drawn.  A row's token goes by its own
    numbers alone, not by the batch or by where the row lies."""
    if not isinstance(logits, torch.Tensor) or logits.dim() != 2:
        raise ValueError("logits must be a tensor [B, vocab]")
    if logits.is_cuda:
        at = _current_device()
        got = (kv._host or kv._native()).sample(logits, u, temperature, top_k, top_p, min_p, at, _raw_stream(at))
        if got is not None:
            return got
    dev = logits.device
    if dev.type != "cuda":
        raise ValueError(f"logits live on a HIP device; got {dev}")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits has dtype {logits.dtype}, expected float32 or bfloat16")
    B, V = logits.shape
    if V < 1:
        raise ValueError("logits has no vocabulary")
    _no_grad("logits", logits)
    if isinstance(u, torch.Tensor):
        _no_grad("u", u)
    u = _tensor("u", u, dev, F32, (B,))
    given = _parameters(dev, B, temperature, top_k, top_p, min_p)
    if V > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    token = torch.empty(B, dtype=I64, device=dev)
    logprob = torch.empty(B, dtype=F32, device=dev)
    d = _SAMPLE.pack(logits.data_ptr(), logits.stride(0), B, V, u, *(a for a, _ in given), token.data_ptr(),
                     logprob.data_ptr(), *(x for _, x in given), _DTYPES[logits.dtype], 0)
    lib = C.load_library()
    status = _call(lib.srw_sample, dev, d, None, 0)
    if status == C.SRW_EWORKSPACE:  # sums of the rows' parts, nothing launched yet
        need = ctypes.c_size_t(0)
        C.check(lib.srw_sample_workspace_size(d, ctypes.byref(need)))
        ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
        status = _call(lib.srw_sample, dev, d, ws.data_ptr(), need.value)
    C.check(status)
    return token, logprob
