"""What the row operators (layers.checkpoints, layers.feed_forward, layers.microscaled) share: a tensor's trailing axis is its
channels, everything in front of it the rows (pixels), and a call runs on the current stream of the tensor's own device."""
from __future__ import annotations

import contextlib

import torch
from torch.autograd import forward_ad

from .._lib import BF16, F32

_CODES = {torch.float32: F32, torch.bfloat16: BF16}
_HERE = contextlib.nullcontext()


def dtype_code(t: torch.Tensor, who: str) -> int:
    try:
        return _CODES[t.dtype]
    except KeyError:
        raise ValueError("{}: float32 or bfloat16 expected, got {}".format(who, t.dtype)) from None


def require_gpu(t, who: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError("{}: a torch tensor expected, got {}".format(who, type(t).__name__))
    if not t.is_cuda:      # the error of the pooling layers
        raise NotImplementedError("{} works only on GPU".format(who))


def refuse_tangents(who: str, *tensors) -> None:
    """The kernels have no forward-mode derivative: a tensor with a tangent would lose it without a word."""
    if getattr(forward_ad, "_current_level", 0) < 0:      # outside every level no tensor has one
        return
    for t in tensors:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError("{}: an input carries a tangent, and there is no forward-mode derivative".format(who))


def on(t: torch.Tensor):
    """The device of `t` as the current one for the length of a call (a no-op where it is)."""
    return _HERE if t.get_device() == torch.cuda.current_device() else torch.cuda.device(t.device)


# the handle of a device's current stream without the Stream object around it (2 us of a 15 us call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_of(t: torch.Tensor) -> int:
    if _raw_stream is not None:
        return _raw_stream(t.get_device())
    return torch.cuda.current_stream(t.device).cuda_stream


FAR = 1 << 20      # the products address a tile's rows with 32-bit offsets: values from one row to the next


def rows_of(t: torch.Tensor, most: int = 1 << 62):
    """(tensor, rows, row stride): `t` itself where its leading axes step evenly, by at most `most` values, over rows of contiguous
    channels - a channel slice of a wider tensor, for instance -, a contiguous copy otherwise."""
    c = t.shape[-1]
    if t.is_contiguous():
        return t, t.numel() // c if c else 0, c
    if t.stride(-1) == 1 or c == 1:
        ld = None
        step = 1
        for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if size == 1:
                continue
            if ld is None:
                ld = stride
            if stride != ld * step:
                break
            step *= size
        else:
            if ld is not None and c <= ld <= most:
                return t, t.numel() // c, ld
    t = t.contiguous()
    return t, t.numel() // c if c else 0, c


def vector(t, n: int, like: torch.Tensor, who: str, what: str, optional: bool = False):
    """A float32 vector of n values beside `like`, dense."""
    if t is None and optional:
        return None
    if not isinstance(t, torch.Tensor) or t.device != like.device or t.dtype != torch.float32 or t.numel() != n:
        raise ValueError("{}: {} must be {} float32 values on {}".format(who, what, n, like.device))
    return t.contiguous()
