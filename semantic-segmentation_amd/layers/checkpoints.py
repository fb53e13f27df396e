"""8-bit activation checkpoints: an activation that waits for the backward pass in one byte per value (and one exponent byte per
pixel and 32 channels) instead of two or four.  `ssmi_act8_*` in include/ssmi.h states the format; a restored value is off by at
most half an e4m3 step, and a group of 32 channels that holds an infinity or a NaN restores as NaN.

    kept = store_8bit(y)                       # float32 or bfloat16, channels last, on the GPU
    y8 = kept.restore()                        # the same shape and type
    y8, out = kept.restore_bn_act(mean, invstd, gamma, beta, activation="leaky", alpha=0.1, drop=table)

The gated feed-forward unit keeps its input so (`checkpoint="8bit"`), the U-Net / SegNet training graphs the raw convolution
outputs of their blocks (`get_model(..., activation_checkpoints="8bit")`)."""
from __future__ import annotations

import ctypes as C

import torch

from .._lib import BnParams, lib
from ._rows import dtype_code, on, refuse_tangents, require_gpu, rows_of, stream_of, vector

GROUP = 32
_ACTS = {"none": 0, "prelu": 1, "leaky": 2}


class Checkpoint8(object):
    """A stored tensor: `codes` uint8 [rows, channels], `scales` uint8 [rows, ceil(channels / 32)], and the shape and type that
    restore() gives back."""

    __slots__ = ("codes", "scales", "shape", "dtype")

    def __init__(self, codes, scales, shape, dtype):
        shape = torch.Size(shape)
        c = shape[-1] if len(shape) else 0
        rows = shape.numel() // c if c else 0
        want = (rows, c), (rows, (c + GROUP - 1) // GROUP)
        if c < 1 or dtype not in (torch.float32, torch.bfloat16) or any(t.dtype != torch.uint8 or tuple(t.shape) != s for t, s in zip((codes, scales), want)) or \
                codes.device != scales.device:
            raise ValueError("Checkpoint8: codes uint8 {} and scales uint8 {} on one device expected for a {} tensor of shape {}, got {} {} and {} {}".format(
                *want, dtype, tuple(shape), codes.dtype, tuple(codes.shape), scales.dtype, tuple(scales.shape)))
        self.codes, self.scales, self.shape, self.dtype = codes.contiguous(), scales.contiguous(), shape, dtype

    @classmethod
    def _made(cls, codes, scales, shape, dtype):
        """Of tensors that store_8bit made."""
        self = object.__new__(cls)
        self.codes, self.scales, self.shape, self.dtype = codes, scales, shape, dtype
        return self

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def _target(self, out, who):
        if out is None:
            return torch.empty(self.shape, dtype=self.dtype, device=self.codes.device)
        if out.shape != self.shape or out.dtype != self.dtype or out.device != self.codes.device or not out.is_contiguous():
            raise ValueError("{}: out must be a dense {} tensor of shape {} on {}".format(who, self.dtype, tuple(self.shape), self.codes.device))
        if out.requires_grad and torch.is_grad_enabled():
            raise ValueError("{}: out must not ask for gradients".format(who))
        if not out.is_inference():
            torch.autograd.graph.increment_version(out)      # what a graph saved of it is stale from here on
        return out

    def restore(self, out=None) -> torch.Tensor:
        """The tensor back, in `out` (dense, of its shape and type) where that is given."""
        y = self._target(out, "restore")
        require_gpu(y, "restore")
        if y.numel():
            rows, c = self.codes.shape
            with on(y):
                lib().act8_restore(self.codes.data_ptr(), self.scales.data_ptr(), rows, c, dtype_code(y, "restore"), y.data_ptr(), c, stream_of(y))
        return y

    def restore_bn_act(self, mean, invstd, gamma, beta, activation="none", alpha=0.1, drop=None):
        """(restored tensor, drop * act(gamma * (restored - mean) * invstd + beta)).  activation: "none", "leaky" (alpha a number) or
        "prelu" (alpha [channels]); drop: [images, channels], the images being the tensor's first axis."""
        who = "restore_bn_act"
        if activation not in _ACTS:
            raise ValueError("{}: activation must be one of {}, got {!r}".format(who, sorted(_ACTS), activation))
        c = self.shape[-1]
        mean, invstd, gamma, beta = (vector(t, c, self.codes, who, n) for t, n in
                                     ((mean, "mean"), (invstd, "invstd"), (gamma, "gamma"), (beta, "beta")))
        slopes = vector(alpha, c, self.codes, who, "alpha") if activation == "prelu" else None
        slope = float(alpha) if activation == "leaky" else 0.0
        hw = 1
        if drop is not None:
            if len(self.shape) < 2:
                raise ValueError("{}: a dropout table needs an axis of images".format(who))
            drop = vector(drop, self.shape[0] * c, self.codes, who, "drop")
            if tuple(drop.shape) != (self.shape[0], c):
                raise ValueError("{}: drop must be [{}, {}], got {}".format(who, self.shape[0], c, tuple(drop.shape)))
            for d in self.shape[1:-1]:
                hw *= d
        require_gpu(self.codes, who)
        y, out = self._target(None, who), self._target(None, who)
        if y.numel():
            rows = self.codes.shape[0]
            bn = BnParams(mean.data_ptr(), invstd.data_ptr(), gamma.data_ptr(), beta.data_ptr())
            with on(y):
                lib().act8_restore_bn_act(self.codes.data_ptr(), self.scales.data_ptr(), rows, c, dtype_code(y, who), C.byref(bn), _ACTS[activation],
                                          None if slopes is None else slopes.data_ptr(), slope, None if drop is None else drop.data_ptr(), hw,
                                          y.data_ptr(), c, out.data_ptr(), c, stream_of(y))
        return y, out


def store_8bit(x: torch.Tensor) -> Checkpoint8:
    """The tensor's checkpoint.  `x`: float32 or bfloat16 with the channels on its last axis, dense or a channel slice of a wider tensor.
    What is restored from it is detached: a checkpoint serves a backward pass and is no part of a graph."""
    require_gpu(x, "store_8bit")
    refuse_tangents("store_8bit", x)
    code = dtype_code(x, "store_8bit")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("store_8bit: a tensor with channels on its last axis expected, got shape {}".format(tuple(x.shape)))
    t, rows, ld = rows_of(x.detach())
    c = x.shape[-1]
    codes = torch.empty(rows, c, dtype=torch.uint8, device=x.device)
    scales = torch.empty(rows, (c + GROUP - 1) // GROUP, dtype=torch.uint8, device=x.device)
    if rows:
        with on(x):
            lib().act8_store(t.data_ptr(), ld, rows, c, code, codes.data_ptr(), scales.data_ptr(), stream_of(x))
    return Checkpoint8._made(codes, scales, x.shape, x.dtype)
