"""4-bit microscaled products for answering (OCP MXFP4: e2m1 values, one power of two per 32 reduction elements; `ssmi_mx4_*` in
include/ssmi.h states the format).  Weights are quantised once, inputs inside the call:

    w4 = quantize_mx4_weights(w)                 # Keras kernel [k, n], float32 or bfloat16, on the GPU
    y = mx4_dense(x, w4, bias)                   # q(x) w4 + bias, x [..., k]
    y = gated_feed_forward(x, g4, u4)            # layers.feed_forward, both projections on 4-bit weights

These calls have no backward pass."""
from __future__ import annotations

import functools

import torch

from .._lib import lib
from ._rows import FAR, dtype_code, on, refuse_tangents, require_gpu, rows_of, stream_of, vector

BLOCK = 32
_GATES = {"swish": 0, "gelu": 1, "relu": 2, "sigmoid": 3}


class MX4Weights(object):
    """A quantised kernel [k, n]: `codes` uint8 [n, 16 ceil(k / 32)], `scales` uint8 [n, ceil(k / 32)]."""

    __slots__ = ("codes", "scales", "k", "n")

    def __init__(self, codes, scales, k):
        who = "MX4Weights"
        require_gpu(codes, who)
        nb = (int(k) + BLOCK - 1) // BLOCK
        if k < 1 or codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.dim() != 2 or scales.shape != (codes.shape[0], nb) or \
                codes.shape[1] != 16 * nb or codes.shape[0] < 1 or scales.device != codes.device:
            raise ValueError("{}: codes uint8 [n, {}] and scales uint8 [n, {}] expected for k = {}, got {} {} and {} {}".format(
                who, 16 * nb, nb, k, codes.dtype, tuple(codes.shape), scales.dtype, tuple(scales.shape)))
        codes = codes.contiguous()
        self.codes = codes.clone() if codes.data_ptr() % 16 else codes
        scales = scales.contiguous()
        self.scales = scales.clone() if scales.data_ptr() % 16 else scales
        self.k, self.n = int(k), codes.shape[0]

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def dequantize(self) -> torch.Tensor:
        """The kernel that the codes stand for, float32 [k, n]."""
        w = torch.empty(self.k, self.n, dtype=torch.float32, device=self.codes.device)
        with on(w):
            lib().mx4_dequantize_kernel(self.codes.data_ptr(), self.scales.data_ptr(), self.k, self.n, w.data_ptr(), stream_of(w))
        return w


def quantize_mx4_weights(w: torch.Tensor) -> MX4Weights:
    who = "quantize_mx4_weights"
    require_gpu(w, who)
    refuse_tangents(who, w)
    code = dtype_code(w, who)
    if w.dim() != 2 or 0 in w.shape:
        raise ValueError("{}: a kernel [k, n] expected, got shape {}".format(who, tuple(w.shape)))
    k, n = w.shape
    w = w.detach().contiguous()
    nb = (k + BLOCK - 1) // BLOCK
    codes = torch.empty(n, 16 * nb, dtype=torch.uint8, device=w.device)
    scales = torch.empty(n, nb, dtype=torch.uint8, device=w.device)
    with on(w):
        lib().mx4_quantize_kernel(w.data_ptr(), k, n, code, codes.data_ptr(), scales.data_ptr(), stream_of(w))
    return MX4Weights(codes, scales, k)


def _operand(x, w: MX4Weights, who, *biases):
    require_gpu(x, who)
    refuse_tangents(who, x, *biases)
    if not isinstance(w, MX4Weights):
        raise TypeError("{}: MX4Weights expected, got {}".format(who, type(w).__name__))
    if x.dim() < 1 or x.shape[-1] != w.k or w.codes.device != x.device:
        raise ValueError("{}: x [..., {}] on {} expected, got {} on {}".format(who, w.k, w.codes.device, tuple(x.shape), x.device))
    if torch.is_grad_enabled() and (x.requires_grad or any(isinstance(b, torch.Tensor) and b.requires_grad for b in biases)):
        raise ValueError("{}: 4-bit products have no backward pass; call them under torch.no_grad() or on detached tensors".format(who))
    t, rows, ld = rows_of(x, FAR)
    return t, rows, ld, torch.empty(x.shape[:-1] + (w.n,), dtype=x.dtype, device=x.device)


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(rows, k):
    return int(lib().mx4_workspace_bytes(rows, k))


def _workspace(rows, k, like):
    n = _workspace_bytes(rows, k)
    return (torch.empty(n, dtype=torch.uint8, device=like.device), n) if n else (None, 0)


def mx4_dense(x: torch.Tensor, w: MX4Weights, bias=None) -> torch.Tensor:
    """q(x) w + bias: x [..., k] float32 or bfloat16, the result in x's type; bias float32 [n] or None."""
    who = "mx4_dense"
    t, rows, ld, y = _operand(x, w, who, bias)
    code = dtype_code(x, who)
    bias = vector(bias, w.n, x, who, "bias", optional=True)
    if rows:
        with on(x):
            ws, size = _workspace(rows, w.k, x)
            lib().mx4_dense(t.data_ptr(), ld, rows, w.k, w.n, code, w.codes.data_ptr(), w.scales.data_ptr(), None if bias is None else bias.data_ptr(),
                            y.data_ptr(), w.n, None if ws is None else ws.data_ptr(), size, stream_of(x))
    return y


def mx4_gated(x, w_gate, w_up, b_gate, b_up, activation):
    """layers.feed_forward.gated_feed_forward on 4-bit weights."""
    who = "gated_feed_forward"
    t, rows, ld, y = _operand(x, w_gate, who, b_gate, b_up)
    if not isinstance(w_up, MX4Weights) or (w_up.k, w_up.n) != (w_gate.k, w_gate.n) or w_up.codes.device != x.device:
        raise ValueError("{}: two MX4Weights of one shape on {} expected".format(who, x.device))
    code = dtype_code(x, who)
    b_gate, b_up = (vector(b, w_gate.n, x, who, "a bias", optional=True) for b in (b_gate, b_up))
    if rows:
        with on(x):
            ws, size = _workspace(rows, w_gate.k, x)
            lib().mx4_gated(t.data_ptr(), ld, rows, w_gate.k, w_gate.n, code, _GATES[activation], w_gate.codes.data_ptr(), w_gate.scales.data_ptr(),
                            w_up.codes.data_ptr(), w_up.scales.data_ptr(), None if b_gate is None else b_gate.data_ptr(),
                            None if b_up is None else b_up.data_ptr(), y.data_ptr(), w_gate.n, None if ws is None else ws.data_ptr(), size, stream_of(x))
    return y
