"""Gated feed-forward unit on the pixels of a channels-last tensor:

    y = act(x w_gate + b_gate) * (x w_up + b_up)

`gated_feed_forward` is the function (differentiable through torch.autograd, its backward pass is HIP kernels too), `GatedFeedForward2D`
the layer in the manner of the pooling layers.  Parameters are Keras kernels [channels, units] and vectors [units]; float32, or
bfloat16 under bfloat16 activations.  Nothing but the input waits for the backward pass - in 8 bits with checkpoint="8bit" (the
gradients are then those at the restored input, layers.checkpoints).  On two MX4Weights (layers.microscaled) the same call answers on
the 4-bit matrix instructions; that form has no backward pass."""
from __future__ import annotations

import ctypes as C
import functools

import torch

from .._lib import BF16, GatedDesc, lib
from ._rows import FAR, dtype_code, on, refuse_tangents, require_gpu, rows_of, stream_of
from .checkpoints import Checkpoint8, store_8bit
from .microscaled import MX4Weights, mx4_gated

ACTIVATIONS = {"swish": 0, "gelu": 1, "relu": 2, "sigmoid": 3}


def _ptr(t):
    return None if t is None else t.data_ptr()


def _aligned_rows(x):
    """rows_of with the 16-byte alignment that the products ask of their operands."""
    t, rows, ld = rows_of(x, FAR)
    if t.data_ptr() % 16:
        t = t.contiguous() if not t.is_contiguous() else t.clone()
        ld = t.shape[-1]
    return t, rows, ld


def _dense(w):
    if not w.is_contiguous():
        w = w.contiguous()
    return w.clone() if w.data_ptr() % 16 else w


@functools.lru_cache(maxsize=4096)
def _plan(rows, x_ld, y_ld, c, f, act, dtype, param_dtype, backward):
    """The descriptor of a call and its workspace size, by sizes and types alone."""
    d = GatedDesc(rows, x_ld, y_ld, c, f, act, dtype, param_dtype)
    ref = C.byref(d)
    return ref, int(lib().gated_ff_workspace_bytes(ref, backward)), d


def _forward(x, wg, wu, bg, bu, act):
    t, rows, ld = _aligned_rows(x)
    c, f = wg.shape
    y = torch.empty(x.shape[:-1] + (f,), dtype=x.dtype, device=x.device)
    if not rows:
        return y
    ref, n, _ = _plan(rows, ld, f, c, f, act, dtype_code(x, "gated_feed_forward"), dtype_code(wg, "gated_feed_forward"), 0)
    with on(x):
        ws = torch.empty(n, dtype=torch.uint8, device=x.device) if n else None
        lib().gated_ff_fwd(ref, t.data_ptr(), wg.data_ptr(), wu.data_ptr(), _ptr(bg), _ptr(bu), y.data_ptr(), _ptr(ws), n, stream_of(x))
    return y


class _GatedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, bg, bu, act, checkpoint):
        wg, wu = _dense(wg), _dense(wu)
        if bg is not None:
            bg, bu = bg.contiguous(), bu.contiguous()
        y = _forward(x, wg, wu, bg, bu, act)
        ctx.act = act
        # the checkpoint's tensors are saved as any others: gone behind the backward pass, seen by saved-tensor hooks
        kept = None if checkpoint is None else store_8bit(x)
        ctx.kept_as = None if kept is None else (kept.shape, kept.dtype)
        ctx.save_for_backward(wg, wu, bg, bu, *((x,) if kept is None else (kept.codes, kept.scales)))
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():      # create_graph=True: what follows is not recorded
            raise RuntimeError("gated_feed_forward has no second derivative")
        wg, wu, bg, bu, *kept = ctx.saved_tensors
        wg, wu = _dense(wg), _dense(wu)      # saved-tensor hooks may give them back in another layout
        if bg is not None:
            bg, bu = bg.contiguous(), bu.contiguous()
        x = kept[0] if ctx.kept_as is None else Checkpoint8(*kept, *ctx.kept_as).restore()
        nx, ng, nu, nbg, nbu = ctx.needs_input_grad[:5]
        c, f = wg.shape
        t, rows, ld = _aligned_rows(x)
        if not rows:
            return (torch.zeros_like(x) if nx else None, *(torch.zeros_like(p) if n else None for p, n in ((wg, ng), (wu, nu), (bg, nbg), (bu, nbu))), None, None)
        if dy.dtype != x.dtype:
            dy = dy.to(x.dtype)
        dt, _, dy_ld = rows_of(dy, FAR)
        if nx and ld != c:      # the row stride of dx is that of x
            t, ld = _dense(t), c
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if nx else None
        dwg = torch.empty_like(wg) if ng else None
        dwu = torch.empty_like(wu) if nu else None
        dbg = torch.empty_like(bg) if nbg else None
        dbu = torch.empty_like(bu) if nbu else None
        ref, n, _ = _plan(rows, ld, dy_ld, c, f, ctx.act, dtype_code(x, "gated_feed_forward"), dtype_code(wg, "gated_feed_forward"), 1)
        with on(x):
            ws = torch.empty(n, dtype=torch.uint8, device=x.device)
            lib().gated_ff_bwd(ref, t.data_ptr(), wg.data_ptr(), wu.data_ptr(), _ptr(bg), _ptr(bu), dt.data_ptr(), _ptr(dx), _ptr(dwg), _ptr(dwu),
                               _ptr(dbg), _ptr(dbu), ws.data_ptr(), n, stream_of(x))
        return dx, dwg, dwu, dbg, dbu, None, None


def gated_feed_forward(x, w_gate, w_up, b_gate=None, b_up=None, activation="swish", checkpoint=None):
    """x [..., channels] float32 or bfloat16 on the GPU; w_gate, w_up [channels, units]; b_gate, b_up [units] or both None.
    activation: "swish", "gelu" (exact), "relu" or "sigmoid".  checkpoint: None, or "8bit" to keep the input in 8 bits for the
    backward pass.  w_gate and w_up may be MX4Weights (biases then float32): answering on 4-bit products."""
    who = "gated_feed_forward"
    require_gpu(x, who)
    refuse_tangents(who, x, w_gate, w_up, b_gate, b_up)
    if activation not in ACTIVATIONS:
        raise ValueError("{}: activation must be one of {}, got {!r}".format(who, sorted(ACTIVATIONS), activation))
    if checkpoint not in (None, "8bit"):
        raise ValueError('{}: checkpoint must be None or "8bit", got {!r}'.format(who, checkpoint))
    if (b_gate is None) != (b_up is None):
        raise ValueError("{}: both biases or none".format(who))
    if isinstance(w_gate, MX4Weights) or isinstance(w_up, MX4Weights):
        if checkpoint is not None:
            raise ValueError("{}: 4-bit weights have no backward pass to keep a checkpoint for".format(who))
        return mx4_gated(x, w_gate, w_up, b_gate, b_up, activation)
    code = dtype_code(x, who)
    if x.dim() < 1 or w_gate.dim() != 2 or w_gate.shape != w_up.shape or w_gate.shape[0] != x.shape[-1] or 0 in w_gate.shape:
        raise ValueError("{}: kernels must both be [{}, units], got {} and {}".format(who, x.shape[-1] if x.dim() else "channels", tuple(w_gate.shape), tuple(w_up.shape)))
    f = w_gate.shape[1]
    params = (w_gate, w_up) if b_gate is None else (w_gate, w_up, b_gate, b_up)
    dev, pt = x.device, w_gate.dtype
    learns = x.requires_grad
    for p in params:
        if p.dtype != pt or p.device != dev or not (pt == torch.float32 or (pt == torch.bfloat16 and code == BF16)):
            raise ValueError("{}: parameters must be float32 (or all bfloat16 under a bfloat16 input) on {}".format(who, dev))
        learns = learns or p.requires_grad
    if b_gate is not None and (b_gate.shape != (f,) or b_up.shape != (f,)):
        raise ValueError("{}: biases must be [{}], got {} and {}".format(who, f, tuple(b_gate.shape), tuple(b_up.shape)))
    if learns and torch.is_grad_enabled():
        return _GatedFn.apply(x, w_gate, w_up, b_gate, b_up, ACTIVATIONS[activation], checkpoint)
    with torch.no_grad():
        if b_gate is not None:
            b_gate, b_up = b_gate.contiguous(), b_up.contiguous()
        return _forward(x, _dense(w_gate), _dense(w_up), b_gate, b_up, ACTIVATIONS[activation])


class GatedFeedForward2D(object):
    """The unit as a layer over NHWC tensors, in the manner of the pooling layers: parameters are made at the first call (he_normal
    kernels as the bottlenecks', zero biases) from `seed`, or given with set_weights.  `checkpoint="8bit"` keeps the input in 8 bits
    for the backward pass; `quantize()` returns the layer's answering form on 4-bit weights."""

    def __init__(self, units, activation="swish", use_bias=True, checkpoint=None, seed=0, name=None, **kwargs):
        if int(units) != units or units < 1:
            raise ValueError("units must be a positive whole number, got {!r}".format(units))
        if activation not in ACTIVATIONS:
            raise ValueError("activation must be one of {}, got {!r}".format(sorted(ACTIVATIONS), activation))
        if checkpoint not in (None, "8bit"):
            raise ValueError('checkpoint must be None or "8bit", got {!r}'.format(checkpoint))
        self.units, self.activation, self.use_bias, self.checkpoint, self.seed, self.name = int(units), activation, use_bias, checkpoint, seed, name
        self.weights = None      # [gate kernel, up kernel(, gate bias, up bias)], float32

    def build(self, input_shape, device="cuda"):
        c = input_shape[-1]
        g = torch.Generator().manual_seed(self.seed)
        with torch.inference_mode(False):      # weights made in a first call that only answers can learn later
            self.weights = [(torch.randn(c, self.units, generator=g) * (2.0 / c) ** 0.5).to(device).requires_grad_() for _ in range(2)]
            if self.use_bias:
                self.weights += [torch.zeros(self.units, device=device, requires_grad=True) for _ in range(2)]

    def set_weights(self, weights, device="cuda"):
        with torch.inference_mode(False):
            ws = [torch.as_tensor(w, dtype=torch.float32).detach().clone().to(device) for w in weights]
        if len(ws) != (4 if self.use_bias else 2) or any(w.dim() != 2 or w.shape != ws[0].shape or w.shape[1] != self.units for w in ws[:2]) or \
                any(b.shape != (self.units,) for b in ws[2:]):
            raise ValueError("expected {} with {} units, got shapes {}".format("two kernels and two biases" if self.use_bias else "two kernels", self.units,
                                                                               [tuple(w.shape) for w in ws]))
        self.weights = [w.requires_grad_() for w in ws]

    def get_weights(self):
        return [w.detach().cpu().numpy() for w in self.weights or []]

    def __call__(self, inputs, **kwargs):
        require_gpu(inputs, type(self).__name__)
        if self.weights is None:
            self.build(inputs.shape, inputs.device)
        return gated_feed_forward(inputs, *self.weights, activation=self.activation, checkpoint=self.checkpoint)

    def quantize(self):
        """A function of the input: the unit on 4-bit weights, made from the present ones."""
        from .microscaled import quantize_mx4_weights
        if self.weights is None:
            raise ValueError("the layer has no weights yet")
        kernels = [quantize_mx4_weights(w.detach()) for w in self.weights[:2]]
        biases = [b.detach().clone() for b in self.weights[2:]]
        return lambda x: gated_feed_forward(x, *kernels, *biases, activation=self.activation)

    def compute_output_shape(self, input_shape):
        return tuple(input_shape[:-1]) + (self.units,)
