"""The row operators (gated feed-forward unit, 8-bit checkpoints, 4-bit products) inside torch's differentiation: what they refuse, what they
keep and for how long."""
import importlib

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu

ff = importlib.import_module("semantic-segmentation_amd.layers.feed_forward")
cp = importlib.import_module("semantic-segmentation_amd.layers.checkpoints")
ms = importlib.import_module("semantic-segmentation_amd.layers.microscaled")
DEV = "cuda:0"


def tensors(rows=40, c=32, f=24, **kw):
    g = torch.Generator().manual_seed(3)
    return [torch.randn(s, generator=g).to(DEV).requires_grad_(kw.get("grad", False)) for s in ((rows, c), (c, f), (c, f), (f,), (f,))]


@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(grad):
    """A forward-mode derivative would come out as zero: every call that a tangent reaches raises, and the same calls in the level without one
    answer as they do outside."""
    x, wg, wu, bg, bu = tensors(grad=grad)
    q = [ms.quantize_mx4_weights(w) for w in (wg, wu)]
    free = [t.detach() for t in (x, wg, wu, bg, bu)]
    want = ff.gated_feed_forward(*free)
    with forward_ad.dual_level():
        for k in range(5):
            args = [x, wg, wu, bg, bu]
            args[k] = forward_ad.make_dual(args[k], torch.ones_like(args[k]))
            with pytest.raises(ValueError, match="tangent"):
                ff.gated_feed_forward(*args)
        dx, db = forward_ad.make_dual(free[0], torch.ones_like(x)), forward_ad.make_dual(free[3], torch.ones_like(bg))
        for call in (lambda: ms.mx4_dense(dx, q[0]), lambda: ms.mx4_dense(free[0], q[0], db), lambda: ff.gated_feed_forward(dx, *q),
                     lambda: ff.gated_feed_forward(free[0], *q, free[3], db), lambda: cp.store_8bit(dx), lambda: ms.quantize_mx4_weights(dx)):
            with pytest.raises(ValueError, match="tangent"):
                call()
        assert torch.equal(ff.gated_feed_forward(*free), want)
        ms.mx4_dense(free[0], q[0]), cp.store_8bit(free[0])
    assert torch.equal(ff.gated_feed_forward(*free), want)


def test_a_checkpoint_lives_as_long_as_the_backward_pass_needs_it():
    """Its tensors are saved tensors: hooks see them, they are gone behind a backward pass (while the output lives), and a second pass without
    retain_graph is refused as it is without a checkpoint."""
    rows, c = 4096, 512      # 2 MiB of codes, a block of its own
    g = torch.Generator().manual_seed(1)
    x = torch.randn(rows, c, generator=g).to(DEV).requires_grad_()
    w = [torch.randn(c, 8, generator=g).to(DEV).requires_grad_() for _ in range(2)]
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append((t.dtype, tuple(t.shape))) or t, lambda t: t):
        y = ff.gated_feed_forward(x, *w, checkpoint="8bit")
    assert (torch.uint8, (rows, c)) in seen and (torch.uint8, (rows, c // 32)) in seen and (torch.float32, (rows, c)) not in seen
    for checkpoint in (None, "8bit"):
        y = ff.gated_feed_forward(x, *w, checkpoint=checkpoint)
        first = torch.autograd.grad(y.sum(), [x, *w], retain_graph=True)
        before = torch.cuda.memory_allocated()
        second = torch.autograd.grad(y.sum(), [x, *w])
        assert all(torch.equal(a, b) for a, b in zip(first, second))
        del second
        freed = before - torch.cuda.memory_allocated()
        assert freed >= (rows * c if checkpoint else 0), freed
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(y.sum(), [x, *w])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_more_than_2_20_values_apart(dtype):
    """The first pixel of every image of a batch: rows a whole image apart.  Results are those of a dense copy."""
    x, wg, wu, bg, bu = (t.to(dtype) for t in tensors(rows=20, c=64))
    images = torch.zeros(20, 130 * 130, 64, dtype=dtype, device=DEV)
    images[:, 0] = x
    leaf = images.requires_grad_()
    view = leaf[:, 0]
    assert view.stride(0) > 1 << 20
    y, want = ff.gated_feed_forward(view, wg, wu, bg, bu), ff.gated_feed_forward(x, wg, wu, bg, bu)
    assert torch.equal(y, want)
    dy = torch.ones(20, 130 * 2000, 24, dtype=dtype, device=DEV)[:, 0]      # and a gradient with rows as far apart
    (d,) = torch.autograd.grad(y, leaf, dy)
    x.requires_grad_()
    (want,) = torch.autograd.grad(ff.gated_feed_forward(x, wg, wu, bg, bu), x, torch.ones_like(y))
    assert torch.equal(d[:, 0], want) and not bool(d[:, 1:].any())
    q = ms.quantize_mx4_weights(wg)
    assert torch.equal(ms.mx4_dense(view.detach(), q), ms.mx4_dense(x.detach(), q))
    assert torch.equal(cp.store_8bit(view).restore(), cp.store_8bit(x).restore())


def test_restore_into_a_tensor_counts_as_a_change_of_it():
    """A graph that saved the target must not go on with what it finds there, and a leaf that learns is no target."""
    x, w = torch.randn(6, 40, device=DEV), torch.randn(6, 40, device=DEV, requires_grad=True)
    kept, buf = cp.store_8bit(x), torch.zeros(6, 40, device=DEV)
    y = (buf * w).sum()
    assert kept.restore(out=buf) is buf and torch.equal(buf, kept.restore())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with pytest.raises(ValueError, match="gradients"):
        kept.restore(out=w)
    with torch.no_grad():
        assert torch.equal(kept.restore(out=w), buf)
    with torch.inference_mode():
        assert torch.equal(kept.restore(out=torch.zeros(6, 40, device=DEV)), buf)


@pytest.mark.parametrize("checkpoint", [None, "8bit"])
def test_saved_tensors_may_come_back_in_another_layout(checkpoint):
    """A hook gives back equal values; how they lie in memory is its own affair."""
    args = tensors(c=48, grad=True)
    want = torch.autograd.grad(ff.gated_feed_forward(*args, checkpoint=checkpoint).sum(), args)

    def other(t):
        return t.t().contiguous().t() if t.dim() == 2 else torch.stack([t, t], -1)[..., 0]
    with torch.autograd.graph.saved_tensors_hooks(other, lambda t: t):
        y = ff.gated_feed_forward(*args, checkpoint=checkpoint)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y.sum(), args), want))
    with torch.autograd.graph.save_on_cpu():
        y = ff.gated_feed_forward(*args, checkpoint=checkpoint)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y.sum(), args), want))
