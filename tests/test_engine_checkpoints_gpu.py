"""U-Net / SegNet with 8-bit activation checkpoints (get_model(..., activation_checkpoints="8bit")).

The forward pass is the plain graph's bit for bit.  The backward pass is the plain graph's on restored tensors: a plain graph whose
stored convolution outputs are replaced, between its forward and its backward pass, by restore(store(.)) and by the block outputs
formed from them has to give the same gradients bit for bit, and the plain graph's kernels are held to the oracle elsewhere."""
import numpy as np
import pytest
import torch

from conftest import pkg

pytestmark = pytest.mark.gpu
DEV = "cuda"
NC = 24


def _pair(name, dtype, hw, n):
    models, losses = pkg("models"), pkg("losses")
    t = losses.ModelLambdaLossType.CLASSIFICATION_CATEGORICAL_CROSS_ENTROPY if "encoder-only" in name else losses.ModelLambdaLossType.SEGMENTATION_CATEGORICAL_CROSS_ENTROPY
    shape = hw + (3,) if "encoder-only" in name else (None, None, 3)
    out = []
    for ck in (None, "8bit"):
        m = models.get_model(name, shape, NC, t, dtype=dtype, activation_checkpoints=ck).model
        m.graph.store.init_values(5)
        out.append(m)
    return out


def _units(g):
    return [u for b in g.blocks for u in getattr(b, "units", [])]


@pytest.mark.parametrize("name,dtype,n,h,w,dropout", [("unet", "f32", 2, 32, 48, True), ("unet", "bf16", 1, 48, 32, True), ("segnet", "f32", 1, 32, 32, False),
                                                      ("segnet", "bf16", 2, 64, 32, True), ("segnet-encoder-only", "f32", 2, 32, 32, True)])
def test_gradients_are_the_plain_graphs_on_restored_tensors(name, dtype, n, h, w, dropout):
    cp = pkg("layers.checkpoints")
    plain, kept = (m.graph for m in _pair(name, dtype, (h, w), n))
    g = torch.Generator().manual_seed(3)
    images = torch.randn(n, h, w, 3, generator=g).to(DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    outs = []
    with torch.cuda.stream(s):
        plain.overlap_weight_gradients = False
        for gr in (plain, kept):
            gr.plan(n, h, w)
            for k, v in gr.drop_views.items():
                if dropout:
                    v.copy_((torch.rand(v.shape, generator=torch.Generator().manual_seed(len(k))) > 0.2).float() / 0.8)
                else:
                    v.fill_(1.0)
            gr.store.grad.fill_(7.0)
            outs.append(gr.forward(images, training=True).clone())
        assert torch.equal(outs[0], outs[1])
        us, ks = _units(plain), _units(kept)
        assert len(us) == len(ks) and all(k.codes.shape == (u.npix, u.cout) for u, k in zip(us, ks))
        for b in plain.blocks:
            for u in getattr(b, "units", []):
                y, out = cp.store_8bit(u.y).restore_bn_act(u.bn.mean, u.bn.invstd, u.bn.gamma, u.bn.beta, activation="leaky" if u.act == 2 else "none", alpha=0.1,
                                                           drop=u.drop_mask if dropout else None)
                u.y.copy_(y)
                if u is not b.units[-1]:      # a run's last output is kept as it is
                    u.out.copy_(out)
        dl = torch.randn(plain.dlogits.shape, generator=g).to(DEV).to(plain.dlogits.dtype)
        for gr in (plain, kept):
            gr.backward(dl)
        torch.cuda.synchronize()
    for k in plain.store.gviews:
        a, b = plain.store.gviews[k], kept.store.gviews[k]
        assert torch.equal(a, b), (k, float((a - b).abs().max()))
        assert bool(torch.isfinite(a).all())


def _held(graph):
    """Bytes of the tensors that the convolution blocks hold, shared ones once."""
    seen = {}
    for u in _units(graph):
        for k in ("y", "out", "dy", "dx", "codes", "scales", "restored_out"):
            t = getattr(u, k, None)
            if t is not None:
                seen[t.untyped_storage().data_ptr()] = t.untyped_storage().nbytes()
    return sum(seen.values())


def test_memory_and_inference():
    """What the blocks hold shrinks.  U-Net at full resolution, values per pixel (a level below counts a quarter per channel, twice the
    channels: half): plain, four convolution blocks of 64: y, out, dy 12 * 64, input gradients 64 + 192 + 64 = 1088 at two bytes; with
    checkpoints 4 * 66 bytes of codes, two kept outputs and one 192-wide input gradient at two bytes and the seven shared buffers of 64
    once: (2 * 64 + 192 + 7 * 64) * 2 + 264 = 1800 bytes of 2176 at this level, and 904 of 2176 / 2 at every level below, which pays no
    shared buffers: under 0.8 of the whole."""
    n, h, w = 2, 128, 128
    images = torch.randn(n, h, w, 3, generator=torch.Generator().manual_seed(1)).to(DEV)
    preds, sizes = [], []
    for ck in (None, "8bit"):
        m = pkg("models").get_model("unet", (None, None, 3), NC, dtype="bf16", activation_checkpoints=ck).model
        m.graph.store.init_values(2)
        preds.append(m.graph.forward(images, training=False).clone())
        sizes.append(_held(m.graph))
    assert torch.equal(*preds)
    assert sizes[1] < 0.8 * sizes[0], sizes


def test_training_steps_replay():
    """A captured step runs on: the first loss is the plain model's, replays equal the eager step's gradients."""
    xo = pkg("keras_extensions.extended_optimizers")
    rng = np.random.RandomState(4)
    n, h, w = 2, 32, 32
    x = [rng.standard_normal((n, h, w, 3)).astype(np.float32), rng.randint(0, NC, (n, h, w)).astype(np.int32), np.ones((n, h, w), np.float32), np.zeros((n, 1), np.int32)]
    first = []
    for m in _pair("segnet", "f32", (h, w), n):
        m.compile(optimizer=xo.Adam(lr=1e-4))
        m.seed = 9
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            losses = [m.train_on_batch(x)[0] for _ in range(4)]
        torch.cuda.synchronize()
        assert all(np.isfinite(v) for v in losses)
        first.append(losses[0])
    assert first[0] == first[1]


def test_other_models_refuse():
    models = pkg("models")
    with pytest.raises(ValueError, match="U-Net and SegNet"):
        models.get_model("enet-naive-upsampling", (None, None, 3), NC, activation_checkpoints="8bit")
    with pytest.raises(ValueError, match="expected None or"):
        models.get_model("unet", (None, None, 3), NC, activation_checkpoints="4bit")
