"""The training step with 8-bit activation checkpoints, captured and replayed, against the same steps launched one by one: the seven buffers
that all blocks share, the codes and the restored tensors are the step's own at every replay."""
import numpy as np
import pytest
import torch

from conftest import pkg

pytestmark = pytest.mark.gpu
NC = 24


def _trained(name, dtype, use_graph, batches):
    xo, models, losses = pkg("keras_extensions.extended_optimizers"), pkg("models"), pkg("losses")
    m = models.get_model(name, (None, None, 3), NC, losses.ModelLambdaLossType.SEGMENTATION_CATEGORICAL_CROSS_ENTROPY, dtype=dtype, activation_checkpoints="8bit").model
    m.graph.store.init_values(5)
    m.compile(optimizer=xo.Adam(lr=1e-3))
    m.seed = 9
    m.use_hip_graph = use_graph
    seen, grads = [], []
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for x in batches:
            seen.append(m.train_on_batch(x)[0])
            grads.append(m.graph.store.grad.clone())
            m.test_on_batch(x)      # a pass that answers goes through the same buffers
    torch.cuda.synchronize()
    assert bool(m._graphs) == use_graph
    return m, seen, grads


@pytest.mark.parametrize("name,dtype", [("segnet", "f32"), ("unet", "bf16")])
def test_replayed_steps_equal_the_steps_launched_one_by_one(name, dtype):
    rng = np.random.RandomState(4)
    n, h, w = 2, 32, 48
    batches = [[rng.standard_normal((n, h, w, 3)).astype(np.float32), rng.randint(0, NC, (n, h, w)).astype(np.int32), np.ones((n, h, w), np.float32),
                np.zeros((n, 1), np.int32)] for _ in range(6)]
    a, la, ga = _trained(name, dtype, True, batches)
    b, lb, gb = _trained(name, dtype, False, batches)
    assert la == lb and all(np.isfinite(la)) and len(set(la)) == len(la)
    for k, (x, y) in enumerate(zip(ga, gb)):
        assert torch.equal(x, y) and bool(x.any()), k
    assert torch.equal(a.graph.store.theta, b.graph.store.theta)
