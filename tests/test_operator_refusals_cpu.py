"""What the row operators refuse, checked without a GPU: argument errors raise before anything is launched."""
import ctypes as C
import importlib

import pytest
import torch

_lib = importlib.import_module("semantic-segmentation_amd._lib")
cp = importlib.import_module("semantic-segmentation_amd.layers.checkpoints")

P = 0x1000      # a pointer that no refused call follows


def test_checkpoints_want_gpu_tensors_of_the_two_types():
    with pytest.raises(NotImplementedError):
        cp.store_8bit(torch.zeros(2, 4))
    with pytest.raises(TypeError):
        cp.store_8bit([1.0])


def test_checkpoint_arguments():
    kept = cp.Checkpoint8(torch.zeros(6, 4, dtype=torch.uint8), torch.zeros(6, 1, dtype=torch.uint8), (2, 3, 4), torch.float32)
    v = torch.ones(4)
    with pytest.raises(ValueError, match="activation"):
        kept.restore_bn_act(v, v, v, v, activation="swish")
    with pytest.raises(ValueError, match="gamma"):
        kept.restore_bn_act(v, v, torch.ones(5), v)
    with pytest.raises(ValueError, match="alpha"):
        kept.restore_bn_act(v, v, v, v, activation="prelu", alpha=0.1)
    with pytest.raises(ValueError, match="drop"):
        kept.restore_bn_act(v, v, v, v, drop=torch.ones(3, 4))
    with pytest.raises(ValueError, match="out must be"):
        kept.restore(out=torch.zeros(2, 3, 5))


@pytest.mark.parametrize("args,text", [
    ((None, 8, 4, 8, 0, P, P, None), "null pointer"),
    ((P, 7, 4, 8, 0, P, P, None), "pixel stride"),
    ((P, 8, 0, 8, 0, P, P, None), "pixels"),
    ((P, 8, 4, 0, 0, P, P, None), "pixels"),
    ((P, 8, 4, 8, 3, P, P, None), "dtype"),
    ((P, 1024, 1 << 40, 1024, 0, P, P, None), "too many"),
])
def test_act8_store_refuses(args, text):
    with pytest.raises(_lib.SsmiError, match=text):
        _lib.lib().act8_store(*args)


def test_act8_restore_refuses():
    L = _lib.lib()
    bn = _lib.BnParams(P, P, P, P)
    with pytest.raises(_lib.SsmiError, match="null pointer"):
        L.act8_restore(P, P, 4, 8, 0, None, 8, None)
    with pytest.raises(_lib.SsmiError, match="pixel stride"):
        L.act8_restore(P, P, 4, 8, 0, P, 7, None)
    full = [P, P, 4, 8, 0, C.byref(bn), 0, None, 0.0, None, 1, P, 8, P, 8, None]
    for at, v, text in ((6, 3, "unknown activation"), (6, 1, "slopes"), (14, 7, "pixel stride"), (13, None, "null pointer"), (12, 3, "pixel stride")):
        a = list(full)
        a[at] = v
        with pytest.raises(_lib.SsmiError, match=text):
            L.act8_restore_bn_act(*a)
    a = list(full)
    a[9], a[10] = P, 3      # four pixels are no whole images of three
    with pytest.raises(_lib.SsmiError, match="whole images"):
        L.act8_restore_bn_act(*a)
