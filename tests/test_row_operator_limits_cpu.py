"""Limits of the row operators that keep every address in reach, checked without a GPU: by what is refused and by the workspaces asked for."""
import ctypes as C
import importlib

import pytest
import torch
from torch.autograd import forward_ad

_lib = importlib.import_module("semantic-segmentation_amd._lib")
P = 0x1000      # a pointer that no refused call follows


def desc(**kw):
    v = dict(rows=1000, x_ld=kw["c"], y_ld=kw["f"], act=0, dtype=0, param_dtype=0)
    v.update(kw)
    return _lib.GatedDesc(*(v[n] for n, _ in _lib.GatedDesc._fields_))


@pytest.mark.parametrize("dtype", [0, 1])
def test_kernels_leave_room_for_the_steps_past_their_end(dtype):
    """The tile loop's last requests lie up to 128 rows behind the kernel; their offsets have to stay in 31 bits."""
    L = _lib.lib()
    f = 65528
    last = (2 ** 31 - 1) // (4 * f) - 128
    assert L.gated_ff_workspace_bytes(C.byref(desc(c=last, f=f, dtype=dtype)), 1) > 0
    for c in (last + 1, 8192):
        d = desc(c=c, f=f, dtype=dtype)
        assert c * f * 4 < 2 ** 31 and L.gated_ff_workspace_bytes(C.byref(d), 1) == 0
        with pytest.raises(_lib.SsmiError, match="2 GiB"):
            L.gated_ff_fwd(C.byref(d), P, P, P, None, None, P, P, 1 << 50, None)


@pytest.mark.parametrize("dtype,es", [(0, 4), (1, 2)])
def test_strips_of_the_weight_gradient_leave_room_for_the_steps_past_their_end(dtype, es):
    """Rows 2^20 values apart: a strip and 128 rows more stay in 31 bits.  The number of strips shows in the workspace, 4 * c * 2 fp bytes each."""
    L = _lib.lib()
    rows, c, f = 1000000, 16, 16
    wide, dense = (L.gated_ff_workspace_bytes(C.byref(desc(rows=rows, x_ld=ld, c=c, f=f, dtype=dtype)), 1) for ld in (1 << 20, c))
    usual = -(-rows // 1984)      # 512 strips of whole 64 rows
    strips = usual + (wide - dense) // (4 * c * 2 * f)
    longest = (2 ** 31 - 1) // (es << 20) - 128
    assert strips * longest >= rows, (strips, longest)


def test_tangents_are_found_on_any_device():
    rows = importlib.import_module("semantic-segmentation_amd.layers._rows")
    x = torch.ones(3)
    rows.refuse_tangents("call", x, None)
    with forward_ad.dual_level():
        rows.refuse_tangents("call", x, None, 1.0)
        with pytest.raises(ValueError, match="call: an input carries a tangent"):
            rows.refuse_tangents("call", None, forward_ad.make_dual(x, x))
    rows.refuse_tangents("call", x)


def test_rows_far_apart_are_copied_where_the_products_cannot_reach_them():
    rows = importlib.import_module("semantic-segmentation_amd.layers._rows")
    far = torch.empty(1).expand(1).as_strided((3, 8), (0, 0))      # only shapes and strides count
    near, over = (torch.empty(2 * s + 8, dtype=torch.uint8).as_strided((3, 8), (s, 1)) for s in (1 << 20, (1 << 20) + 1))
    t, n, ld = rows.rows_of(near, rows.FAR)
    assert t is near and (n, ld) == (3, 1 << 20)
    t, n, ld = rows.rows_of(over, rows.FAR)
    assert t is not over and (n, ld) == (3, 8) and torch.equal(t, over)
    t, n, ld = rows.rows_of(over)      # the checkpoints reach every row
    assert t is over and ld == (1 << 20) + 1
    assert rows.rows_of(far)[2] == 8


def test_checkpoints_made_by_hand_have_to_fit_together():
    """What restore() reads goes by the shape: codes and scales that are shorter would be read past their ends."""
    cp = importlib.import_module("semantic-segmentation_amd.layers.checkpoints")
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)      # noqa: E731
    kept = cp.Checkpoint8(u8(40, 6).t(), u8(6, 2), (2, 3, 40), torch.bfloat16)
    assert kept.codes.is_contiguous() and kept.shape == (2, 3, 40)
    for codes, scales, shape, dtype in ((u8(5, 40), u8(6, 2), (2, 3, 40), torch.float32), (u8(6, 40), u8(6, 1), (2, 3, 40), torch.float32),
                                        (u8(6, 40), u8(6, 2), (3, 3, 40), torch.float32), (u8(6, 40), u8(6, 2), (6, 41), torch.float32),
                                        (u8(6, 40), u8(6, 2), (6, 40), torch.float16), (u8(6, 40).float(), u8(6, 2), (6, 40), torch.float32),
                                        (u8(6, 40), u8(6, 2), (), torch.float32), (u8(240), u8(6, 2), (6, 40), torch.float32),
                                        (u8(6, 40), u8(6, 2).to("meta"), (6, 40), torch.float32)):
        with pytest.raises(ValueError, match="Checkpoint8"):
            cp.Checkpoint8(codes, scales, shape, dtype)
    v = torch.ones(40)
    for call in (kept.restore, lambda: kept.restore_bn_act(v, v, v, v)):
        with pytest.raises(NotImplementedError):
            call()
    with pytest.raises(ValueError, match="drop must be"):      # a table of the other order has as many values
        kept.restore_bn_act(v, v, v, v, drop=torch.ones(40, 2))


def test_weights_made_under_inference_mode_can_learn():
    ff = importlib.import_module("semantic-segmentation_amd.layers.feed_forward")
    made, given = ff.GatedFeedForward2D(4, seed=2), ff.GatedFeedForward2D(4)
    with torch.inference_mode():
        made.build((2, 3, 8), device="cpu")
        given.set_weights([torch.ones(8, 4), torch.ones(8, 4), torch.ones(4), torch.ones(4)], device="cpu")
    again = ff.GatedFeedForward2D(4, seed=2)
    again.build((2, 3, 8), device="cpu")
    for layer in (made, given):
        assert all(w.requires_grad and w.is_leaf and not w.is_inference() for w in layer.weights)
        (layer.weights[0] * layer.weights[1]).sum().backward()
    assert all(torch.equal(a, b) for a, b in zip(made.weights, again.weights))


def test_launches_that_are_too_large_are_refused_in_front_of_the_first():
    L = _lib.lib()
    rows = (1 << 30) + 64
    d = desc(rows=rows, c=8, f=8, dtype=1, param_dtype=1)
    assert L.gated_ff_workspace_bytes(C.byref(d), 1) > 0
    with pytest.raises(_lib.SsmiError, match="too many for one launch"):
        L.gated_ff_bwd(C.byref(d), P, P, P, None, None, P, P, P, P, None, None, P, 1 << 50, None)
    d = desc(rows=(1 << 31) - 1, c=8, f=8)
    with pytest.raises(_lib.SsmiError, match="too many for one launch"):
        L.gated_ff_fwd(C.byref(d), P, P, P, None, None, P, P, 1 << 50, None)
    with pytest.raises(_lib.SsmiError, match="too many for one launch"):
        L.mx4_dense(P, 64, (1 << 31) - 1, 64, 8, 0, P, P, None, P, 8, P, 1 << 50, None)
