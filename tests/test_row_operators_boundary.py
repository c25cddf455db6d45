"""Refusals of s2_group_norm, s2_linear and s2_grouped_linear and of their
bindings, all before a device is touched."""
import ctypes

import pytest

from seedvr2_ncnn_amd import capi

F32, BF16, F16 = capi.DTYPE_F32, capi.DTYPE_BF16, capi.DTYPE_F16
P = 0x10000   # stands for a device address; none of these calls gets to use it

NORM = dict(x=P, x_dtype=F32, x_frame=163840, x_pixel=64, frames=2, pixels=2560, channels=64, groups=8,
            gamma=P, beta=P, epsilon=1e-6, activation=capi.ACT_NONE, y=2 * P, y_dtype=F32,
            y_frame=163840, y_pixel=64, workspace=P, workspace_bytes=1 << 20, stream=None)
LINEAR = dict(x=P, x_dtype=BF16, x_stride=64, m=4, weight=P, w_dtype=BF16, bias=P, n=32, k=64,
              activation=capi.ACT_NONE, residual=P, residual_stride=32, y=2 * P, y_dtype=F32,
              y_stride=32, workspace=None, workspace_bytes=0, stream=None)
GROUPED = dict(x=P, x_dtype=BF16, x_stride=64, m=4, offsets=P, groups=2, weight=P, w_dtype=BF16,
               bias=P, n=32, k=64, activation=capi.ACT_NONE, residual=P, residual_stride=32, y=2 * P,
               y_dtype=F32, y_stride=32, workspace=None, workspace_bytes=0, stream=None)


def _call(name, base, **changes):
    assert set(changes) <= set(base)
    return getattr(capi.lib(), name)(*dict(base, **changes).values())


@pytest.mark.parametrize("changes", [
    dict(frames=-1), dict(frames=65536), dict(pixels=-1), dict(groups=0), dict(groups=-8),
    dict(groups=7), dict(channels=0), dict(channels=4104, groups=8), dict(x_dtype=3), dict(y_dtype=-1),
    dict(activation=capi.ACT_SWIGLU), dict(activation=5), dict(epsilon=-1e-6),
    dict(epsilon=float("nan")), dict(x=None), dict(y=None), dict(x_frame=-1), dict(x_pixel=-64),
    dict(y_pixel=63), dict(y_frame=63), dict(y_frame=163839), dict(x=P + 2), dict(y=P + 2),
    dict(gamma=P + 2), dict(beta=P + 1), dict(workspace=None), dict(workspace_bytes=8),
    dict(workspace=P + 4), dict(y=P, y_dtype=BF16), dict(y=P, y_frame=327680)], ids=str)
def test_group_norm_refuses(changes):
    assert _call("s2_group_norm", NORM, **changes) == capi.S2_ERR_INVALID
    assert capi.last_error()


def test_group_norm_takes_interleaved_frames_as_far_as_the_device():
    """Frames interleaved by pixel pass the checks of the strides."""
    if capi.device_count():
        pytest.skip("the call would run")
    assert _call("s2_group_norm", NORM, y_frame=64, y_pixel=128) == capi.S2_ERR_DEVICE


def test_group_norm_of_nothing():
    assert _call("s2_group_norm", NORM, frames=0, x=None, y=None) == capi.S2_OK
    assert _call("s2_group_norm", NORM, pixels=0, workspace=None) == capi.S2_OK
    assert capi.group_norm_workspace(0, 5, 8, 2) == capi.group_norm_workspace(3, 20, 8, 2) == 0
    assert capi.group_norm_workspace(3, 50000, 8, 2) > 0
    for bad in ((1, 1, 9, 2), (1, 1, 8192, 2), (-1, 1, 8, 2), (1, -1, 8, 2)):
        with pytest.raises(capi.S2Error):
            capi.group_norm_workspace(*bad)


MATMUL = [
    dict(m=-1), dict(n=0), dict(k=0), dict(n=-4), dict(x_dtype=3), dict(y_dtype=7),
    dict(w_dtype=F32), dict(w_dtype=F16), dict(x_dtype=F16), dict(x_dtype=F32, w_dtype=F16),
    dict(activation=capi.ACT_SWIGLU), dict(activation=-1), dict(x=None), dict(weight=None),
    dict(y=None), dict(x_stride=63), dict(y_stride=31), dict(residual_stride=31), dict(x=P + 1),
    dict(weight=P + 1), dict(y=P + 2), dict(residual=P + 2), dict(bias=P + 2),
    dict(residual=2 * P, residual_stride=40), dict(y=P), dict(x=3 * P, y=P)]


@pytest.mark.parametrize("changes", MATMUL + [dict(workspace=P + 8, workspace_bytes=64)], ids=str)
def test_linear_refuses(changes):
    assert _call("s2_linear", LINEAR, **changes) == capi.S2_ERR_INVALID
    assert capi.last_error()


@pytest.mark.parametrize("changes", MATMUL + [dict(groups=-1), dict(offsets=None), dict(offsets=P + 2),
                                              dict(workspace=P + 8, workspace_bytes=64)],
                         ids=str)
def test_grouped_linear_refuses(changes):
    assert _call("s2_grouped_linear", GROUPED, **changes) == capi.S2_ERR_INVALID
    assert capi.last_error()


@pytest.mark.parametrize("size", ["m", "n", "k"])
def test_sizes_past_the_kernels_indexes_are_refused(size):
    """2^30 at most: steps past the last k or tile stay in 32 bits."""
    changes = {"m": 1, "x_stride": 1 << 31, "y_stride": 1 << 31, "residual_stride": 1 << 31,
               size: (1 << 30) + 1}
    assert _call("s2_linear", LINEAR, **changes) == capi.S2_ERR_INVALID
    assert _call("s2_grouped_linear", GROUPED, **changes) == capi.S2_ERR_INVALID
    sizes = {"m": 8, "n": 8, "k": 8, size: (1 << 30) + 1}
    with pytest.raises(capi.S2Error):
        capi.linear_workspace(**sizes)
    with pytest.raises(capi.S2Error):
        capi.grouped_linear_workspace(groups=2, **sizes)


def test_groups_past_the_kernels_indexes_are_refused():
    assert _call("s2_grouped_linear", GROUPED, groups=(1 << 30) + 1) == capi.S2_ERR_INVALID
    with pytest.raises(capi.S2Error):
        capi.grouped_linear_workspace(8, (1 << 30) + 1, 8, 8)
    assert _call("s2_grouped_linear", GROUPED, m=(1 << 28) + 1) == capi.S2_ERR_INVALID
    with pytest.raises(capi.S2Error):
        capi.grouped_linear_workspace((1 << 28) + 1, 2, 8, 8)


def test_linear_of_nothing():
    assert _call("s2_linear", LINEAR, m=0, x=None, y=None) == capi.S2_OK
    assert _call("s2_grouped_linear", GROUPED, m=0) == capi.S2_OK
    assert _call("s2_grouped_linear", GROUPED, groups=0, offsets=None) == capi.S2_OK
    assert capi.linear_workspace(0, 8, 8) == 0
    for bad in ((-1, 8, 8), (1, 0, 8), (1, 8, 0)):
        with pytest.raises(capi.S2Error):
            capi.linear_workspace(*bad)
    assert capi.grouped_linear_workspace(0, 2, 8, 8) == capi.grouped_linear_workspace(9, 0, 8, 8) == 0
    assert capi.grouped_linear_workspace(900, 2, 8, 8, F32) > 0   # fp32 rows are repacked
    for bad in ((-1, 1, 8, 8), (1, -1, 8, 8), (1, 1, 0, 8), (1, 1, 8, 0), (1, 1, 8, 8, 3), (1, 1, 8, 8, 0, 3)):
        with pytest.raises(capi.S2Error):
            capi.grouped_linear_workspace(*bad)
    assert capi.lib().s2_linear_workspace_bytes(1, 1, 1, 0, 0, None) == capi.S2_ERR_INVALID
    assert capi.lib().s2_grouped_linear_workspace_bytes(1, 1, 1, 1, 0, 0, None) == capi.S2_ERR_INVALID
    assert capi.lib().s2_group_norm_workspace_bytes(1, 1, 1, 1, None) == capi.S2_ERR_INVALID


def test_other_entry_points_do_not_take_the_new_activations():
    n = ctypes.c_void_p(P)
    for act in (capi.ACT_SILU, capi.ACT_GELU_TANH):
        assert capi.lib().s2_shared_linear_forward(n, 8, None, 0, BF16, n, None, 64, 64, act, n, None,
                                                   BF16, None) == capi.S2_ERR_INVALID


def test_bindings_check_shapes_and_types():
    import torch
    x, w = torch.zeros(4, 64), torch.zeros(32, 64, dtype=torch.bfloat16)
    offs = torch.zeros(3, dtype=torch.int32)
    wg = torch.zeros(2, 32, 64, dtype=torch.bfloat16)
    frames = torch.zeros(2, 8, 64)
    for call in (lambda: capi.linear(x[:, :32], w), lambda: capi.linear(x.t().contiguous().t(), w),
                 lambda: capi.linear(x, w.t().contiguous().t()),
                 lambda: capi.linear(x, w, torch.zeros(31)),
                 lambda: capi.linear(x, w, torch.zeros(32, dtype=torch.float64)),
                 lambda: capi.linear(x, w, residual=torch.zeros(4, 31)),
                 lambda: capi.linear(x, w, residual=torch.zeros(4, 32).half()),
                 lambda: capi.linear(x, w, out=torch.zeros(5, 32)),
                 lambda: capi.grouped_linear(x, offs.long(), wg),
                 lambda: capi.grouped_linear(x, offs[:2], wg),
                 lambda: capi.grouped_linear(x, offs, wg, torch.zeros(32)),
                 lambda: capi.group_norm(frames[0], 8), lambda: capi.group_norm(frames.transpose(1, 2), 8),
                 lambda: capi.group_norm(frames, 8, torch.zeros(8)),
                 lambda: capi.group_norm(frames, 8, out=torch.zeros(2, 8, 65)),
                 # host memory
                 lambda: capi.group_norm(frames, 8), lambda: capi.linear(x, w),
                 lambda: capi.grouped_linear(x, offs, wg)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        capi.linear(x.double(), w)
    with pytest.raises(TypeError):
        capi.group_norm(frames.double(), 8)


def test_workspaces_of_strided_and_unaligned_operands():
    """Room to repack 16-bit rows that are apart by no multiple of eight elements or start
    at no 16-byte boundary, and weights that do; the strides of a single row say nothing."""
    for dtype in (BF16, F16):
        base = capi.linear_workspace(8000, 2001, 2560, dtype, dtype)
        assert capi.linear_workspace(8000, 2001, 2560, dtype, dtype, x_stride=2560) == base
        assert capi.linear_workspace(8000, 2001, 2560, dtype, dtype, x_stride=2568, x_start=32) == base
        rows = 8000 * 2560 * 2
        for change in (dict(x_stride=2564), dict(x_start=8), dict(x_stride=2561, x_start=2)):
            assert capi.linear_workspace(8000, 2001, 2560, dtype, dtype, **change) >= base + rows
            assert capi.grouped_linear_workspace(8000, 2, 2001, 2560, dtype, dtype, **change) >= rows
        assert capi.linear_workspace(8000, 2001, 2560, dtype, dtype, weight_start=2) >= rows + 2001 * 2560 * 2
        assert capi.grouped_linear_workspace(8000, 3, 2001, 2560, dtype, dtype,
                                             weight_start=6) >= rows + 3 * 2001 * 2560 * 2
        one = capi.linear_workspace(1, 2001, 2560, dtype, dtype)
        assert capi.linear_workspace(1, 2001, 2560, dtype, dtype, x_stride=3) == one
    for bad in (dict(x_stride=63), dict(x_start=1), dict(weight_start=3)):
        with pytest.raises(capi.S2Error):
            capi.linear_workspace(9, 32, 64, BF16, BF16, **bad)
        with pytest.raises(capi.S2Error):
            capi.grouped_linear_workspace(9, 2, 32, 64, BF16, BF16, **bad)
    assert capi.lib().s2_linear_view_workspace_bytes(None, BF16, 64, 9, None, 32, 64, BF16,
                                                     None) == capi.S2_ERR_INVALID
    assert capi.lib().s2_grouped_linear_view_workspace_bytes(None, BF16, 64, 9, 2, None, 32, 64, BF16,
                                                             None) == capi.S2_ERR_INVALID


@pytest.mark.parametrize("wrap", [1 << 31, (1 << 32) + 3, -(1 << 32) + 3], ids=str)
def test_sizes_that_32_bits_would_wrap_are_refused(wrap):
    """A C int would take 2^32 + 3 for 3."""
    for at in range(4):
        sizes = [2, 8, 8, 2]
        sizes[at] = wrap
        with pytest.raises(capi.S2Error):
            capi.group_norm_workspace(*sizes)
        with pytest.raises(capi.S2Error):
            capi.grouped_linear_workspace(*sizes)
    for at in range(3):
        sizes = [8, 8, 8]
        sizes[at] = wrap
        with pytest.raises(capi.S2Error):
            capi.linear_workspace(*sizes)
    with pytest.raises(capi.S2Error):
        capi.linear_workspace(8, 8, 8, wrap, BF16)
    with pytest.raises(capi.S2Error):
        capi.grouped_linear_workspace(8, 2, 8, 8, BF16, wrap)


def test_bindings_refuse_sizes_that_32_bits_would_wrap():
    """Before anything of that size is made."""
    import torch
    many = (1 << 32) + 3
    w, wide = torch.zeros(1, 1, dtype=torch.bfloat16), torch.zeros(1, 1, dtype=torch.bfloat16).expand(many, 1)
    offs = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: capi.linear(wide, w), lambda: capi.linear(w, wide),
                 lambda: capi.grouped_linear(wide, offs, w[None]),
                 lambda: capi.group_norm(wide[None], 1), lambda: capi.group_norm(wide[:, None], 1),
                 lambda: capi.group_norm(wide.t()[None], 1),
                 lambda: capi.group_norm(w[None], many),
                 lambda: capi.linear(w, w, activation=many), lambda: capi.group_norm(w[None], 1, activation=many),
                 lambda: capi.grouped_linear(w, offs, w[None], activation=1 << 32)):
        with pytest.raises(capi.S2Error):
            call()


def test_streams_of_another_device_are_refused(monkeypatch):
    import torch

    class On:
        def __init__(self, index):
            self.device_index, self.cuda_stream = index, 64 + index

        def get_device(self):
            return self.device_index

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    assert capi._raw_stream(On(0), On(0), On(0), None) == 64
    for stream, tensors in ((On(1), [On(0)]), (On(1), [On(1)]), (On(0), [On(0), On(1)])):
        with pytest.raises(ValueError):
            capi._raw_stream(tensors[0], stream, *tensors[1:])


@pytest.mark.parametrize("types", [(F32, BF16), (F32, F32), (BF16, BF16), (F16, F32)], ids=str)
@pytest.mark.parametrize("mnk", [(1, 640, 2560), (77, 2560, 5120), (300, 257, 133), (21600, 2560, 132)], ids=str)
def test_workspaces_of_contiguous_operands(mnk, types):
    """The queries without a view are those of contiguous, aligned operands."""
    m, n, k = mnk
    size = ctypes.c_size_t()
    assert capi.lib().s2_linear_workspace_bytes(m, n, k, *types, ctypes.byref(size)) == capi.S2_OK
    assert size.value == capi.linear_workspace(m, n, k, *types, x_stride=k)
    assert capi.lib().s2_grouped_linear_workspace_bytes(m, 2, n, k, *types, ctypes.byref(size)) == capi.S2_OK
    assert size.value == capi.grouped_linear_workspace(m, 2, n, k, *types, x_stride=k)
