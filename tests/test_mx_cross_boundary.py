"""Refusals of the MXFP4 entry points, of s2_cross_attention and of their bindings, all
before a device is touched."""
import ctypes

import pytest
import torch

from seedvr2_ncnn_amd import capi

F32, BF16, F16 = capi.DTYPE_F32, capi.DTYPE_BF16, capi.DTYPE_F16
P = 0x10000   # stands for a device address; none of these calls gets to use it

QUANTIZE = dict(x=P, x_dtype=BF16, x_stride=100, m=4, k=100, codes=2 * P, code_stride=64, scales=3 * P,
                scale_stride=16, stream=None)
DEQUANTIZE = dict(codes=2 * P, code_stride=64, scales=3 * P, scale_stride=16, m=4, k=100, y=P, y_dtype=BF16,
                  y_stride=100, stream=None)
LINEAR = dict(x_codes=P, x_code_stride=64, x_scales=2 * P, x_scale_stride=16, m=4, w_codes=3 * P,
              w_scales=4 * P, w_scale_stride=16, bias=P, n=32, k=100, activation=capi.ACT_NONE, residual=P,
              residual_stride=32, y=5 * P, y_dtype=F32, y_stride=32, workspace=None, workspace_bytes=0,
              stream=None)
WEIGHT = dict(x=P, x_dtype=BF16, x_stride=100, m=4, w_codes=3 * P, w_scales=4 * P, w_scale_stride=16, bias=P,
              n=32, k=100, activation=capi.ACT_NONE, residual=P, residual_stride=32, y=5 * P, y_dtype=F32,
              y_stride=32, workspace=None, workspace_bytes=0, stream=None)
SHAPE = dict(batch=2, lq=10, lk=20, heads=4, kv_heads=2, head_dim=64, dtype=BF16, out_dtype=BF16, scale=0.125)
CROSS = dict(q=P, k=2 * P, v=3 * P, out=4 * P,
             strides=(2560, 256, 64, 2560, 128, 64, 2560, 128, 64, 2560, 256, 64), q_offsets=None,
             k_offsets=None, key_lengths=None, key_mask=None, mask_stride=0, workspace=None,
             workspace_bytes=0, stream=None)


def _call(name, base, **changes):
    assert set(changes) <= set(base)
    return getattr(capi.lib(), name)(*dict(base, **changes).values())


def _cross(**changes):
    shape = capi.CrossAttentionShape(**{k: changes.pop(k, v) for k, v in SHAPE.items()})
    assert set(changes) <= set(CROSS)
    args = dict(CROSS, **changes)
    if args["strides"] is not None:
        args["strides"] = (ctypes.c_long * 12)(*args["strides"])
    return capi.lib().s2_cross_attention(ctypes.byref(shape), *args.values())


@pytest.mark.parametrize("changes", [
    dict(m=-1), dict(k=0), dict(k=-3), dict(k=(1 << 30) + 1), dict(m=(1 << 30) + 1), dict(x_dtype=3), dict(x=None),
    dict(x=P + 1), dict(x_stride=-1), dict(codes=None), dict(scales=None), dict(codes=2 * P + 8),
    dict(code_stride=72), dict(code_stride=48), dict(scale_stride=3), dict(codes=P), dict(scales=P),
    dict(scales=2 * P)], ids=str)
def test_quantize_refuses(changes):
    assert _call("s2_mx_quantize", QUANTIZE, **changes) == capi.S2_ERR_INVALID
    assert capi.last_error()


@pytest.mark.parametrize("changes", [
    dict(m=-1), dict(k=0), dict(y_dtype=-1), dict(y=None), dict(y=P + 1), dict(y_stride=99), dict(codes=None),
    dict(scales=None), dict(codes=2 * P + 4), dict(code_stride=40), dict(scale_stride=2), dict(y=2 * P),
    dict(y=3 * P)], ids=str)
def test_dequantize_refuses(changes):
    assert _call("s2_mx_dequantize", DEQUANTIZE, **changes) == capi.S2_ERR_INVALID
    assert capi.last_error()


PRODUCT = [
    dict(m=-1), dict(n=0), dict(k=0), dict(n=(1 << 30) + 1), dict(y_dtype=7), dict(activation=capi.ACT_SWIGLU),
    dict(activation=-1), dict(w_codes=None), dict(w_scales=None), dict(w_codes=3 * P + 8), dict(w_scale_stride=3),
    dict(y=None), dict(y=5 * P + 2), dict(y_stride=31), dict(residual_stride=31), dict(residual=P + 2),
    dict(bias=P + 2), dict(residual=5 * P, residual_stride=40), dict(y=3 * P), dict(y=4 * P), dict(y=P),
    dict(workspace=P + 8, workspace_bytes=64)]


@pytest.mark.parametrize("changes", PRODUCT + [
    dict(x_codes=None), dict(x_scales=None), dict(x_codes=P + 8), dict(x_code_stride=48), dict(x_code_stride=72),
    dict(x_scale_stride=3), dict(y=2 * P)], ids=str)
def test_linear_refuses(changes):
    assert _call("s2_mx_linear", LINEAR, **changes) == capi.S2_ERR_INVALID
    assert capi.last_error()


@pytest.mark.parametrize("changes", PRODUCT + [
    dict(x=None), dict(x=P + 1), dict(x_stride=99), dict(x_dtype=3)], ids=str)
def test_weight_linear_refuses(changes):
    assert _call("s2_mx_weight_linear", WEIGHT, **changes) == capi.S2_ERR_INVALID
    assert capi.last_error()


def test_products_of_nothing_and_workspaces():
    assert _call("s2_mx_quantize", QUANTIZE, m=0, x=None, codes=None) == capi.S2_OK
    assert _call("s2_mx_dequantize", DEQUANTIZE, m=0, y=None) == capi.S2_OK
    assert _call("s2_mx_linear", LINEAR, m=0, x_codes=None, y=None) == capi.S2_OK
    assert _call("s2_mx_weight_linear", WEIGHT, m=0, x=None, y=None) == capi.S2_OK
    assert capi.mx_linear_workspace(0, 8, 8) == capi.mx_linear_workspace(0, 8, 8, F32) == 0
    for bad in ((-1, 8, 8), (1, 0, 8), (1, 8, 0), (1, 8, 8, 3), (1, 8, 8, None, 3), (1 << 31, 8, 8),
                (1, (1 << 30) + 1, 8)):
        with pytest.raises(capi.S2Error):
            capi.mx_linear_workspace(*bad)
    assert capi.lib().s2_mx_linear_workspace_bytes(1, 1, 1, 0, None) == capi.S2_ERR_INVALID
    assert capi.lib().s2_mx_weight_linear_workspace_bytes(1, 1, 1, 0, 0, None) == capi.S2_ERR_INVALID


def _strides(**at):
    s = list(CROSS["strides"])
    for i, v in at.items():
        s[int(i[1:])] = v
    return dict(strides=tuple(s))


@pytest.mark.parametrize("changes", [
    dict(batch=-1), dict(lq=-1), dict(lk=-1), dict(lq=(1 << 30) + 1), dict(lq=1 << 30), dict(lk=(1 << 30) + 1),
    dict(heads=0), dict(kv_heads=0),
    dict(kv_heads=3), dict(heads=65536, kv_heads=1), dict(head_dim=0), dict(head_dim=60), dict(head_dim=264),
    dict(dtype=3), dict(out_dtype=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=None),
    dict(k=None), dict(v=None), dict(out=None), dict(strides=None), dict(q=P + 8), dict(k=2 * P + 2),
    dict(v=3 * P + 4), dict(out=4 * P + 1), _strides(s0=2564), _strides(s1=260), _strides(s2=68), _strides(s4=129),
    _strides(s7=-128), _strides(s3=-8), _strides(s10=255), _strides(s11=63), _strides(s9=2559), _strides(s11=0), _strides(s4=(1 << 23) + 8, s3=1 << 30), _strides(s7=1 << 24, s6=1 << 30),
    dict(q_offsets=P), dict(k_offsets=P), dict(q_offsets=P, k_offsets=P, key_lengths=P),
    dict(q_offsets=P + 2, k_offsets=P), dict(key_lengths=P + 1), dict(key_mask=P, mask_stride=-1), dict(key_mask=P, mask_stride=1 << 41),
    dict(out=P, out_dtype=F32), dict(out=P, **_strides(s10=512, s9=5120)), dict(out=2 * P), dict(out=3 * P),
    dict(workspace=P + 8, workspace_bytes=64)], ids=str)
def test_cross_attention_refuses(changes):
    assert _cross(**changes) == capi.S2_ERR_INVALID
    assert capi.last_error()


def test_cross_attention_of_nothing_and_workspaces():
    assert _cross(batch=0, q=None) == capi.S2_OK
    assert _cross(lq=0, q=None, out=None) == capi.S2_OK
    assert capi.cross_attention_workspace(0, 5, 5, 2, 1, 64) == 0
    for bad in ((-1, 5, 5, 2, 1, 64), (1, 5, 5, 3, 2, 64), (1, 5, 5, 2, 1, 65), (1, 5, 5, 2, 1, 64, 3),
                (1 << 31, 5, 5, 2, 1, 64)):
        with pytest.raises(capi.S2Error):
            capi.cross_attention_workspace(*bad)
    shape = capi.CrossAttentionShape(**SHAPE)
    assert capi.lib().s2_cross_attention_workspace_bytes(ctypes.byref(shape), 0, None) == capi.S2_ERR_INVALID
    assert capi.lib().s2_cross_attention_workspace_bytes(None, 0, ctypes.byref(ctypes.c_size_t())) == (
        capi.S2_ERR_INVALID)


def _rows(m, k, pad=0):
    b = (k + 31) // 32
    return capi.MxRows(torch.zeros(m, 16 * b, dtype=torch.uint8), torch.zeros(m, b + pad, dtype=torch.uint8)[:, :b], k)


def test_mx_bindings_check_shapes_and_types():
    x, w = torch.zeros(4, 64), _rows(32, 64)
    q = _rows(4, 64, 3)
    for call in (lambda: capi.mx_quantize(torch.zeros(4)), lambda: capi.mx_quantize(torch.zeros(4, 6).t()),
                 lambda: capi.mx_quantize(x, out=_rows(3, 64)), lambda: capi.mx_quantize(x, out=_rows(4, 65)),
                 lambda: capi.mx_quantize(x, out=q._replace(codes=q.codes.int())),
                 lambda: capi.mx_dequantize(q._replace(k=65)), lambda: capi.mx_dequantize(q, out=torch.zeros(4, 63)),
                 lambda: capi.mx_dequantize(q._replace(scales=q.scales[:3])),
                 lambda: capi.mx_dequantize(q._replace(scales=q.scales.int())),
                 lambda: capi.mx_linear(x[:, :32], w), lambda: capi.mx_linear(_rows(4, 32), w),
                 lambda: capi.mx_linear(x, w._replace(codes=torch.zeros(32, 64, dtype=torch.uint8)[:, :32])),
                 lambda: capi.mx_linear(x, w, torch.zeros(31)), lambda: capi.mx_linear(x, w, residual=torch.zeros(4, 31)),
                 lambda: capi.mx_linear(x, w, residual=torch.zeros(4, 32).half()),
                 lambda: capi.mx_linear(x, w, out=torch.zeros(4, 33)),
                 lambda: capi.mx_linear(q, w), lambda: capi.mx_quantize(x), lambda: capi.mx_linear(x, w)):
        with pytest.raises(ValueError):   # the last ones: no operand is on a device
            call()
    with pytest.raises(capi.S2Error):
        capi.mx_linear(x, w, activation=capi.ACT_SWIGLU)


def test_cross_attention_binding_checks_shapes_and_types():
    q, k = torch.zeros(2, 5, 4, 64), torch.zeros(2, 7, 2, 64)
    q3, k3 = torch.zeros(10, 4, 64), torch.zeros(14, 2, 64)
    o = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: capi.cross_attention(q3, k3, k3), lambda: capi.cross_attention(q, k, k[:, :6]),
                 lambda: capi.cross_attention(q, k.half(), k), lambda: capi.cross_attention(q, k[..., :32], k[..., :32]),
                 lambda: capi.cross_attention(q, k[:1], k[:1]), lambda: capi.cross_attention(q, k, k, k_offsets=o),
                 lambda: capi.cross_attention(q3, k3, k3, q_offsets=o),
                 lambda: capi.cross_attention(q3, k3, k3, q_offsets=o, k_offsets=o[:2]),
                 lambda: capi.cross_attention(q3, k3, k3, q_offsets=o.long(), k_offsets=o),
                 lambda: capi.cross_attention(q3, k3, k3, q_offsets=o, k_offsets=o, key_lengths=o[:2]),
                 lambda: capi.cross_attention(q, k, k, key_lengths=o), lambda: capi.cross_attention(q, k, k, key_lengths=o[:2].long()),
                 lambda: capi.cross_attention(q, k, k, key_mask=torch.zeros(2, 6, dtype=torch.bool)),
                 lambda: capi.cross_attention(q, k, k, key_mask=torch.zeros(2, 7)),
                 lambda: capi.cross_attention(q, k, k, out=torch.zeros(2, 5, 4, 32)),
                 lambda: capi.cross_attention(q.transpose(2, 3).contiguous().transpose(2, 3), k, k),
                 lambda: capi.cross_attention(q, k, k)):
        with pytest.raises(ValueError):   # the last one: no operand is on a device
            call()


def test_cross_attention_binding_refuses_heads_of_no_elements():
    for scale in (None, 1.0):
        with pytest.raises(ValueError):
            capi.cross_attention(torch.zeros(2, 5, 4, 0), torch.zeros(2, 7, 2, 0), torch.zeros(2, 7, 2, 0), scale)
