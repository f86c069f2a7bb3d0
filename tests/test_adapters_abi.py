"""CPU tests: argument checks of the adapter and distillation entry points, all
before any device work.  No GPU."""
import ctypes

import pytest
import torch

import qw_b200
from qw_b200 import _lib

U32, F16, BF16, F32 = _lib.QW_U32, _lib.QW_F16, _lib.QW_BF16, _lib.QW_F32


def arr(shape, dtype, ptr=0x10000, strides=None):
    a = _lib.QwArray()
    a.data, a.dtype, a.ndim = ptr, dtype, len(shape)
    for i, s in enumerate(shape):
        a.shape[i] = s
    for i, s in enumerate(strides or []):
        a.strides[i] = s
    return ctypes.pointer(a)


def err():
    return _lib.load().qw_last_error().decode()


M, N, K, R, L = 3, 256, 512, 16, 4


def forward(**change):
    v = dict(x=arr([M, K], F16), w=arr([N, K // 8], U32), s=arr([N, K // 64], F16), b=arr([N, K // 64], F16),
             bias=None, la=arr([L, R, K], F16), lb=arr([L, N, R], F16), ls=arr([L], F32), idx=arr([M], U32), gs=64,
             bits=4, mode=b"affine", y=arr([M, N], F16, 0x900000), ws=None, wsb=0)
    v.update(change)
    return _lib.load().qw_quantized_linear_lora(v["x"], v["w"], v["s"], v["b"], v["bias"], v["la"], v["lb"], v["ls"],
                                                v["idx"], v["gs"], v["bits"], v["mode"], v["y"], v["ws"], v["wsb"],
                                                None)


@pytest.mark.parametrize("change,code,msg", [
    (dict(la=None), _lib.QW_EINVAL, "lora_a is null"),
    (dict(lb=None), _lib.QW_EINVAL, "lora_b is null"),
    (dict(la=arr([L, R, K], BF16)), _lib.QW_EUNSUPPORTED, "float16"),
    (dict(la=arr([R, K], F16)), _lib.QW_EINVAL, "3-D"),
    (dict(la=arr([L, R, K - 64], F16)), _lib.QW_EINVAL, "width"),
    (dict(lb=arr([L, N + 1, R], F16)), _lib.QW_EINVAL, "lora_b must be"),
    (dict(lb=arr([L + 1, N, R], F16)), _lib.QW_EINVAL, "lora_b must be"),
    (dict(la=arr([L, 0, K], F16), lb=arr([L, N, 0], F16)), _lib.QW_EINVAL, "rank"),
    (dict(la=arr([L, 129, K], F16), lb=arr([L, N, 129], F16)), _lib.QW_EUNSUPPORTED, "rank"),
    (dict(la=arr([4097, R, K], F16), lb=arr([4097, N, R], F16)), _lib.QW_EUNSUPPORTED, "adapters"),
    (dict(ls=arr([L + 1], F32)), _lib.QW_EINVAL, "lora_scales"),
    (dict(ls=arr([L], F16)), _lib.QW_EINVAL, "lora_scales"),
    (dict(idx=arr([M + 1], U32)), _lib.QW_EINVAL, "adapter_idx"),
    (dict(idx=arr([M], F32)), _lib.QW_EINVAL, "adapter_idx"),
    (dict(la=arr([L, R, K], F16, 0x10008)), _lib.QW_EINVAL, "aligned"),
    (dict(la=arr([L, R, K], F16, strides=[R * K * 2, K, 1])), _lib.QW_EINVAL, "row-contiguous"),
    (dict(bias=arr([N + 1], F16)), _lib.QW_EINVAL, "linear_bias"),
    (dict(y=arr([M, N], F32, 0x900000)), _lib.QW_EINVAL, "float16"),
    (dict(y=arr([M, N], F16, 0x10000 + 2 * K)), _lib.QW_EINVAL, "overlap"),
    (dict(x=arr([M, K], BF16)), _lib.QW_EUNSUPPORTED, "float16"),
    (dict(gs=32), _lib.QW_EUNSUPPORTED, "group_size"),
    (dict(b=None), _lib.QW_EINVAL, "biases"),
])
def test_forward_refusals(change, code, msg):
    assert forward(**change) == code
    assert msg in err()


def test_forward_without_rows_is_a_no_op():
    assert forward(x=arr([0, K], F16, 0), idx=arr([0], U32, 0), y=arr([0, N], F16, 0)) == _lib.QW_OK


def backward(**change):
    v = dict(x=arr([M, K], F16), dy=arr([M, N], F16, 0x40000), la=arr([L, R, K], F16), lb=arr([L, N, R], F16),
             ls=arr([L], F32), idx=arr([M], U32), add=0, dx=arr([M, K], F16, 0x900000),
             da=arr([L, R, K], F32, 0xa00000), db=arr([L, N, R], F32, 0xb00000), ws=None, wsb=0)
    v.update(change)
    return _lib.load().qw_lora_backward(v["x"], v["dy"], v["la"], v["lb"], v["ls"], v["idx"], v["add"], v["dx"],
                                        v["da"], v["db"], v["ws"], v["wsb"], None)


@pytest.mark.parametrize("change,code,msg", [
    (dict(x=None), _lib.QW_EINVAL, "x is null"),
    (dict(dy=None), _lib.QW_EINVAL, "dy is null"),
    (dict(x=arr([M, 96], F16), la=arr([L, R, 96], F16)), _lib.QW_EINVAL, "multiple of 64"),
    (dict(dy=arr([M, N], F32)), _lib.QW_EUNSUPPORTED, "float16"),
    (dict(dy=arr([M + 1, N], F16)), _lib.QW_EINVAL, "dy must have shape"),
    (dict(dy=arr([M, N], F16, 0x40000, [N + 8, 1])), _lib.QW_EINVAL, "row-contiguous"),
    (dict(dx=None, da=None, db=None), _lib.QW_EINVAL, "all null"),
    (dict(dx=arr([M, K], F32, 0x900000)), _lib.QW_EINVAL, "dx must be"),
    (dict(dx=arr([M, K], F16, 0x10010)), _lib.QW_EINVAL, "overlap"),
    (dict(dx=arr([M, K], F16, 0x40000)), _lib.QW_EINVAL, "overlap"),
    (dict(da=arr([L, R, K], F16, 0xa00000)), _lib.QW_EINVAL, "da must be"),
    (dict(da=arr([L, K, R], F32, 0xa00000)), _lib.QW_EINVAL, "da must be"),
    (dict(db=arr([L, R, N], F32, 0xb00000)), _lib.QW_EINVAL, "db must be"),
    (dict(da=arr([L, R, K], F32, 0xa00004)), _lib.QW_EINVAL, "aligned"),
    (dict(la=arr([L, 129, K], F16), lb=arr([L, N, 129], F16)), _lib.QW_EUNSUPPORTED, "rank"),
    (dict(idx=arr([M - 1], U32)), _lib.QW_EINVAL, "adapter_idx"),
])
def test_backward_refusals(change, code, msg):
    assert backward(**change) == code
    assert msg in err()


def test_workspace_queries_check_their_sizes():
    lib, n = _lib.load(), ctypes.c_int64(0)
    assert lib.qw_quantized_linear_lora_workspace(1, 8, 129, ctypes.byref(n)) == _lib.QW_EINVAL
    assert lib.qw_quantized_linear_lora_workspace(-1, 8, 8, ctypes.byref(n)) == _lib.QW_EINVAL
    assert lib.qw_quantized_linear_lora_workspace(1, 8, 8, None) == _lib.QW_EINVAL
    assert lib.qw_lora_backward_workspace(1, 8, 64, 0, 1, ctypes.byref(n)) == _lib.QW_EINVAL
    assert lib.qw_lora_backward_workspace(1, 8, 64, 8, 5000, ctypes.byref(n)) == _lib.QW_EINVAL
    assert lib.qw_lora_backward_workspace(1, 8, 64, 8, 1, None) == _lib.QW_EINVAL


V, TOP = 1000, 8


def distill(**change):
    v = dict(z=arr([M, V], F16), idx=arr([M, TOP], U32), t=arr([M, TOP], F16), T=arr([1], F32), w=arr([M], F32),
             loss=arr([M], F32), dz=arr([M, V], F16, 0x900000))
    v.update(change)
    return _lib.load().qw_topk_distill(v["z"], v["idx"], v["t"], v["T"], v["w"], v["loss"], v["dz"], None)


@pytest.mark.parametrize("change,code,msg", [
    (dict(z=None), _lib.QW_EINVAL, "logits is null"),
    (dict(z=arr([M, V], U32)), _lib.QW_EUNSUPPORTED, "float16"),
    (dict(t=arr([M, TOP], U32)), _lib.QW_EUNSUPPORTED, "float16"),
    (dict(z=arr([M, 0], F16, 0)), _lib.QW_EINVAL, "empty"),
    (dict(idx=arr([M, 0], U32, 0)), _lib.QW_EINVAL, "at least one"),
    (dict(idx=arr([M, 1025], U32), t=arr([M, 1025], F16)), _lib.QW_EUNSUPPORTED, "1025"),
    (dict(idx=arr([M, TOP], F16)), _lib.QW_EINVAL, "teacher_idx"),
    (dict(idx=arr([M + 1, TOP], U32)), _lib.QW_EINVAL, "teacher_idx"),
    (dict(t=arr([M, TOP + 1], F16)), _lib.QW_EINVAL, "teacher_values"),
    (dict(T=arr([2], F32)), _lib.QW_EINVAL, "temperature"),
    (dict(T=arr([1], F16)), _lib.QW_EINVAL, "temperature"),
    (dict(w=arr([M + 1], F32)), _lib.QW_EINVAL, "row_weights"),
    (dict(loss=arr([M], F16)), _lib.QW_EINVAL, "loss"),
    (dict(loss=None), _lib.QW_EINVAL, "loss is null"),
    (dict(dz=arr([M, V], F32, 0x900000)), _lib.QW_EINVAL, "dlogits"),
    (dict(dz=arr([M, V - 1], F16, 0x900000)), _lib.QW_EINVAL, "dlogits"),
    (dict(dz=arr([M, V], F16, 0x10002)), _lib.QW_EINVAL, "overlap"),
    (dict(z=arr([M, V], F16, 0x10001)), _lib.QW_EINVAL, "misaligned"),
])
def test_distill_refusals(change, code, msg):
    assert distill(**change) == code
    assert msg in err()


def test_adapter_stack_shapes_are_checked():
    with pytest.raises(ValueError, match="adapters must be"):
        qw_b200.LoraAdapters(torch.zeros(2, 4, 8), torch.zeros(2, 8, 5))
    with pytest.raises(ValueError, match="global scale"):
        qw_b200.QuantizedLinear(None, None, None, global_scale=torch.ones(1),
                                lora=qw_b200.LoraAdapters(torch.zeros(2, 4, 8), torch.zeros(2, 8, 4)))


@pytest.mark.parametrize("change", [dict(dx=arr([M, K], F16, 0x10100), x=arr([M, K], F16, 0x70000)),
                                    dict(da=arr([L, R, K], F32, 0x40010)), dict(da=arr([L, R, K], F32, 0x9000c0)),
                                    dict(db=arr([L, N, R], F32, 0xa1ff00)), dict(db=arr([L, N, R], F32, 0x10000))])
def test_gradients_must_not_overlap_operands(change):
    assert backward(**change) == _lib.QW_EINVAL
    assert "overlap" in err()


@pytest.mark.parametrize("change", [dict(dz=arr([M, V], F16, 0x10000 + 0x1000), z=arr([M, V], F16, 0x500000),
                                         idx=arr([M, TOP], U32, 0x11770)),
                                    dict(loss=arr([M], F32, 0x900000)), dict(loss=arr([M], F32, 0x10004))])
def test_distillation_outputs_must_not_overlap_operands(change):
    assert distill(**change) == _lib.QW_EINVAL
    assert "overlap" in err()


def test_a_misaligned_bias_is_refused():
    assert forward(bias=arr([N], F16, 0x20001)) == _lib.QW_EINVAL
    assert "misaligned" in err()
    assert _lib.load().qw_quantized_linear_forward(
        arr([M, K], F16), arr([N, K // 8], U32), arr([N, K // 64], F16), arr([N, K // 64], F16),
        arr([N], F16, 0x20001), 64, 4, b"affine", arr([M, N], F16, 0x900000), None) == _lib.QW_EINVAL
    assert "misaligned" in err()


def test_a_bias_without_weights_is_refused():
    assert forward(w=None, bias=arr([N], F16)) == _lib.QW_EINVAL
    assert _lib.load().qw_quantized_linear_forward(
        arr([M, K], F16), None, arr([N, K // 64], F16), arr([N, K // 64], F16), arr([N], F16), 64, 4, b"affine",
        arr([M, N], F16, 0x900000), None) == _lib.QW_EINVAL
    assert "w is null" in err()
