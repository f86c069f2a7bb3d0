"""CPU tests of the Python side of adapters and distillation: what reaches the
library, and how the layer types pass adapters on.  No GPU."""
import pytest
import torch

from qw_b200 import ops


@pytest.mark.parametrize("pack", [ops._desc, ops._arr])
@pytest.mark.parametrize("shape", [(5,), (3, 4), (2, 3, 4)])
def test_one_value_over_a_shape_is_no_array(pack, shape):
    """All its strides are zero, which the library takes for row-contiguous: it would read past the value."""
    with pytest.raises(ValueError, match="row-contiguous"):
        pack(torch.ones(()).expand(shape))
    pack(torch.ones(1).expand(1))
    pack(torch.ones(shape))
    pack(torch.ones(4).expand(3, 4))  # strides (0, 1): refused by the library itself
    pack(torch.ones(0).expand(2, 0))


def linear(n, k=64, lora=None):
    return ops.QuantizedLinear(torch.zeros(n, k // 8, dtype=torch.int32), torch.zeros(n, 1, dtype=torch.float16),
                               torch.zeros(n, 1, dtype=torch.float16), lora=lora)


def stack(n, k=64, adapters=2, rank=4):
    return ops.LoraAdapters(torch.zeros(adapters, rank, k).half(), torch.zeros(adapters, n, rank).half())


def test_a_fused_gate_and_up_with_adapters_is_not_split():
    """Its halves would have lost them."""
    with pytest.raises(ValueError, match="adapters"):
        ops.QuantizedMlp.from_fused(linear(32, lora=stack(32)), 16, linear(64, 16 * 4))
    assert ops.QuantizedMlp.from_fused(linear(32), 16, linear(64)).fused


@pytest.fixture
def calls(monkeypatch):
    """Calls of the operators below the layer types, as (name, keyword arguments); each returns zeros."""
    log = []

    def fake(name, width):
        def f(x, *args, **kw):
            log.append((name, args, kw))
            return torch.zeros(*x.shape[:-1], width or args[0].shape[0])
        monkeypatch.setattr(ops, name, f)
    for name in ("quantized_matmul_swiglu", "quantized_linear_lora", "quantized_linear_forward"):
        fake(name, None)
    fake("compiled_swiglu_activation", 16)
    return log


@pytest.mark.parametrize("which", ["gate", "up"])
def test_adapters_attached_to_an_mlp_in_use(calls, which):
    mlp = ops.QuantizedMlp(linear(16), linear(16), linear(64, 64))
    x, idx = torch.zeros(3, 64), torch.zeros(3, dtype=torch.int32)
    mlp.forward_hidden(x)
    assert [c[0] for c in calls] == ["quantized_matmul_swiglu"]
    calls.clear()
    setattr(getattr(mlp, which), "lora", stack(16))
    mlp.forward_hidden(x, adapter_idx=idx)
    names = [c[0] for c in calls]
    assert sorted(names) == ["compiled_swiglu_activation", "quantized_linear_forward", "quantized_linear_lora"]
    assert calls[names.index("quantized_linear_lora")][1][6] is idx
    calls.clear()
    getattr(mlp, which).lora = None
    mlp.forward_hidden(x)
    assert [c[0] for c in calls] == ["quantized_matmul_swiglu"]


def test_adapters_attached_beside_a_global_scale_are_refused(calls):
    """The adapters' kernel would leave the scale out."""
    lin = linear(16, lora=stack(16))
    lin.global_scale = torch.ones(1)
    with pytest.raises(ValueError, match="global scale"):
        lin(torch.zeros(3, 64))
    assert not calls


class OwnLinear:
    """A caller's projection, as the layer types took it before there were adapters."""
    weight, scales, biases = torch.zeros(16, 8, dtype=torch.int32), torch.zeros(16, 1).half(), torch.zeros(16, 1).half()
    group_size, bits, mode, bias, global_scale, in_features, out_features = 64, 4, "affine", None, None, 64, 16

    def __call__(self, x, out=None):
        return torch.full((*x.shape[:-1], 16), 2.0)


def test_projections_that_know_no_adapters(calls):
    x = torch.zeros(3, 64)
    mlp = ops.QuantizedMlp(OwnLinear(), OwnLinear(), lambda h, out=None: h + 1)
    assert mlp.fused and torch.equal(mlp(x), torch.ones(3, 16))
    other = OwnLinear()
    other.bias = torch.zeros(16)
    assert torch.equal(ops.QuantizedMlp(OwnLinear(), other, lambda h, out=None: h + 1)(x), torch.ones(3, 16))
    a, b = ops.QuantizedFusedLinear(OwnLinear(), [10, 6])(x)
    assert a.shape == (3, 10) and b.shape == (3, 6)
    assert ops.QuantizedFusedLinear.from_linears([OwnLinear(), OwnLinear()]).linear.out_features == 32
    assert ops.QuantizedMlp.from_fused(OwnLinear(), 8, lambda h, out=None: h).fused


def test_a_projection_stored_before_there_were_adapters(calls):
    lin = linear(16)
    del lin.__dict__["lora"]
    lin(torch.zeros(3, 64))
    assert [c[0] for c in calls] == ["quantized_linear_forward"]
