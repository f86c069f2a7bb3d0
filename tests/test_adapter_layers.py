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
