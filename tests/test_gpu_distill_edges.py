"""Distillation where a row's cluster, its shared memory or its teacher reach
their limits (topk_distillation against float64)."""
import pytest
import torch

import qw_b200
from tests.adapter_ref import close, distill
from tests.test_gpu_distill import batch, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [8200, 8201, 66000])
@pytest.mark.parametrize("M", [1, 3, 60, 400])
def test_clusters_whose_first_rows_are_short_or_skipped(cuda_dev, M, V):
    """Rows of few columns a CTA, and whole first rounds without weight: the first shares go to CTAs that have only
    just begun."""
    z, idx, t, w = batch(M, V, 3, torch.float16, seed=M)
    w[torch.arange(M, device="cuda") % 5 < 2] = 0.0
    want, bound = distill(z, idx, t, 1.0, w)
    first = qw_b200.topk_distillation(z, idx, t, row_weights=w)
    close(first[0], want[0], bound[0], "loss")
    close(first[1], want[1], bound[1], "dlogits")
    for _ in range(50):
        again = qw_b200.topk_distillation(z, idx, t, row_weights=w)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
