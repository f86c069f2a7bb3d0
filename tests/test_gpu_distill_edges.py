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


@pytest.mark.parametrize("V", [700, 30001])
@pytest.mark.parametrize("vdtype", [torch.float16, torch.float32])
def test_a_teacher_of_nan_is_not_a_row_without_entries(cuda_dev, V, vdtype):
    """p is NaN: so are the loss and the columns that the teacher names; the others keep w T q."""
    nan = float("nan")
    z, idx, t, w = batch(5, V, 7, torch.float32, seed=2, vdtype=vdtype)
    plain = qw_b200.topk_distillation(z, idx, t, row_weights=w)[1]
    t[0] = nan
    t[1, 3] = nan
    t[2], t[2, 6] = -float("inf"), nan
    t[3], w[3] = nan, 0.0
    loss, dz = qw_b200.topk_distillation(z, idx, t, row_weights=w)
    assert loss[:3].isnan().all() and loss[3] == 0 and loss[4].isfinite()
    assert not dz[3].any() and torch.equal(dz[4], plain[4])
    named = torch.zeros(3, V, dtype=torch.bool, device="cuda").scatter_(1, idx[:3].long(), True)
    assert torch.equal(dz[:3].isnan(), named)
    assert torch.equal(dz[:3][~named], plain[:3][~named])
