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


@pytest.mark.parametrize("dtype,V", [(torch.float32, 500000), (torch.float32, 500003), (torch.float16, 1000000),
                                     (torch.bfloat16, 1000003)])
def test_rows_longer_than_a_cluster_s_shared_memory(cuda_dev, dtype, V):
    """What a share has beyond shared memory is read again; teacher ids all over the row, the ends of every CTA's share
    (the part that is read again) among them."""
    M, k = 3, 64
    z, idx, t, w = batch(M, V, k, dtype, seed=5)
    ends = (torch.arange(1, 9, device="cuda") * V) // 8
    idx[:, :24] = torch.cat([ends - 40, ends - 8, ends - 1]).int()
    idx[:, 24:28] = torch.tensor([0, 1, V - 17, V // 3], device="cuda", dtype=torch.int32)
    z[0, V - 30], z[1, V // 8 - 50] = 9.0, 11.0  # a maximum where it is not held
    w[2] = 0.0
    want, bound = distill(z, idx, t, 1.0, w)
    loss, dz = check(z, idx, t, 1.0, w)
    for shift in (0, 1):  # in place, from an aligned and an odd start
        own = torch.empty(M * V + shift, dtype=dtype, device="cuda")[shift:].view(M, V)
        own.copy_(z)
        loss, _ = qw_b200.topk_distillation(own, idx, t, row_weights=w, dlogits=own)
        close(loss, want[0], bound[0], "loss in place")
        close(own, want[1], bound[1], "dlogits in place")


def test_a_temperature_without_dimensions(cuda_dev):
    z, idx, t, w = batch(3, 900, 5, torch.float16)
    want = qw_b200.topk_distillation(z, idx, t, torch.tensor([2.0], device="cuda"), w)
    got = qw_b200.topk_distillation(z, idx, t, torch.tensor(2.0, device="cuda"), w)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
