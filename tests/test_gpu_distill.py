"""Distillation from a teacher's top logits (topk_distillation) against
float64: types, odd vocabularies, missing entries, repeated ids, masked logits,
rows without weight, in place, and in a graph."""
import pytest
import torch

import qw_b200
from tests.adapter_ref import close, distill

pytestmark = pytest.mark.gpu

INF = float("inf")


def rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def batch(M, V, k, dtype, seed=0, vdtype=None):
    g = rng(seed)
    base = torch.randn(M, V, generator=g, device="cuda") * 2.5
    z = (base + torch.randn(M, V, generator=g, device="cuda") * 0.7).to(dtype)
    vals, idx = base.topk(min(k, V), -1)
    if k > V:
        pad = k - V
        vals = torch.cat([vals, torch.zeros(M, pad, device="cuda")], -1)
        idx = torch.cat([idx, torch.full((M, pad), -1, device="cuda")], -1)
    w = torch.rand(M, generator=g, device="cuda") * 128 + 32
    return z, idx.to(torch.int32), vals.to(vdtype or dtype), w


def check(z, idx, t, T=1.0, w=None):
    temp = None if T == 1.0 else torch.tensor([T], device="cuda")
    want, bound = distill(z, idx, t, T, w)
    loss, dz = qw_b200.topk_distillation(z, idx, t, temperature=temp, row_weights=w)
    close(loss, want[0], bound[0], "loss")
    close(dz, want[1], bound[1], "dlogits")
    alone, none = qw_b200.topk_distillation(z, idx, t, temperature=temp, row_weights=w, grad=False)
    assert none is None
    close(alone, want[0], bound[0], "loss without the gradient")
    return loss, dz


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,V,k", [(1, 1, 1), (2, 3, 1), (3, 8, 3), (1, 1000, 7), (4, 1025, 50), (2, 8191, 128),
                                   (3, 20011, 16), (2, 40960, 1024), (2, 151936, 64), (5, 5, 16)])
def test_against_float64(cuda_dev, M, V, k, dtype):
    z, idx, t, w = batch(M, V, k, dtype, seed=V)
    check(z, idx, t, 2.0, w)


def test_rows_longer_than_registers_hold(cuda_dev):
    for dtype, V in ((torch.float16, 300000), (torch.float32, 270001)):
        check(*batch(2, V, 32, dtype, seed=1)[:3], 1.0, torch.tensor([64.0, 1.5], device="cuda"))


def test_defaults_and_mixed_types(cuda_dev):
    z, idx, t, _ = batch(4, 3000, 20, torch.float32, vdtype=torch.float16)
    check(z, idx, t)
    z, idx, t, _ = batch(4, 3000, 20, torch.float16, vdtype=torch.float32)
    check(z, idx, t, 0.5, torch.full((4,), 300.0, device="cuda"))
    loss, dz = qw_b200.topk_distillation(z.view(2, 2, -1), idx.view(2, 2, -1).long(), t.view(2, 2, -1))
    flat = qw_b200.topk_distillation(z, idx, t)
    assert loss.shape == (2, 2) and torch.equal(loss.flatten(), flat[0]) and torch.equal(dz.view(4, -1), flat[1])


@pytest.mark.parametrize("V", [777, 30000, 300001])
def test_entries_missing_repeated_or_weightless(cuda_dev, V):
    z, idx, t, w = batch(8, V, 12, torch.float32, seed=3)
    idx[0, 5:] = -1                      # fewer entries
    idx[1] = -1                          # none
    idx[2, 3:6] = idx[2, 0]              # an id three times more
    idx[3] = idx[3, 0]                   # one id only
    t[4, 4:] = -INF                      # entries without mass
    t[5] = -INF                          # no mass at all
    idx[6, 0], idx[6, 1] = V, V - 1      # just past the end, and the last column
    t[7, 1] = torch.finfo(torch.float32).min
    loss, dz = check(z, idx, t, 1.5, w)
    for m in (1, 5):
        assert loss[m] == 0 and not dz[m].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_masked_logits_and_rows(cuda_dev, dtype):
    z, idx, t, w = batch(7, 2500, 9, dtype, seed=4)
    keep = torch.zeros(2500, dtype=torch.bool, device="cuda")
    keep[idx[0].long()] = True
    z[0, ~keep] = -INF                              # only the teacher's columns left
    z[1, ~torch.isin(torch.arange(2500, device="cuda"), idx[1].long())] = torch.finfo(dtype).min
    z[2, idx[2, 0].long()] = -INF                   # a column the teacher wants: infinite loss
    z[3] = -INF                                     # nothing left
    z[4], w[4] = float("nan"), 0.0                  # a padded position holding anything
    z[5], w[5] = INF, 0.0
    loss, dz = check(z, idx, t, 1.0, w)
    assert loss[2] == INF and loss[3] == INF and loss[4] == 0 and loss[5] == 0
    assert not dz[4].any() and not dz[5].any() and torch.isfinite(dz).all()


@pytest.mark.parametrize("M,V,dtype", [(3, 1001, torch.float16), (9, 40000, torch.bfloat16), (2, 300000, torch.float16)])
def test_in_place_unaligned_and_repeatable(cuda_dev, M, V, dtype):
    z, idx, t, w = batch(M, V, 10, dtype, seed=5)
    loss, dz = qw_b200.topk_distillation(z, idx, t, row_weights=w)
    own = torch.empty(M * V + 1, dtype=dtype, device="cuda")[1:].view(M, V)  # a row start of 2-byte alignment
    own.copy_(z)
    loss2, dz2 = qw_b200.topk_distillation(own, idx, t, row_weights=w, dlogits=own)
    assert dz2.data_ptr() == own.data_ptr()
    want, bound = distill(z, idx, t, 1.0, w)
    close(loss2, want[0], bound[0], "loss in place")
    close(own, want[1], bound[1], "dlogits in place")
    again = qw_b200.topk_distillation(z, idx, t, row_weights=w)
    assert torch.equal(loss, again[0]) and torch.equal(dz, again[1])


def test_gradient_against_differences(cuda_dev):
    z, idx, t, w = batch(3, 500, 20, torch.float32, seed=6)
    T = 2.0
    _, dz = qw_b200.topk_distillation(z, idx, t, temperature=torch.tensor([T], device="cuda"), row_weights=w)
    bound = distill(z, idx, t, T, w)[1][1]
    d = torch.randn(3, 500, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    h = 1e-4
    zz = z.cpu().double()
    hi, lo = distill(zz + h * d, idx, t, T, w)[0][0], distill(zz - h * d, idx, t, T, w)[0][0]
    diff, got = (hi - lo) / (2 * h), (dz.cpu().double() * d).sum(1)
    # third derivatives of T^2 w KL are at most 2 w / T, directions of up to |d|^3 with q-weights: h^2 of it
    assert ((diff - got).abs() <= (bound * d.abs()).sum(1) + h * h * w.cpu() * d.abs().max() ** 3).all()


def test_in_a_graph_on_another_stream(cuda_dev):
    sets = [batch(6, 5003, 8, torch.float16, seed=i) for i in range(2)]
    want = [qw_b200.topk_distillation(s[0], s[1], s[2], row_weights=s[3]) for s in sets]
    buf = [x.clone() for x in sets[0]]
    torch.cuda.synchronize()
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=side):
        out = qw_b200.topk_distillation(buf[0], buf[1], buf[2], row_weights=buf[3])
    for i in (1, 0):
        for dst, src in zip(buf, sets[i]):
            dst.copy_(src)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[i][0]) and torch.equal(out[1], want[i][1])


def test_no_rows(cuda_dev):
    z, idx, t, w = batch(0, 100, 4, torch.float16)
    loss, dz = qw_b200.topk_distillation(z, idx, t, row_weights=w)
    assert loss.shape == (0,) and dz.shape == (0, 100)


def test_int64_ids_past_int32_are_no_entries(cuda_dev):
    z, idx, t, w = batch(3, 500, 6, torch.float16, seed=1)
    far = idx.to(torch.int64)
    idx[0, 2], idx[1, 0], idx[2, 5] = -1, -1, -1
    far[0, 2], far[1, 0], far[2, 5] = 2 ** 32 + 7, -2 ** 32 + 7, 2 ** 40
    want = qw_b200.topk_distillation(z, idx, t, row_weights=w)
    got = qw_b200.topk_distillation(z, far, t, row_weights=w)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
