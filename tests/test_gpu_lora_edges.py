"""Adapters beside a projection where the values of one operand leave fp16 or
the real numbers, and where a tile has hardly any work (quantized_linear_lora
against float64)."""
import pytest
import torch

import qw_b200
from tests.adapter_ref import close
from tests.test_gpu_lora import adapters, delta_of, real_weights, zero_weights

pytestmark = pytest.mark.gpu

INF = float("inf")


def with_bad_b(y, x, a, b, s, idx, bad):
    """y (float64, of the finite lora_b) with what the `bad` entries (adapter, column, rank, value) make of it."""
    y = y.clone()
    for l, n, r, v in bad:
        for m in (idx.cpu() == l).nonzero().flatten().tolist():
            y[m, n] += float(s[l]) * float(x[m].double().cpu() @ a[l, r].double().cpu()) * v
    return y


@pytest.mark.parametrize("M,N,K", [(20, 40000, 64), (20, 40000, 128), (32, 57000, 192), (300, 40000, 64)])
def test_infinite_b_in_tiles_of_few_blocks(cuda_dev, M, N, K):
    """Three row tiles a CTA and more, each of two or three k blocks: several are under way at once."""
    R, L = 8, 2
    x, a, b, s, idx = adapters(M, N, K, R, L, seed=M + K, none=0.0)
    idx[0], idx[1] = 0, 1
    want, bound = delta_of(x, a, b, s, idx)
    bad = [(0, 5, 3, INF), (1, 130, 0, -INF), (0, 148 * 128 + 7, 1, INF), (1, 2 * 148 * 128 + 60, 7, INF), (0, N - 1, 2, INF)]
    for l, n, r, v in bad:
        b[l, n, r] = v
    want = with_bad_b(want, x, a, b, s, idx, bad)
    for _ in range(5):
        close(qw_b200.quantized_linear_lora(x, *zero_weights(N, K), a, b, s, idx), want, bound, "y")


@pytest.mark.parametrize("M,R,bits,gs", [(17, 8, 4, 64), (32, 12, 8, 128), (40, 5, 4, 128), (300, 64, 8, 64),
                                         (600, 40, 4, 64)])
def test_non_finite_b_of_an_adapter_in_use(cuda_dev, M, R, bits, gs):
    N, K, L = 264, 256, 4
    x, a, b, s, idx = adapters(M, N, K, R, L, seed=R)
    idx[:6] = torch.tensor([0, 1, 2, 3, 2, -1], dtype=torch.int32)
    want, bound = delta_of(x, a, b, s, idx)
    bad = [(0, 0, R - 1, INF), (2, 129, 0, -INF), (2, N - 1, 1, INF), (1, 64, 2, float("nan"))]
    for l, n, r, v in bad:
        b[l, n, r] = v
    want = with_bad_b(want, x, a, b, s, idx, bad)
    y = qw_b200.quantized_linear_lora(x, *zero_weights(N, K, bits, gs), a, b, s, idx, group_size=gs, bits=bits)
    close(y, want, bound, "y")
    assert not torch.isfinite(y[0, 0]) and torch.isfinite(y[5]).all()


@pytest.mark.parametrize("M,R", [(600, 64), (513, 33), (1025, 128)])
def test_an_empty_stack_of_a_high_rank(cuda_dev, M, R):
    N, K = 136, 256
    x, a, b, s, _ = adapters(M, N, K, R, 1, seed=R)
    w = real_weights(N, K)
    empty = qw_b200.quantized_linear_lora(x, *w, a[:0], b[:0], s[:0], None)
    none = torch.full((M,), -1, dtype=torch.int32, device="cuda")
    assert torch.equal(empty, qw_b200.quantized_linear_lora(x, *w, a, b, s, none))
    dx, da, db = qw_b200.lora_backward(x, empty, a[:0], b[:0], s[:0], None)
    assert not dx.any() and da.shape == (0, R, K) and db.shape == (0, N, R)


@pytest.mark.parametrize("M,R,L", [(17, 8, 3), (32, 5, 2), (48, 16, 6), (300, 12, 300), (600, 48, 4), (700, 128, 2)])
def test_rank_products_beyond_fp16(cuda_dev, M, R, L):
    """h of some rows passes 65504, y does not: as finite as up to 16 rows.  One such rank meets an infinite lora_b."""
    N, K = 200, 256
    x, a, b, s, idx = adapters(M, N, K, R, L, seed=M + R)
    a, b = (a * 16).half(), (b * 2.0 ** -8).half()
    x[::3] = (x[::3] * 8192).half()
    idx[0], idx[3], idx[4] = 0, 1, 0
    h = s[idx.long().clamp_min(0)][:, None] * torch.einsum("mk,mrk->mr", x.float(), a.float()[idx.long().clamp_min(0)])
    assert (h.abs() > 66000).any() and (h.abs() < 60000).any()
    want, bound = delta_of(x, a, b, s, idx)
    assert want.abs().max() < 60000
    y = qw_b200.quantized_linear_lora(x, *zero_weights(N, K), a, b, s, idx)
    close(y, want, bound, "y")
    few = torch.cat([qw_b200.quantized_linear_lora(x[i:i + 16], *zero_weights(N, K), a, b, s, idx[i:i + 16])
                     for i in range(0, M, 16)])
    close(few, want, bound, "y in calls of 16 rows")
    bad = [(0, 7, R - 1, INF), (1, 150, 0, -INF)]
    for l, n, r, v in bad:
        b[l, n, r] = v
    close(qw_b200.quantized_linear_lora(x, *zero_weights(N, K), a, b, s, idx),
          with_bad_b(want, x, a, b, s, idx, bad), bound, "y")


@pytest.mark.parametrize("M,R", [(20, 5), (40, 12), (300, 3), (600, 44)])
def test_an_infinite_input_is_no_nan(cuda_dev, M, R):
    """Ranks that pad h stay zero: infinity times the zeros beside them would be NaN."""
    N, K = 136, 128
    x, a, b, s, _ = adapters(M, N, K, R, 1, seed=R)
    x, a, b = x.abs(), a.abs() + 2.0 ** -6, b.abs() + 2.0 ** -6
    ones = torch.ones(N, K // 64, dtype=torch.float16, device="cuda")
    w = (torch.zeros(N, K // 8, dtype=torch.int32, device="cuda"), torch.zeros_like(ones), ones)
    x[1, 70] = INF
    y = qw_b200.quantized_linear_lora(x, *w, a.half(), b.half(), s, None)
    assert (y[1] == INF).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[2:]).all()
