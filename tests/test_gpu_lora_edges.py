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
