"""The adapters' gradient to the bits it states (lora_backward against float64)."""
import pytest
import torch

import qw_b200
from tests.adapter_ref import U, close, half_step, owners
from tests.test_gpu_adapter_edges import runs
from tests.test_gpu_lora import adapters, rng

pytestmark = pytest.mark.gpu


def dx_of(dy, a, b, s, idx, base=None):
    """(dx, bound) of s (dy B) A + base in float64.  The bound: g's fp32 sums (N terms, the scale), its two fp16 terms
    (2^-21 of its largest magnitude in the adapter), the 2 R products of a sum and the scale back, base's addition, one
    rounding of the result."""
    dy, a, b, s = (t.cpu().double() for t in (dy, a, b, s))
    N, R = dy.shape[1], a.shape[1]
    own = owners(idx, len(dy), len(a))
    out = torch.zeros(len(dy), a.shape[2]).double() if base is None else base.cpu().double().clone()
    bound = torch.zeros_like(out)
    for l in range(len(a)):
        r = (own == l).nonzero().flatten()
        if not len(r):
            continue
        g = s[l] * (dy[r] @ b[l])
        dg = (N + 4) * U * s[l].abs() * (dy[r].abs() @ b[l].abs()) + 2.0 ** -21 * g.abs().max()
        out[r] += g @ a[l]
        bound[r] = dg @ a[l].abs() + (2 * R + 8) * U * (g.abs() @ a[l].abs() + out[r].abs())
    return out, bound + half_step(torch.float16) * (out.abs() + bound) + 2.0 ** -25


@pytest.mark.parametrize("M,N,K,R,L", [(64, 96, 256, 16, 1), (130, 72, 192, 8, 2), (300, 257, 320, 40, 3),
                                       (700, 128, 128, 64, 2), (260, 136, 448, 128, 3), (1500, 64, 64, 20, 4)])
def test_dx_keeps_what_an_fp32_product_would(cuda_dev, M, N, K, R, L):
    x, a, b, s, idx = adapters(M, N, K, R, L, seed=M + 5)
    dy = torch.randn(M, N, generator=rng(M), device="cuda").half()
    want, bound = dx_of(dy, a, b, s, idx)
    close(qw_b200.lora_backward(x, dy, a, b, s, idx)[0], want, bound, "dx")
    base = torch.randn(M, K, generator=rng(6), device="cuda").half()
    want, bound = dx_of(dy, a, b, s, idx, base)
    close(qw_b200.lora_backward(x, dy, a, b, s, idx, dx=base.clone())[0], want, bound, "dx added")


@pytest.mark.parametrize("layout", [[(0, 128), (1, 3)], [(-1, 1), (0, 257), (1, 640)]])
def test_dx_of_runs(cuda_dev, layout):
    idx = runs(*layout)
    M, N, K, R = len(idx), 200, 256, 64
    x, a, b, s, _ = adapters(M, N, K, R, 2, seed=M)
    dy = torch.randn(M, N, generator=rng(M), device="cuda").half()
    want, bound = dx_of(dy, a, b, s, idx)
    close(qw_b200.lora_backward(x, dy, a, b, s, idx)[0], want, bound, "dx")
