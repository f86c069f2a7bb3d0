"""The adapter and distillation operators in a run, as they are used together:
an 8-bit head teaches a 4-bit head's adapter through its stored top logits, one
step per batch, then the trained stack serves rows of several requests."""
import pytest
import torch

import qw_b200
from tests.adapter_ref import lora_delta

pytestmark = pytest.mark.gpu


def dequantized(w, bits, gs):
    q = (w[0].cpu()[..., None] >> torch.arange(0, 32, bits, dtype=torch.int32)) & (2 ** bits - 1)
    N = w[0].shape[0]
    return (q.view(N, -1, gs).double() * w[1].cpu().double()[..., None] + w[2].cpu().double()[..., None]).view(N, -1)


def test_distil_a_head_into_its_adapter(cuda_dev):
    M, V, K, R, L, k = 96, 3001, 256, 8, 3, 16
    g = torch.Generator(device="cuda").manual_seed(0)
    w = (torch.randn(V, K, generator=g, device="cuda") * K ** -0.5 * 2).half()
    teacher = qw_b200.quantize_weights(w, bits=8)
    student = qw_b200.quantize_weights(w, bits=4)
    lora = qw_b200.LoraAdapters((torch.randn(L, R, K, generator=g, device="cuda") * K ** -0.5).half(),
                                (torch.randn(L, V, R, generator=g, device="cuda") * 0.1).half(),
                                torch.full((L,), 2.0, device="cuda"))
    head = qw_b200.QuantizedLinear(*student, lora=lora)
    x = torch.randn(M, K, generator=g, device="cuda").half()
    idx = torch.randint(-1, L - 1, (M,), generator=g, device="cuda", dtype=torch.int32)  # adapter 2 has no rows
    scale = torch.full((M,), 512.0, device="cuda")
    ids, values = qw_b200.quantized_matmul_topk(x, *teacher, k, bits=8)
    logits = head(x, adapter_idx=idx)
    loss, dlogits = qw_b200.topk_distillation(logits, ids, values, row_weights=scale)
    dx, da, db = lora.backward(x, dlogits, idx)

    # the same step in float64 with automatic differentiation
    a, b = lora.a.cpu().double().requires_grad_(), lora.b.cpu().double().requires_grad_()
    own = idx.cpu().long()
    z = x.cpu().double() @ dequantized(student, 4, 64).T
    parts = [(2.0 * (x.cpu().double() @ a[l].T) @ b[l].T) * (own == l)[:, None] for l in range(L)]
    z = z + sum(parts)
    logq, p = torch.log_softmax(z, -1), torch.softmax(values.cpu().double(), -1)
    want = 512.0 * (p * (p.log() - logq.gather(-1, ids.cpu()))).sum(-1)
    want.sum().backward()
    # logits and dlogits are fp16 arrays (errors of up to 1e-2 rms in the projection's parity tolerance), so the
    # step's outputs are held to the same measure
    assert float((loss.cpu().double() - want.detach()).abs().max() / want.detach().square().mean().sqrt()) <= 1e-2
    for got, ref in ((da, a.grad), (db, b.grad)):
        assert float((got.cpu().double() - ref).norm() / ref.norm()) <= 1e-2
        assert not got[L - 1].any()

    # an update reaches the next call, one adapter per request, single rows and batches alike
    lora.a.sub_((da * (0.01 / 512)).half())
    lora.b.sub_((db * (0.01 / 512)).half())
    y = head(x, adapter_idx=idx)
    ref = x.cpu().double() @ dequantized(student, 4, 64).T + lora_delta(x, lora.a, lora.b, lora.scales, idx, False)[0]
    tol = 1e-2 * float(ref.square().mean().sqrt())
    assert float((y.cpu().double() - ref).abs().max()) <= tol
    for m in (0, 1, M - 1):
        one = head(x[m:m + 1], adapter_idx=idx[m:m + 1])
        assert float((one.cpu().double() - ref[m:m + 1]).abs().max()) <= tol
