"""Adapters and distillation where layouts and sizes reach other code: runs of
consecutive rows (whole and broken tiles), adapters without rows among very many,
infinities beside finite ranks, calls of two streams at once, and arrays beyond
2^31 elements."""
import ctypes

import pytest
import torch

import qw_b200
from qw_b200 import _lib, ops
from tests.adapter_ref import close, distill, lora_grads
from tests.test_gpu_lora import adapters, rng, zero_weights

pytestmark = pytest.mark.gpu


def runs(*lengths):
    """adapter_idx of (adapter, rows) runs."""
    return torch.cat([torch.full((n,), a, dtype=torch.int32) for a, n in lengths]).cuda()


@pytest.mark.parametrize("N,K,R", [(200, 256, 16), (333, 192, 40), (136, 448, 64), (128, 128, 128)])
@pytest.mark.parametrize("layout", [
    [(0, 128)], [(0, 129)], [(0, 127), (1, 1)], [(0, 256), (1, 8)],
    [(1, 300), (0, 5), (2, 3), (1, 77), (-1, 9), (0, 250), (2, 127), (0, 640)],
    [(-1, 130), (0, 1), (1, 700), (0, 2), (1, 333)],
])
def test_gradients_of_runs_of_rows(cuda_dev, layout, N, K, R):
    idx = runs(*layout)
    M, L = len(idx), 3
    x, a, b, s, _ = adapters(M, N, K, R, L, seed=M + R)
    dy = (torch.randn(M, N, generator=rng(M), device="cuda") * 1e-2).half()
    want, bound = lora_grads(x, dy, a, b, s, idx)
    for g, w, e, n in zip(qw_b200.lora_backward(x, dy, a, b, s, idx), want, bound, ("dx", "da", "db")):
        close(g, w, e, n)


def test_gradients_of_few_rows_among_many_adapters(cuda_dev):
    M, N, K, R, L = 40, 24, 64, 8, 4096
    x, a, b, s, idx = adapters(M, N, K, R, L, seed=2, none=0.3)
    idx[:3] = torch.tensor([0, 4095, 4095], dtype=torch.int32)
    dy = torch.randn(M, N, generator=rng(3), device="cuda").half()
    want, bound = lora_grads(x, dy, a, b, s, idx)
    for g, w, e, n in zip(qw_b200.lora_backward(x, dy, a, b, s, idx), want, bound, ("dx", "da", "db")):
        close(g, w, e, n)


def test_an_infinite_rank_leaves_the_others_their_values(cuda_dev):
    """lora_b is infinite for one rank: that rank's gradients are, those of the others stay within their bounds,
    with their own scale (g is beyond fp16)."""
    M, N, K, R, L = 150, 96, 128, 8, 2
    x, a, b, s, idx = adapters(M, N, K, R, L, seed=9, none=0.0)
    dy = (torch.rand(M, N, generator=rng(8), device="cuda") * 30000 + 100).half()
    finite = b.clone()
    finite[1, :, 3] = 0
    b[1, 5, 3] = float("inf")
    (wx, wa, wb), (_, ea, eb) = lora_grads(x, dy, a, finite, s, idx)
    dx, da, db = qw_b200.lora_backward(x, dy, a, b, s, idx)
    keep = torch.ones(L, R, dtype=torch.bool)
    keep[1, 3] = False
    close(da[keep.cuda()], wa[keep], ea[keep], "da")
    close(db, wb, eb, "db")  # of h, which does not meet lora_b
    assert not da[1, 3].isfinite().any()
    own = (idx == 1).cpu()
    # fp16 results beyond 65504 are infinite, whatever lora_b holds; the others are finite
    assert dx.cpu()[~own][wx[~own].abs() < 65000].isfinite().all()
    assert not dx.cpu()[own].isfinite().any()


def test_calls_of_two_streams_at_once(cuda_dev):
    N, K, R, L = 520, 640, 16, 5
    sets = []
    for M in (24, 700):
        x, a, b, s, idx = adapters(M, N, K, R, L, seed=M)
        dy = torch.randn(M, N, generator=rng(M), device="cuda").half()
        ids = torch.randint(0, N, (M, 9), generator=rng(1), device="cuda", dtype=torch.int32)
        t = torch.randn(M, 9, generator=rng(2), device="cuda").half()
        sets.append((x, a, b, s, idx, dy, ids, t))
    w = zero_weights(N, K)

    def step(x, a, b, s, idx, dy, ids, t):
        y = qw_b200.quantized_linear_lora(x, *w, a, b, s, idx)
        loss, dz = qw_b200.topk_distillation(y, ids, t)
        return (y, loss, dz, *qw_b200.lora_backward(x, dy, a, b, s, idx))

    want = [step(*c) for c in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        got = []
        for c, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(step(*c))
        torch.cuda.synchronize()
        for p, q in zip(want, got):
            assert all(torch.equal(u, v) for u, v in zip(p, q))


def test_arrays_beyond_2_31_elements(cuda_dev):
    """The last rows of y, dy, dx and of the logits lie past 2^31 elements."""
    if torch.cuda.get_device_properties(0).total_memory < 60 << 30:
        pytest.skip("takes 20 GB")
    M, N, K, R, L = 131200, 16400, 64, 4, 2
    x, a, b, s, _ = adapters(1, N, K, R, L, seed=1)
    rows = torch.cat([torch.arange(3), torch.arange(M - 3, M)])
    x = torch.zeros(M, K, dtype=torch.float16, device="cuda")
    x[rows.cuda()] = torch.randn(6, K, generator=rng(2), device="cuda").half()
    idx = torch.full((M,), -1, dtype=torch.int32, device="cuda")
    idx[rows.cuda()] = torch.tensor([0, 1, 1, 1, 0, 1], dtype=torch.int32, device="cuda")
    y = qw_b200.quantized_linear_lora(x, *zero_weights(N, K), a, b, s, idx)
    some = qw_b200.quantized_linear_lora(x[rows.cuda()].repeat(5, 1), *zero_weights(N, K), a, b, s,
                                         idx[rows.cuda()].repeat(5))[:6]  # 30 rows: the same kernels' h in fp16
    scale = float(some.double().square().mean().sqrt())
    assert float((y[rows.cuda()].double() - some.double()).abs().max()) <= 2.0 ** -8 * scale
    assert not y[3:M - 3].any()
    y.zero_()
    y[rows.cuda()] = torch.randn(6, N, generator=rng(3), device="cuda").half()
    want, bound = lora_grads(x[rows.cuda()], y[rows.cuda()], a, b, s, idx[rows.cuda()])
    dx, da, db = qw_b200.lora_backward(x, y, a, b, s, idx)
    close(dx[rows.cuda()], want[0], bound[0], "dx")
    assert not dx[3:M - 3].any()
    close(da, want[1], bound[1], "da")
    close(db, want[2], bound[2], "db")
    ids = torch.randint(0, N, (M, 4), generator=rng(4), device="cuda", dtype=torch.int32)
    t = torch.randn(M, 4, generator=rng(5), device="cuda").half()
    rw = torch.zeros(M, device="cuda")
    rw[rows.cuda()] = 64.0
    loss, dz = qw_b200.topk_distillation(y, ids, t, row_weights=rw)
    r = rows.cuda()
    want, bound = distill(y[r], ids[r], t[r], 1.0, rw[r])
    close(loss[r], want[0], bound[0], "loss")
    close(dz[r], want[1], bound[1], "dlogits")
    assert not loss[3:M - 3].any() and not dz[3:M - 3].any()


def test_workspaces_are_checked(cuda_dev):
    """One that is too small is refused."""
    M, N, K, R, L = 40, 72, 128, 8, 3
    x, a, b, s, idx = adapters(M, N, K, R, L, seed=4)
    dy = torch.randn(M, N, generator=rng(4), device="cuda").half()
    lib = _lib.load()
    n = ctypes.c_int64(0)
    _lib.check(lib.qw_lora_backward_workspace(M, N, K, R, L, ctypes.byref(n)))
    assert n.value > 0
    ops._WORKSPACE_BYTES.clear()
    try:
        ops._WORKSPACE_BYTES[("qw_lora_backward_workspace", x.get_device(), (M, N, K, R, L))] = n.value // 2 - 256
        with pytest.raises(Exception, match="workspace"):
            qw_b200.lora_backward(x, dy, a, b, s, idx)
    finally:
        ops._WORKSPACE_BYTES.clear()
    want, bound = lora_grads(x, dy, a, b, s, idx)
    close(qw_b200.lora_backward(x, dy, a, b, s, idx)[1], want[1], bound[1], "da")
