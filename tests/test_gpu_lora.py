"""Adapters beside a quantized projection (quantized_linear_lora) and their
gradient (lora_backward) against float64, where masks, sizes, strides, streams
and graphs can go wrong.

The projection's own arithmetic is held to its parity tolerance elsewhere; here
most cases give it zero scales and biases, so that y is the adapters' term alone
and its bound is that term's (tests/adapter_ref.py)."""
import pytest
import torch

import qw_b200
from qw_b200 import _lib
from tests.adapter_ref import U, close, half_step, lora_delta, lora_grads
from tests.conftest import TOL, rel_err

pytestmark = pytest.mark.gpu

# M, N, K, R, L, bits, group: one row, either side of the decode kernel's 16 rows, of the 32-row and 256-row tiles,
# ranks that are no multiple of 8, more adapters than rows of a tile, N of no alignment
FORWARD = [
    (1, 8, 64, 1, 1, 4, 64), (1, 640, 1024, 16, 3, 4, 64), (3, 129, 192, 8, 3, 4, 64), (7, 1000, 256, 12, 5, 8, 128),
    (16, 200, 1024, 16, 40, 4, 64), (17, 130, 512, 12, 5, 4, 64), (32, 128, 256, 8, 64, 8, 64),
    (33, 257, 320, 5, 7, 4, 64), (64, 96, 192, 33, 4, 4, 64), (300, 520, 640, 64, 300, 4, 128),
    (513, 128, 256, 128, 2, 4, 64), (700, 1027, 384, 24, 9, 8, 64),
]


def rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def adapters(M, N, K, R, L, seed=0, none=0.2):
    g = rng(seed)
    x = torch.randn(M, K, generator=g, device="cuda").half()
    a = (torch.randn(L, R, K, generator=g, device="cuda") * K ** -0.5).half()
    b = torch.randn(L, N, R, generator=g, device="cuda").half()
    s = torch.rand(L, generator=g, device="cuda") + 0.5
    idx = torch.randint(0, L, (M,), generator=g, device="cuda", dtype=torch.int32)
    idx[torch.rand(M, generator=g, device="cuda") < none] = -1
    return x, a, b, s, idx


def zero_weights(N, K, bits=4, gs=64):
    z = torch.zeros(N, K // gs, dtype=torch.float16, device="cuda")
    return torch.zeros(N, K * bits // 32, dtype=torch.int32, device="cuda"), z, z.clone()


def real_weights(N, K, bits=4, gs=64, seed=5):
    w = (torch.randn(N, K, generator=rng(seed), device="cuda") * 0.02).half()
    return qw_b200.quantize_weights(w, group_size=gs, bits=bits)


def delta_of(x, a, b, s, idx):
    out, bound = lora_delta(x, a, b, s, idx, half_h=x.shape[0] > 16)
    return out, bound + half_step(torch.float16) * (out.abs() + bound) + 2.0 ** -25


@pytest.mark.parametrize("M,N,K,R,L,bits,gs", FORWARD)
def test_adapter_term(cuda_dev, M, N, K, R, L, bits, gs):
    x, a, b, s, idx = adapters(M, N, K, R, L, seed=M)
    y = qw_b200.quantized_linear_lora(x, *zero_weights(N, K, bits, gs), a, b, s, idx, group_size=gs, bits=bits)
    close(y, *delta_of(x, a, b, s, idx), "y")


@pytest.mark.parametrize("M,N,K,R,L,bits,gs", FORWARD)
def test_with_projection(cuda_dev, M, N, K, R, L, bits, gs):
    x, a, b, s, idx = adapters(M, N, K, R, L, seed=M + 1)
    w = real_weights(N, K, bits, gs)
    bias = torch.randn(N, generator=rng(3), device="cuda").half()
    y = qw_b200.quantized_linear_lora(x, *w, a, b, s, idx, linear_bias=bias, group_size=gs, bits=bits)
    q = (w[0].cpu()[..., None] >> torch.arange(0, 32, bits, dtype=torch.int32)) & (2 ** bits - 1)
    W = (q.view(N, -1, gs).double() * w[1].cpu().double()[..., None] + w[2].cpu().double()[..., None]).view(N, K)
    want = x.cpu().double() @ W.T + bias.cpu().double() + lora_delta(x, a, b, s, idx, False)[0]
    assert rel_err(y.cpu().numpy(), want.numpy()) <= TOL


@pytest.mark.parametrize("bits,gs", [(4, 64), (8, 128)])
@pytest.mark.parametrize("M", [1, 5, 16, 20, 300])
def test_rows_without_adapter_are_the_projection(cuda_dev, M, bits, gs):
    """Bit for bit up to 16 rows.  Above, the weights are rounded to fp16 once (half a step each) and y once; the
    K products are added in fp32."""
    N, K = 264, 512
    x, a, b, s, _ = adapters(M, N, K, 16, 4, seed=M)
    a[:], b[:] = float("nan"), float("inf")
    w = real_weights(N, K, bits, gs)
    w[1][0], w[2][0] = 1e-4, -5e-4  # rows of a scale near fp16's subnormals, and beyond either side of the tensor
    w[1][1], w[2][1] = 3.0, -20.0    # cores' dequantization rule
    w[1][2], w[2][2] = 0.01, 0.1
    w[1][3], w[2][3] = -3e-8, 0.25
    plain = qw_b200.quantized_matmul(x, *w, group_size=gs, bits=bits)
    q = (w[0].cpu()[..., None] >> torch.arange(0, 32, bits, dtype=torch.int32)) & (2 ** bits - 1)
    W = (q.view(N, -1, gs).double() * w[1].cpu().double()[..., None] + w[2].cpu().double()[..., None]).view(N, K)
    want, mags = x.cpu().double() @ W.T, x.cpu().double().abs() @ W.abs().T
    bound = (half_step(torch.float16) + (K + 4) * U) * mags + 2.0 ** -25 * x.cpu().double().abs().sum(1, keepdim=True)
    bound = bound + half_step(torch.float16) * (want.abs() + bound) + 2.0 ** -25
    for none in (-1, 4, -2, 2 ** 31 - 1):
        idx = torch.full((M,), none, dtype=torch.int32, device="cuda")
        y = qw_b200.quantized_linear_lora(x, *w, a, b, s, idx, group_size=gs, bits=bits)
        if M <= 16:
            assert torch.equal(y, plain)
        else:
            close(y, want, bound, "y")
    empty = qw_b200.quantized_linear_lora(x, *w, a[:0], b[:0], s[:0], None, group_size=gs, bits=bits)
    assert torch.equal(empty, y)


@pytest.mark.parametrize("M", [2, 16, 40, 280])
def test_non_finite_values_stay_in_their_rows(cuda_dev, M):
    N, K, R, L = 136, 256, 8, 5
    x, a, b, s, idx = adapters(M, N, K, R, L, seed=M, none=0.0)
    idx[:] = torch.arange(M, device="cuda") % (L - 1)
    want, bound = delta_of(x, a, b, s, idx)
    x2, a2 = x.clone(), a.clone()
    x2[0], x2[M - 1] = float("nan"), float("inf")
    a2[L - 1] = float("nan")  # nobody's adapter
    a2[(M - 1) % (L - 1)] = float("inf")
    bad = idx == (M - 1) % (L - 1)
    bad[0] = True
    bad = bad.cpu()
    y = qw_b200.quantized_linear_lora(x2, *zero_weights(N, K), a2, b, s, idx).cpu()
    close(y[~bad], want[~bad], bound[~bad], "the other rows")
    assert not torch.isfinite(y[bad]).all(1).any()


@pytest.mark.parametrize("M", [4, 48])
def test_single_adapter_defaults_and_strided_x(cuda_dev, M):
    N, K, R = 192, 256, 16
    x, a, b, _, _ = adapters(M, N, K, R, 1, seed=M)
    wide = torch.full((M, K + 64), float("nan"), dtype=torch.float16, device="cuda")
    wide[:, 8:8 + K] = x
    y = qw_b200.quantized_linear_lora(wide[:, 8:8 + K], *zero_weights(N, K), a, b)
    close(y, *delta_of(x, a, b, None, None), "y")
    y3 = qw_b200.quantized_linear_lora(x.view(2, M // 2, K), *zero_weights(N, K), a, b)
    assert y3.shape == (2, M // 2, N) and torch.equal(y3.view(M, N), y)


def test_no_rows(cuda_dev):
    x, a, b, s, idx = adapters(0, 64, 128, 4, 2)
    assert qw_b200.quantized_linear_lora(x, *zero_weights(64, 128), a, b, s, idx).shape == (0, 64)
    dx, da, db = qw_b200.lora_backward(x, torch.empty(0, 64, dtype=torch.float16, device="cuda"), a, b, s, idx)
    assert dx.shape == (0, 128) and not da.any() and not db.any()


@pytest.mark.parametrize("M", [1, 16, 100])
def test_graphs_and_streams(cuda_dev, M):
    """Two graphs captured on one stream replay at the same time on two others
    with new inputs; eager calls on a side stream agree."""
    N, K, R, L = 520, 512, 16, 6
    w = real_weights(N, K)
    sets = [adapters(M, N, K, R, L, seed=i) for i in range(2)]
    want = [qw_b200.quantized_linear_lora(s[0], *w, *s[1:]) for s in sets]
    bufs = [[t.clone() for t in sets[0]] for _ in range(2)]
    outs = [torch.empty(M, N, dtype=torch.float16, device="cuda") for _ in range(2)]
    graphs, side = [], torch.cuda.Stream()
    torch.cuda.synchronize()
    for bf, o in zip(bufs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            qw_b200.quantized_linear_lora(bf[0], *w, *bf[1:], out=o)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for rep in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                for dst, src in zip(bufs[i], sets[(i + rep) % 2]):
                    dst.copy_(src)
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], want[(i + rep) % 2])
    with torch.cuda.stream(side):
        y = qw_b200.quantized_linear_lora(sets[1][0], *w, *sets[1][1:])
    side.synchronize()
    assert torch.equal(y, want[1])
    assert qw_b200.device_status(0) == 0


def test_linear_and_mlp_take_adapters(cuda_dev):
    H, I, L, M = 256, 192, 3, 9
    x, a, b, s, idx = adapters(M, I, H, 8, L, seed=1)
    gw, uw, dw = real_weights(I, H, seed=1), real_weights(I, H, seed=2), real_weights(H, I, seed=3)
    lora = qw_b200.LoraAdapters(a, b, s)
    gate = qw_b200.QuantizedLinear(*gw, lora=lora)
    assert torch.equal(gate(x, adapter_idx=idx), qw_b200.quantized_linear_lora(x, *gw, a, b, s, idx))
    up, down = qw_b200.QuantizedLinear(*uw), qw_b200.QuantizedLinear(*dw)
    mlp = qw_b200.QuantizedMlp(gate, up, down)
    assert not mlp.fused
    hidden = qw_b200.compiled_swiglu_activation(gate(x, adapter_idx=idx), up(x))
    assert torch.equal(mlp(x, adapter_idx=idx), down(hidden))
    qkv = qw_b200.QuantizedFusedLinear(gate, [100, 60, 32])
    assert torch.equal(torch.cat(qkv(x, adapter_idx=idx), -1), gate(x, adapter_idx=idx))
    with pytest.raises(ValueError, match="adapters"):
        qw_b200.QuantizedFusedLinear.from_linears([gate, up])


# M, N, K, R, L: one row, a row tile more or less, ranks of no alignment, odd N, several row splits, empty adapters
BACKWARD = [(1, 8, 64, 1, 1), (5, 129, 192, 8, 3), (16, 200, 1024, 16, 40), (63, 130, 512, 12, 5), (64, 64, 64, 64, 1),
            (65, 257, 320, 5, 7), (300, 520, 640, 64, 300), (513, 128, 256, 128, 2), (1500, 260, 384, 24, 3),
            (2050, 1027, 128, 16, 1)]


@pytest.mark.parametrize("M,N,K,R,L", BACKWARD)
def test_gradients(cuda_dev, M, N, K, R, L):
    x, a, b, s, idx = adapters(M, N, K, R, L, seed=M)
    dy = (torch.randn(M, N, generator=rng(M + 1), device="cuda") * 1e-3).half()
    want, bound = lora_grads(x, dy, a, b, s, idx)
    got = qw_b200.lora_backward(x, dy, a, b, s, idx)
    for g, w, e, n in zip(got, want, bound, ("dx", "da", "db")):
        close(g, w, e, n)
    again = qw_b200.lora_backward(x, dy, a, b, s, idx)
    assert all(torch.equal(p, q) for p, q in zip(got, again)), "the same inputs give the same bits"


@pytest.mark.parametrize("M", [6, 200])
def test_accumulated_dx_and_strided_x(cuda_dev, M):
    N, K, R, L = 72, 128, 8, 3
    x, a, b, s, idx = adapters(M, N, K, R, L, seed=M, none=0.3)
    dy = torch.randn(M, N, generator=rng(4), device="cuda").half()
    base = torch.randn(M, K, generator=rng(6), device="cuda").half()
    wide = torch.full((M, K + 24), float("nan"), dtype=torch.float16, device="cuda")
    wide[:, 16:16 + K] = x
    dx = base.clone()
    out, da, db = qw_b200.lora_backward(wide[:, 16:16 + K], dy, a, b, s, idx, dx=dx)
    assert out.data_ptr() == dx.data_ptr()
    (wx, wa, wb), (ex, ea, eb) = lora_grads(x, dy, a, b, s, idx)
    total = wx + base.cpu().double()
    close(dx, total, ex + half_step(torch.float16) * total.abs() + 2.0 ** -23 * base.cpu().double().abs(), "dx")
    close(da, wa, ea, "da")
    close(db, wb, eb, "db")
    none = (idx == -1).cpu()
    assert torch.equal(dx.cpu()[none], base.cpu()[none])


def test_gradients_against_differences(cuda_dev):
    M, N, K, R, L = 50, 70, 128, 6, 3
    x, a, b, s, idx = adapters(M, N, K, R, L, seed=8)
    dy = torch.randn(M, N, generator=rng(9), device="cuda").half()
    dx, da, db = qw_b200.lora_backward(x, dy, a, b, s, idx)
    (_, _, _), (ex, ea, eb) = lora_grads(x, dy, a, b, s, idx)
    cpu = [t.cpu().double() for t in (x, a, b)]

    def f(x_, a_, b_):
        return float((lora_delta(x_, a_, b_, s, idx, False)[0] * dy.cpu().double()).sum())

    for i, (grad, e) in enumerate(zip((dx, da, db), (ex, ea, eb))):
        d = torch.randn(cpu[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
        hi, lo = list(cpu), list(cpu)
        hi[i], lo[i] = cpu[i] + d, cpu[i] - d  # f is linear in each operand: any step is exact
        diff = (f(*hi) - f(*lo)) / 2
        got = float((grad.cpu().double() * d).sum())
        assert abs(diff - got) <= float((e * d.abs()).sum()) + 1e-9 * abs(diff)


def test_partial_outputs_and_non_finite_gradients(cuda_dev):
    M, N, K, R, L = 130, 96, 192, 16, 4
    x, a, b, s, idx = adapters(M, N, K, R, L, seed=2, none=0.0)
    idx[:] = torch.arange(M, device="cuda") % L
    dy = torch.randn(M, N, generator=rng(3), device="cuda").half()
    full = qw_b200.lora_backward(x, dy, a, b, s, idx)
    lib = _lib.load()
    from qw_b200.ops import _arr, _stream, _workspace
    for keep in range(3):
        outs = [torch.empty_like(t) if i == keep else None for i, t in enumerate(full)]
        ws = _workspace("qw_lora_backward_workspace", x, M, N, K, R, L)
        _lib.check(lib.qw_lora_backward(_arr(x), _arr(dy), _arr(a), _arr(b), _arr(s), _arr(idx), 0, _arr(outs[0]),
                                        _arr(outs[1]), _arr(outs[2]), ws.data_ptr(), ws.nbytes, _stream(x)))
        assert torch.equal(outs[keep], full[keep])
    dy[2] = float("inf")  # a row of adapter 2
    dx, da, db = qw_b200.lora_backward(x, dy, a, b, s, idx)
    for l in range(L):
        assert torch.equal(da[l], full[1][l]) == (l != 2) and torch.equal(db[l], full[2][l]) == (l != 2)
    assert not torch.isfinite(da[2]).all() and not torch.isfinite(db[2]).all()
    others = (idx != 2).cpu()
    assert torch.equal(dx.cpu()[others], full[0].cpu()[others])


def test_gradient_graphs_replay_together(cuda_dev):
    M, N, K, R, L = 260, 200, 256, 16, 3
    sets = [adapters(M, N, K, R, L, seed=i) for i in range(2)]
    dys = [torch.randn(M, N, generator=rng(7 + i), device="cuda").half() for i in range(2)]
    want = [qw_b200.lora_backward(s[0], d, *s[1:]) for s, d in zip(sets, dys)]
    side, streams = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s, d in zip(sets, dys):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(qw_b200.lora_backward(s[0], d, *s[1:]))
        graphs.append(g)
    for _ in range(10):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(p, q) for p, q in zip(o, w))
            for t in o:
                t.zero_()
        torch.cuda.synchronize()


def test_operands_on_different_devices_are_refused(cuda_dev):
    x, a, b, s, idx = adapters(2, 64, 64, 4, 2)
    with pytest.raises(ValueError, match="operands on"):
        qw_b200.quantized_linear_lora(x, *zero_weights(64, 64), a, b, s, idx.cpu())
    with pytest.raises(_lib.QwError, match="overlap"):
        buf = torch.zeros(4, 64, dtype=torch.float16, device="cuda")
        qw_b200.quantized_linear_lora(buf[:2], *zero_weights(64, 64), a, b, s, idx, out=buf[1:3])
