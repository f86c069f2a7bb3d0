"""Plain float64 implementations of the adapter and distillation operators,
with elementwise bounds on what fp32 arithmetic may differ from them by."""
import torch

U = 2.0 ** -23  # one fp32 step: the tensor cores' fp32 sums may truncate, so a whole step per addition


def half_step(t):
    """Largest relative error of one rounding to type t."""
    return torch.finfo(t).eps / 2


def owners(idx, M, L):
    """Adapter of each row as int64, L for none; ids are unsigned 32-bit."""
    a = torch.zeros(M, dtype=torch.int64) if idx is None else idx.cpu().to(torch.int64) & 0xFFFFFFFF
    return a.clamp(max=L)


def lora_delta(x, a, b, s, idx, half_h):
    """(delta, bound) of s (x A^T) B^T per row; half_h: the rank-space product is rounded to fp16."""
    x, a, b = x.cpu().double(), a.cpu().double(), b.cpu().double()
    L, R, K = a.shape
    M, N = x.shape[0], b.shape[1]
    s = torch.ones(L, dtype=torch.float64) if s is None else s.cpu().double()
    out, bound = torch.zeros(M, N, dtype=torch.float64), torch.zeros(M, N, dtype=torch.float64)
    own = owners(idx, M, L)
    for l in range(L):
        r = (own == l).nonzero().flatten()
        if not len(r):
            continue
        h, habs = s[l] * (x[r] @ a[l].T), s[l].abs() * (x[r].abs() @ a[l].abs().T)
        dh = (K + 4) * U * habs  # K products added in fp32, the scale multiplied in
        if half_h:  # one rounding to fp16, or to its subnormals
            dh = dh + half_step(torch.float16) * (h.abs() + dh) + 2.0 ** -25
        out[r] = h @ b[l].T
        bound[r] = dh @ b[l].abs().T + (R + 4) * U * (h.abs() @ b[l].abs().T)
    return out, bound


def lora_grads(x, dy, a, b, s, idx):
    """((dx, da, db), bounds): float64 gradients of the adapters' term.  The
    bounds count fp32 sums and h, g held as two fp16 terms relative to their
    largest magnitude in the adapter (2^-21 of it covers both terms' rounding);
    dx, an fp16 result, takes g rounded to one fp16 term (half a step of g, or of
    the smallest fp16 where the largest magnitude is scaled to 2^14 at least:
    2^-25 / 2^14 of it)."""
    x, dy, a, b = x.cpu().double(), dy.cpu().double(), a.cpu().double(), b.cpu().double()
    L, R, K = a.shape
    M, N = dy.shape
    s = torch.ones(L, dtype=torch.float64) if s is None else s.cpu().double()
    own = owners(idx, M, L)
    dx, da, db = torch.zeros(M, K).double(), torch.zeros(L, R, K).double(), torch.zeros(L, N, R).double()
    ex, ea, eb = torch.zeros_like(dx), torch.zeros_like(da), torch.zeros_like(db)
    for l in range(L):
        r = (own == l).nonzero().flatten()
        if not len(r):
            continue
        h, dh = s[l] * (x[r] @ a[l].T), (K + 4) * U * s[l].abs() * (x[r].abs() @ a[l].abs().T)
        g, dg = s[l] * (dy[r] @ b[l]), (N + 4) * U * s[l].abs() * (dy[r].abs() @ b[l].abs())
        dh, dg = dh + 2.0 ** -21 * h.abs().max(), dg + 2.0 ** -21 * g.abs().max()
        m = len(r) + 8
        dx[r] = g @ a[l]
        dgx = dg + half_step(torch.float16) * (g.abs() + dg) + 2.0 ** -39 * g.abs().max()
        ex[r] = dgx @ a[l].abs() + (R + 8) * U * (g.abs() @ a[l].abs())
        da[l] = g.T @ x[r]
        ea[l] = dg.T @ x[r].abs() + m * U * (g.abs().T @ x[r].abs())
        db[l] = dy[r].T @ h
        eb[l] = dy[r].abs().T @ dh + m * U * (dy[r].abs().T @ h.abs())
    ex = ex + half_step(torch.float16) * (dx.abs() + ex) + 2.0 ** -25
    return (dx, da, db), (ex, ea, eb)


def distill(z, idx, t, T, w):
    """((loss, dlogits), bounds) in float64.  Bounds: the fp32 exponentials and
    sums of V terms in partial sums of at most V/32 (relative 2^-23 each, and the
    rounding of arguments as large as their span), then the output's rounding."""
    dt = z.dtype
    z, t = z.cpu().double(), t.cpu().double()
    M, V = z.shape
    ids = idx.cpu().to(torch.int64) & 0xFFFFFFFF
    w = torch.ones(M, dtype=torch.float64) if w is None else w.cpu().double()
    loss, dz = torch.zeros(M).double(), torch.zeros(M, V).double()
    eloss, edz = torch.zeros(M).double(), torch.zeros(M, V).double()
    for m in range(M):
        ok = ids[m] < V
        tv, iv = t[m][ok] / T, ids[m][ok]
        if w[m] == 0 or not len(tv) or torch.isinf(tv).all():
            continue
        lp = tv - torch.logsumexp(tv, 0)
        p = lp.exp()
        zz = z[m] / T
        lse = torch.logsumexp(zz, 0)
        q = (zz - lse).exp() if torch.isfinite(lse) else torch.zeros(V).double()
        use = p > 0
        gap = lp[use] - (zz[iv[use]] - lse)
        gap = torch.where(torch.isinf(zz[iv[use]]), torch.full_like(gap, float("inf")), gap)
        loss[m] = w[m] * T * T * (p[use] * gap).sum()
        g = q.clone()
        g.index_add_(0, iv, -p)
        dz[m] = w[m] * T * g
        fin = zz[torch.isfinite(zz)]
        span = float((zz.max() - fin.min()) if len(fin) else 0) + float(tv.max() - tv[torch.isfinite(tv)].min())
        span = min(span, 110.0)  # beyond it an exponential is zero
        e = U * (V / 32 / 8 + 32 + 2 * span)  # sums: the terms of a partial sum round independently
        big = gap[torch.isfinite(gap)].abs().max() if torch.isfinite(gap).any() else 0.0
        eloss[m] = w[m].abs() * T * T * e * (2 * big + 1 + span) + 1e-30
        mass = q.clone()
        mass.index_add_(0, iv, p)
        edz[m] = w[m].abs() * T * e * mass
    edz = edz + half_step(dt) * (dz.abs() + edz) + torch.finfo(dt).tiny * torch.finfo(dt).eps
    return (loss, dz), (eloss, edz)


def close(got, want, bound, what):
    got = got.cpu().double()
    assert got.shape == want.shape, f"{what}: shape {got.shape} vs {want.shape}"
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin].nan_to_num(nan=7.0), want[~fin].nan_to_num(nan=7.0)), f"{what}: non-finite values"
    over = ((got - want).abs() - bound)[fin]
    assert len(over) == 0 or float(over.max()) <= 0, \
        f"{what}: {int((over > 0).sum())} of {len(over)} off, worst {float(over.max())} above its bound"
