"""What is measured of the adapter and distillation operators: low-rank
adapters of many requests beside a quantized projection (forward and
gradient) and distillation from a teacher's top logits.

Every case is one call as a user's program makes it.  ``run`` computes it with
elementary torch operations in float32, or, where ``own`` is true, through the
framework; ``exact`` is the same from the definitions in float64.
"""
import math

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    return [
        # decode of one request with its adapter: the o projection (6144 -> 5120) of a 27B layer, latency-bound
        dict(name="adapter decode 1 row", op="lora", rows=1, n=5120, k=6144, rank=16, adapters=8, bits=4, group=64,
             layout="mixed", none=0.0),
        # decode of 16 requests, each with an adapter of its own out of 32 resident ones: q|k|v (5120 -> 8192)
        dict(name="adapters decode 16 rows", op="lora", rows=16, n=8192, k=5120, rank=16, adapters=32, bits=4,
             group=64, layout="mixed", none=0.1),
        # a batch too large for the decode kernel, 8-bit override weights, odd row count, odd width, odd rank
        dict(name="adapters 37 rows odd", op="lora", rows=37, n=4099, k=2560, rank=12, adapters=6, bits=8, group=128,
             layout="mixed", none=0.25),
        # a prefill chunk of 2048 rows holding several requests' prompts: the gate projection (5120 -> 17408)
        dict(name="adapters prefill 2048", op="lora", rows=2048, n=17408, k=5120, rank=32, adapters=8, bits=4,
             group=64, layout="segments", none=0.1),
        # one adapter's training step on a short batch: the o projection
        dict(name="adapter grad 256 rows", op="lora_grad", rows=256, n=5120, k=6144, rank=16, adapters=1,
             layout="segments", none=0.0),
        # five adapters trained side by side, rows shuffled, odd width and rank
        dict(name="adapters grad 777 odd", op="lora_grad", rows=777, n=1003, k=1536, rank=20, adapters=5,
             layout="mixed", none=0.2),
        # a long batch over four high-rank adapters: the down projection (17408 -> 5120)
        dict(name="adapters grad 4096 rows", op="lora_grad", rows=4096, n=5120, k=17408, rank=64, adapters=4,
             layout="segments", none=0.05),
        # the positions of one draft block against 16 stored teacher logits each, full vocabulary
        dict(name="distill 4 positions", op="distill", rows=4, vocab=151936, top=16, dtype="float16", padded=0.0),
        # a ragged batch: padded positions, rows with fewer teacher logits, odd vocabulary, bf16
        dict(name="distill 333 odd bf16", op="distill", rows=333, vocab=32003, top=50, dtype="bfloat16", padded=0.3),
        # fp32 logits over a compact draft vocabulary
        dict(name="distill 128 fp32", op="distill", rows=128, vocab=80922, top=16, dtype="float32", padded=0.1),
        # a training batch of 2048 positions over the full vocabulary
        dict(name="distill 2048 rows", op="distill", rows=2048, vocab=151936, top=64, dtype="float16", padded=0.05),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lora", "lora", "lora_grad", "distill"])
    if op == "distill":
        rows, vocab = _log(rng, 1, 2048), _log(rng, 1000, 151936)
        dtype = rng.choice(["float16", "bfloat16", "float32"])
        if dtype == "float32":
            rows = min(rows, 1024)
        return dict(op=op, rows=rows, vocab=vocab, top=_log(rng, 1, 256), dtype=dtype,
                    padded=rng.choice([0.0, 0.1, 0.3]))
    rank = rng.choice([8, 16, 32, 64, _log(rng, 2, 64)])
    adapters = _log(rng, 1, 64)
    layout, none = rng.choice(["mixed", "segments"]), rng.choice([0.0, 0.1, 0.4])
    if op == "lora_grad":
        rows, n, k = _log(rng, 16, 4096), _log(rng, 256, 17408), 64 * _log(rng, 4, 272)
        while rows * (n + k) > 4096 * (5120 + 17408):
            rows //= 2
        return dict(op=op, rows=rows, n=n, k=k, rank=rank, adapters=min(adapters, 16), layout=layout, none=none)
    group = rng.choice([64, 64, 128])
    rows, n, k = _log(rng, 1, 2048), _log(rng, 256, 17408), 128 * _log(rng, 4, 136)
    while n * k > 17408 * 5120:
        n = n // 2 + 1
    return dict(op=op, rows=rows, n=n, k=k, rank=rank, adapters=adapters, bits=rng.choice([4, 4, 8]), group=group,
                layout=layout, none=none)


def _quantize(w, bits, group):
    """Affine codes of float32 w [N, K]: packed int32 words along K, fp16 scales and biases."""
    N, K = w.shape
    g = w.view(N, K // group, group)
    lo, hi = g.amin(-1), g.amax(-1)
    s = ((hi - lo) / (2 ** bits - 1)).clamp_min(1e-7).half()
    b = lo.half()
    q = ((g - b.float()[..., None]) / s.float()[..., None]).round_().clamp_(0, 2 ** bits - 1).to(torch.int32)
    q = q.view(N, K * bits // 32, 32 // bits)
    shifts = torch.arange(0, 32, bits, device=w.device, dtype=torch.int32)
    return (q << shifts).sum(-1, dtype=torch.int64).to(torch.int32), s, b


def _adapter_rows(case, gen, dev):
    """Adapter of each row, -1 for none: shuffled rows, or a few runs of rows as prompts lie in a batch."""
    M, L = case["rows"], case["adapters"]
    if case["layout"] == "mixed":
        idx = torch.randint(0, L, (M,), generator=gen, device=dev)
        off = torch.rand(M, generator=gen, device=dev) < case["none"]
    else:
        runs = min(M, 8)
        cuts = torch.randint(0, M, (runs,), generator=gen, device=dev).sort().values
        run = torch.searchsorted(cuts, torch.arange(M, device=dev), right=True)
        idx = torch.randint(0, L, (runs + 1,), generator=gen, device=dev)[run]
        off = (torch.rand(runs + 1, generator=gen, device=dev) < case["none"])[run]
    return torch.where(off, -1, idx).to(torch.int32)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    st = dict(case=case)
    if case["op"] == "distill":
        M, V, k, dt = case["rows"], case["vocab"], case["top"], DTYPES[case["dtype"]]
        # teacher and student agree up to noise; the teacher's top k of its own row
        base = rand(M, V).mul_(2.5)
        st["logits"] = (base + rand(M, V).mul_(0.7)).to(dt)
        vals, idx = base.topk(k, dim=-1)
        st["teacher_values"] = vals.to(dt)
        # rows stored with fewer candidates end in -1
        keep = torch.randint((k + 1) // 2, k + 1, (M, 1), generator=gen, device=dev)
        keep = torch.where(torch.rand(M, 1, generator=gen, device=dev) < case["padded"], keep, k)
        st["teacher_idx"] = torch.where(torch.arange(k, device=dev) < keep, idx, -1).to(torch.int32)
        # padded positions weigh nothing; the others carry the loss scale of an fp16 step
        w = torch.rand(M, generator=gen, device=dev) + 0.5
        st["row_weights"] = torch.where(torch.rand(M, generator=gen, device=dev) < case["padded"], 0.0, 256.0 * w)
        st["temperature"] = torch.tensor([2.0], device=dev)
        return st
    M, N, K, R, L = (case[n] for n in ("rows", "n", "k", "rank", "adapters"))
    st["x"] = rand(M, K).half()
    st["lora_a"] = (rand(L, R, K) * K ** -0.5).half()
    st["lora_b"] = (rand(L, N, R) * 0.05).half()
    st["lora_scales"] = torch.rand(L, generator=gen, device=dev) * 1.5 + 0.5
    st["adapter_idx"] = _adapter_rows(case, gen, dev)
    if case["op"] == "lora":
        st["w"], st["scales"], st["biases"] = _quantize(rand(N, K).mul_(0.02), case["bits"], case["group"])
    else:
        st["dy"] = (rand(M, N) * 0.1).half()
    return st


def _dequantize(st, bits, group, dtype):
    w = st["w"]
    shifts = torch.arange(0, 32, bits, device=w.device, dtype=torch.int32)
    q = (w[..., None] >> shifts) & (2 ** bits - 1)
    q = q.view(w.shape[0], -1, group).to(dtype)
    return (q * st["scales"].to(dtype)[..., None] + st["biases"].to(dtype)[..., None]).view(w.shape[0], -1)


def _own_columns(st):
    """[M, L] float32: the scale of each row's adapter in its column, zero elsewhere."""
    L = st["lora_a"].shape[0]
    mine = st["adapter_idx"].long()[:, None] == torch.arange(L, device=st["x"].device)
    return mine.float() * st["lora_scales"]


def _plain_lora(st, case):
    x = st["x"].float()
    y = x @ _dequantize(st, case["bits"], case["group"], torch.float32).T
    L, R, K = st["lora_a"].shape
    h = (x @ st["lora_a"].float().view(L * R, K).T).view(-1, L, R) * _own_columns(st)[..., None]
    y += h.view(-1, L * R) @ st["lora_b"].float().transpose(1, 2).reshape(L * R, -1)
    return y.half()


def _plain_lora_grad(st):
    x, dy = st["x"].float(), st["dy"].float()
    L, R, K = st["lora_a"].shape
    N = dy.shape[1]
    a = st["lora_a"].float().view(L * R, K)
    b = st["lora_b"].float().transpose(1, 2).reshape(L * R, N)
    s = _own_columns(st)[..., None]
    h = ((x @ a.T).view(-1, L, R) * s).view(-1, L * R)
    g = ((dy @ b.T).view(-1, L, R) * s).view(-1, L * R)
    da = (g.T @ x).view(L, R, K)
    db = (h.T @ dy).view(L, R, N).transpose(1, 2).contiguous()
    return (g @ a).half(), da, db


def _plain_distill(st):
    z, T, w = st["logits"].float(), st["temperature"], st["row_weights"]
    valid = st["teacher_idx"] >= 0
    idx = st["teacher_idx"].long().clamp_min(0)
    t = (st["teacher_values"].float() / T).masked_fill(~valid, -math.inf)
    t = t - t.amax(-1, keepdim=True)
    logp = t - t.exp().sum(-1, keepdim=True).log()
    p = logp.exp()
    z = z / T
    z = z - z.amax(-1, keepdim=True)
    e = z.exp()
    total = e.sum(-1, keepdim=True)
    gap = (logp - (z.gather(-1, idx) - total.log())).masked_fill(~valid, 0.0)
    loss = w * T * T * (p * gap).sum(-1)
    grad = (e / total).scatter_add_(-1, idx, -p) * (w * T)[:, None]
    return loss, grad.to(st["logits"].dtype)


def run(st):
    case = st["case"]
    if own:
        import qw_b200
        if case["op"] == "lora":
            return qw_b200.quantized_linear_lora(st["x"], st["w"], st["scales"], st["biases"], st["lora_a"],
                                                 st["lora_b"], st["lora_scales"], st["adapter_idx"],
                                                 group_size=case["group"], bits=case["bits"])
        if case["op"] == "lora_grad":
            return qw_b200.lora_backward(st["x"], st["dy"], st["lora_a"], st["lora_b"], st["lora_scales"],
                                         st["adapter_idx"])
        return qw_b200.topk_distillation(st["logits"], st["teacher_idx"], st["teacher_values"],
                                         temperature=st["temperature"], row_weights=st["row_weights"])
    if case["op"] == "lora":
        return _plain_lora(st, case)
    if case["op"] == "lora_grad":
        return _plain_lora_grad(st)
    return _plain_distill(st)


def work(case):
    M = case["rows"]
    if case["op"] == "distill":
        V, k, sz = case["vocab"], case["top"], 4 if case["dtype"] == "float32" else 2
        return {"bytes": 2 * M * V * sz + M * k * (4 + sz) + 8 * M, "flops": 8 * M * V}
    N, K, R = case["n"], case["k"], case["rank"]
    used = min(case["adapters"], M if case["layout"] == "mixed" else 9)
    if case["op"] == "lora":
        weights = N * K * case["bits"] // 8 + 4 * N * (K // case["group"])
        return {"bytes": weights + 2 * M * (K + N) + 2 * used * R * (K + N) + 4 * M,
                "flops": 2 * M * N * K + 2 * M * R * (K + N)}
    return {"bytes": 2 * M * (2 * K + N) + 2 * used * R * (K + N) + 4 * case["adapters"] * R * (K + N) + 4 * M,
            "flops": 2 * M * R * (3 * K + 2 * N)}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "distill":
        M = case["rows"]
        T, losses, grads = float(st["temperature"]), [], []
        for m0 in range(0, M, 128):  # rows in blocks: float64 logits of a whole batch are large
            z = st["logits"][m0:m0 + 128].double() / T
            ids = st["teacher_idx"][m0:m0 + 128].long()
            t = st["teacher_values"][m0:m0 + 128].double() / T
            ok = ids >= 0
            t = torch.where(ok, t, torch.full_like(t, -math.inf))
            lp = torch.log_softmax(t, -1)
            lq = torch.log_softmax(z, -1)
            p = lp.exp()
            at = ids.clamp(min=0)
            terms = torch.where(ok, p * (lp - torch.gather(lq, 1, at)), torch.zeros_like(p))
            w = st["row_weights"][m0:m0 + 128].double()
            losses.append(T * T * w * terms.sum(1))
            target = torch.zeros_like(z).scatter_add_(1, at, p)
            grads.append((T * w[:, None] * (lq.exp() - target)).to(torch.float64))
        return torch.cat(losses), torch.cat(grads)
    x = st["x"].double()
    rows = [(st["adapter_idx"] == l).nonzero().flatten() for l in range(case["adapters"])]
    s = st["lora_scales"].double().tolist()
    if case["op"] == "lora":
        y = x @ _dequantize(st, case["bits"], case["group"], torch.float64).T
        for l, r in enumerate(rows):
            y[r] += s[l] * ((x[r] @ st["lora_a"][l].double().T) @ st["lora_b"][l].double().T)
        return y
    dy = st["dy"].double()
    dx, da, db = torch.zeros_like(x), [], []
    for l, r in enumerate(rows):
        a, b = st["lora_a"][l].double(), st["lora_b"][l].double()
        g = s[l] * (dy[r] @ b)
        dx[r] = g @ a
        da.append(g.T @ x[r])
        db.append(s[l] * (dy[r].T @ (x[r] @ a.T)))
    return dx, torch.stack(da), torch.stack(db)
