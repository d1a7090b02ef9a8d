"""The operators of the catalogue head, with the sizes they are measured at.

A trained network answers with a distribution over the item catalogue.  Four operators stand on that path:

  norm      root-mean-square norm of hidden rows with the residual's addition, written as 8-bit codes with one scale a row
  product   codes of the user rows times codes of the item rows, with a scale for each row of either side
  sample    one item a row from its scores: temperature, top-k, top-p and min-p, from given random numbers
  distill   the loss that fits a student's scores to a teacher's top scores, with its gradient

`run` computes a case in its plain form, or through the framework's operators where `own` is true.
"""
import math

import numpy as np
import torch

own = False

# ---- the cases --------------------------------------------------------------------------------------------------------
# 10677 items and 69878 users are the MovieLens-10M graph of the benchmark, 3706 and 1682 the items of MovieLens-1M and
# -100K, 10^6 the items of the benchmark's large graph; 256 is the benchmark's width, 250 and 75 the widths of the network's
# layers, 10000 the training example's batch.  The other sizes are generic.


def listed():
    return [
        # one user's hidden row enters the head: nothing but latency
        dict(name="norm one row", op="norm", rows=1, dim=250, dtype="float32", residual=True),
        # all users of the MovieLens-10M graph, once per refresh of the served rows
        dict(name="norm all users", op="norm", rows=69878, dim=256, dtype="float32", residual=True),
        # a wide hidden layer in 16 bits
        dict(name="norm wide bf16", op="norm", rows=8192, dim=4096, dtype="bfloat16", residual=True),
        # one user against the catalogue
        dict(name="product one user", op="product", m=1, n=10677, k=256, out="float32", bias=True),
        # a batch of users against the catalogue, at the layers' odd width
        dict(name="product batch", op="product", m=10000, n=10677, k=250, out="float32", bias=True),
        # a large dense layer, where the matrix units count
        dict(name="product large bf16", op="product", m=8192, n=8192, k=4096, out="bfloat16", bias=False),
        # one request, nucleus sampling over the catalogue
        dict(name="sample one row", op="sample", rows=1, items=10677, dtype="float32", temperature=0.8, top_k=0, top_p=0.9,
             min_p=0.0, per_row=False),
        # a batch of requests, each with its own settings
        dict(name="sample batch", op="sample", rows=512, items=10677, dtype="bfloat16", temperature=1.0, top_k=100, top_p=0.95,
             min_p=0.01, per_row=True),
        # the large catalogue
        dict(name="sample large catalogue", op="sample", rows=64, items=1000000, dtype="float32", temperature=1.0, top_k=0,
             top_p=0.95, min_p=0.0, per_row=False),
        # a small training step: forward and backward
        dict(name="distill small", op="distill", rows=33, items=1682, k=10, dtype="float32", temperature=2.0),
        # the training example's batch over the MovieLens-10M items
        dict(name="distill batch bf16", op="distill", rows=10000, items=10677, k=64, dtype="bfloat16", temperature=2.0),
        # the large catalogue, few rows
        dict(name="distill large catalogue", op="distill", rows=64, items=1000000, k=128, dtype="float32", temperature=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "product", "sample", "distill"))
    dtype = rng.choice(("float32", "bfloat16", "float16"))
    if op == "norm":
        dim = _log(rng, 16, 8192)
        return dict(op=op, rows=_log(rng, 1, min(69878, 8192 * 4096 // dim)), dim=dim, dtype=dtype,
                    residual=rng.random() < 0.7)
    if op == "product":
        k, n = _log(rng, 16, 4096), _log(rng, 16, 16384)
        return dict(op=op, m=_log(rng, 1, min(10000, 10677 * 10000 // n)), n=n, k=k, out=dtype, bias=rng.random() < 0.5)
    items = _log(rng, 50, 1000000)
    if op == "sample":
        return dict(op=op, rows=_log(rng, 1, min(2048, 64 * 1000000 // items)), items=items, dtype=dtype,
                    temperature=round(rng.uniform(0.5, 1.5), 2), top_k=rng.choice((0, 0, _log(rng, 1, 2000))),
                    top_p=rng.choice((1.0, round(rng.uniform(0.5, 0.99), 3))),
                    min_p=rng.choice((0.0, round(rng.uniform(0.001, 0.2), 4))), per_row=rng.random() < 0.5)
    return dict(op=op, rows=_log(rng, 1, min(10000, 64 * 1000000 // items)), items=items,
                k=_log(rng, 1, min(items, 200)), dtype=dtype, temperature=round(rng.uniform(0.5, 4.0), 2))


# ---- the inputs -------------------------------------------------------------------------------------------------------


def _quantised(x):
    scale = (x.abs().amax(1) / 127.0).contiguous()
    return torch.round(x / scale[:, None]).to(torch.int8), scale


def _scores(rows, items, gen, dev):
    """Scores of a catalogue: each item's popularity (long-tailed), each row's taste, and 2 % of the items masked out because
    the row has had them already."""
    pop = torch.rand(items, generator=gen, device=dev).clamp_min_(1e-6).log_().neg_().mul_(1.5)
    s = torch.randn(rows, items, generator=gen, device=dev)
    s.mul_(1.7).add_(pop)
    masked = torch.rand(rows, items, generator=gen, device=dev) < 0.02
    masked[:, 0] = False
    return s, masked


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    st = dict(case)
    op = case["op"]
    if op == "norm":
        dt = getattr(torch, case["dtype"])
        rows, dim = case["rows"], case["dim"]
        st["x"] = torch.randn(rows, dim, generator=gen, device=dev).to(dt)
        st["weight"] = (1.0 + 0.2 * torch.randn(dim, generator=gen, device=dev)).to(dt)
        st["res"] = (2.0 * torch.randn(rows, dim, generator=gen, device=dev)).to(dt) if case["residual"] else None
        st["eps"] = 1e-6
    elif op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        st["a"], st["sa"] = _quantised(torch.randn(m, k, generator=gen, device=dev))
        st["b"], st["sb"] = _quantised(torch.randn(n, k, generator=gen, device=dev) * k ** -0.5)
        st["bias_t"] = torch.randn(n, generator=gen, device=dev) if case["bias"] else None
    elif op == "sample":
        rows, items = case["rows"], case["items"]
        s, masked = _scores(rows, items, gen, dev)
        st["logits"] = s.masked_fill_(masked, -math.inf).to(getattr(torch, case["dtype"]))
        st["u"] = torch.rand(rows, generator=gen, device=dev)
        if case["per_row"]:
            r = torch.rand(4, rows, generator=gen, device=dev)
            st["temperature"] = case["temperature"] * (0.75 + 0.5 * r[0])
            k = (case["top_k"] * (0.5 + r[1])).to(torch.int32)
            st["top_k"] = torch.where(r[1] < 0.25, torch.zeros_like(k), k)            # some rows without it
            st["top_p"] = torch.where(r[2] < 0.25, torch.ones_like(r[2]), case["top_p"] - 0.1 * r[2])
            st["min_p"] = case["min_p"] * r[3]
    else:
        rows, items, k, dt = case["rows"], case["items"], case["k"], getattr(torch, case["dtype"])
        s, masked = _scores(rows, items, gen, dev)
        t = s + 0.7 * torch.randn(rows, items, generator=gen, device=dev)
        val, idx = t.masked_fill_(masked, -math.inf).topk(k, dim=1)
        st["student"] = s.to(dt)
        st["teacher"], st["index"] = val.contiguous(), idx.to(torch.int32)
        st["scale"] = 1.0 / rows
    return st


# ---- one pass ---------------------------------------------------------------------------------------------------------


def _norm(st):
    h = st["x"] if st["res"] is None else (st["x"].float() + st["res"].float()).to(st["x"].dtype)
    # a code is a decision at the border between two whole numbers: 64 bits up to it
    hd = h.double()
    y = hd * torch.rsqrt(hd.square().mean(1, keepdim=True) + st["eps"]) * st["weight"].double()
    scale = (y.abs().amax(1) / 127.0).float()
    codes = torch.round(y / scale.double()[:, None]).clamp(-127, 127).to(torch.int8)
    return codes, scale, h


def _product(st):
    # whole numbers: a 32-bit sum of at most 1024 products of codes is exact
    acc = 0.0
    for lo in range(0, st["k"], 1024):
        acc = acc + st["a"][:, lo:lo + 1024].float() @ st["b"][:, lo:lo + 1024].float().t()
    out = acc * st["sa"][:, None] * st["sb"]
    if st["bias_t"] is not None:
        out = out + st["bias_t"]
    return out.to(getattr(torch, st["out"]))


def _column(v, rows, dtype, dev):
    return v.to(dtype).view(-1, 1) if torch.is_tensor(v) else torch.full((rows, 1), v, dtype=dtype, device=dev)


def _sample(st):
    # 64 bits: which item is drawn is a decision at the border of two sums over the catalogue
    z, rows, n, dev = st["logits"].double(), st["rows"], st["items"], st["logits"].device
    temp, p, m = (_column(st[name], rows, torch.float64, dev) for name in ("temperature", "top_p", "min_p"))
    w = torch.exp((z - z.amax(1, keepdim=True)) / temp)
    if st["per_row"] or st["top_k"] > 0 or st["top_p"] < 1.0 or st["min_p"] > 0.0:
        k = _column(st["top_k"], rows, torch.int64, dev)
        k = torch.where(k <= 0, n, k.clamp(max=n))
        order = torch.sort(z, dim=1, descending=True, stable=True).indices
        ws = w.gather(1, order)
        c = ws.cumsum(1)
        before = torch.cat([torch.zeros_like(c[:, :1]), c[:, :-1]], 1)
        keep = torch.arange(n, device=dev) < k
        keep &= (before < p * c.gather(1, k - 1)) | (p >= 1.0)
        keep &= ws >= m
        keep[:, 0] = True
        w = torch.zeros_like(w).scatter_(1, order, ws * keep)
    c = w.cumsum(1)
    ids = (c <= st["u"].double()[:, None] * c[:, -1:]).sum(1)
    return ids.to(torch.int32), (w.gather(1, ids[:, None]) / c[:, -1:]).squeeze(1).float()


def _distill(st):
    t, scale = st["temperature"], st["scale"]
    z = st["student"].float() / t
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    a = st["teacher"].float() / t
    a = a - a.amax(1, keepdim=True)
    ea = torch.exp(a)
    p = ea / ea.sum(1, keepdim=True)
    idx = st["index"].long()
    log_q = z.gather(1, idx) - torch.log(total)
    row = (p * (a - torch.log(ea.sum(1, keepdim=True)) - log_q)).sum(1)
    loss = scale * t * t * row.sum()
    grad = e / total
    grad.scatter_add_(1, idx, -p)
    return loss, (grad * (scale * t)).to(st["student"].dtype)


def run(st):
    op = st["op"]
    if not own:
        return {"norm": _norm, "product": _product, "sample": _sample, "distill": _distill}[op](st)
    from star_gcn_amd import functional, ops
    if op == "norm":
        return ops.rms_norm_i8(st["x"], st["weight"], residual=st["res"], eps=st["eps"])
    if op == "product":
        return ops.gemm_i8(st["a"], st["sa"], st["b"], st["sb"], bias=st["bias_t"], out_dtype=getattr(torch, st["out"]))
    if op == "sample":
        return ops.sample_rows(st["logits"], st["u"], temperature=st["temperature"], top_k=st["top_k"], top_p=st["top_p"],
                               min_p=st["min_p"])
    student = st["student"].detach().requires_grad_(True)
    loss = functional.distill_loss(student, st["teacher"], st["index"], st["scale"], temperature=st["temperature"])
    grad, = torch.autograd.grad(loss, student)
    return loss.detach(), grad


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

_BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}


def work(case):
    op = case["op"]
    if op == "norm":
        n, s = case["rows"] * case["dim"], _BYTES[case["dtype"]]
        # the rows (and the residual) in, the codes and the sum out; without a residual the sum is the input itself
        return {"bytes": n * (s * (3 if case["residual"] else 1) + 1) + case["dim"] * s + 4 * case["rows"], "flops": 8 * n}
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * (k + 4) + m * n * _BYTES[case["out"]] + 4 * n * case["bias"], "flops": 2 * m * n * k}
    n, s = case["rows"] * case["items"], _BYTES[case["dtype"]]
    if op == "sample":
        return {"bytes": n * s + case["rows"] * (12 + 16 * case["per_row"]), "flops": 12 * n}
    # forward reads the scores; backward, a separate pass after it, reads them again and writes the gradient
    return {"bytes": 3 * n * s + 2 * case["rows"] * case["k"] * 8, "flops": 10 * n}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    return {"norm": _exact_norm, "product": _exact_product, "sample": _exact_sample, "distill": _exact_distill}[case["op"]](st)


def _exact_norm(st):
    x = st["x"]
    if st["res"] is not None:
        x = (x.double() + st["res"].double()).to(x.dtype)      # one rounding to the stored type; what follows reads that
    v = x.double()
    r = 1.0 / torch.sqrt((v * v).sum(1) / v.shape[1] + st["eps"])
    y = torch.einsum("i,ij,j->ij", r, v, st["weight"].double())
    scale = torch.maximum(y.amax(1), -y.amin(1)).div(127.0).float()
    q = (y / scale.double().unsqueeze(1)).round()
    return q.clamp_(-127.0, 127.0).to(torch.int8), scale, x


def _exact_product(st):
    out = torch.mm(st["a"].double(), st["b"].double().t().contiguous())
    out *= torch.outer(st["sa"].double(), st["sb"].double())
    return out if st["bias_t"] is None else out + st["bias_t"].double()


def _exact_sample(st):
    z = st["logits"].double().cpu().numpy()
    u = st["u"].double().cpu().numpy()
    rows, n = z.shape

    def of(name, i):
        v = st[name]
        return v[i].item() if torch.is_tensor(v) else v

    ids, prob = np.empty(rows, np.int32), np.empty(rows, np.float64)
    par = {k: (st[k].cpu() if torch.is_tensor(st[k]) else st[k]) for k in ("temperature", "top_k", "top_p", "min_p")}
    st = dict(st, **par)
    for i in range(rows):
        row = z[i]
        w = np.exp((row - row.max()) / of("temperature", i))
        rank = np.argsort(-row, kind="stable")
        k = int(of("top_k", i))
        rank = rank[:k] if 0 < k < n else rank
        mass = np.cumsum(w[rank])
        p = of("top_p", i)
        if p < 1.0:      # the shortest prefix that holds at least the share p
            rank = rank[:int(np.searchsorted(mass, p * mass[-1], side="left")) + 1]
        rank = rank[w[rank] >= of("min_p", i)] if of("min_p", i) <= 1.0 else rank[:1]
        rank = np.sort(rank)
        c = np.cumsum(w[rank])
        at = min(int(np.searchsorted(c, u[i] * c[-1], side="right")), rank.size - 1)
        ids[i], prob[i] = rank[at], w[rank[at]] / c[-1]
    return torch.from_numpy(ids), torch.from_numpy(prob)


def _exact_distill(st):
    t, scale = st["temperature"], st["scale"]
    log_q = torch.log_softmax(st["student"].double() / t, 1)
    log_p = torch.log_softmax(st["teacher"].double() / t, 1)
    idx, p = st["index"].long(), log_p.exp()
    loss = scale * t * t * (p * (log_p - log_q.gather(1, idx))).sum()
    grad = log_q.exp_()
    grad.scatter_(1, idx, grad.gather(1, idx) - p)             # the teacher's top items are distinct
    return loss, grad.mul_(scale * t)
