"""The vocabulary-end operators as they are measured: rules on logits, choosing a token, distillation from a teacher's
top logits, and the scaled token lookup with its gradient.

Each case is one call of one operator.  `run` computes it in elementary torch operations in 32 bits (own = False), or
through the package's entry points (own = True).  `exact` gives the same outputs from the definitions in 64 bits.

Definitions
  rules    x = float(logit); a token that occurs in history[:len] has x / r where x > 0 and x * r elsewhere; a token
           that occurs g times in history[prompt:len] has x - f * g, and x - p where g > 0; then the sum of its bias
           entries is added; a token whose mask bit is 0 becomes -inf.
  choice   with m the row's largest x: t = (x - m) / T, and the token's mass is exp(t) held as a whole number of
           2^-40.  In the order (x descending, index ascending) the first top_k tokens are kept, of those the ones
           whose preceding mass is below top_p of the mass kept so far; the token is the first one, in index order,
           whose running kept mass exceeds u times the kept mass.  T = 0 takes the largest x.  A row whose mask leaves
           nothing has the token -1.
  distill  q = softmax(s / T), p = softmax over the row's teacher entries at T (or exp(t / T - lse) where the teacher's
           log-sum-exp is given, the rest of its mass being one more event); the loss of a row is
           w * (alpha * T^2 * KL(p | q) + (1 - alpha) * cross-entropy of the target), its gradient by s beside it.
  lookup   out = scale * table[id]; gradient: table row v gets scale * the sum of dout over the positions of v.
"""
import math

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
UNIT = float(2 ** 40)  # masses are whole numbers of 2^-40 of the largest token's


def listed():
    return [
        # one chat stream: a short history, a few biases, a grammar's mask: latency
        dict(name="rules-1", op="rules", S=1, V=32768, dt="f32", hist=40, bias=4, mask=True),
        # the decode batch of the benchmark, 256 streams after 2,048 tokens
        dict(name="rules-256", op="rules", S=256, V=32768, dt="bf16", hist=2048, bias=16, mask=True),
        # one stream that takes the likeliest token under a repetition penalty: latency
        dict(name="choose-1", op="choose", S=1, V=32768, dt="bf16", hist=100, bias=0, mask=False, temp=0.0, top_k=0,
             top_p=1.0),
        # the decode batch sampled with top-k and top-p, some streams under a grammar
        dict(name="choose-256", op="choose", S=256, V=32768, dt="bf16", hist=512, bias=8, mask=True, temp=0.8,
             top_k=50, top_p=0.95),
        # a ragged batch over an odd vocabulary, nucleus sampling after long texts
        dict(name="choose-nucleus-33", op="choose", S=33, V=50021, dt="f32", hist=4096, bias=0, mask=False, temp=1.0,
             top_k=0, top_p=0.9),
        # a toy student's step in float32
        dict(name="distill-48", op="distill", N=48, V=1000, dt="f32", k=8, temp=1.0, alpha=0.5, hard=True, tail=False,
             grad=True),
        # a training step of 8 rows x 2,048 tokens: loss and gradient, soft and hard targets mixed
        dict(name="distill-16384", op="distill", N=16384, V=32768, dt="bf16", k=64, temp=2.0, alpha=0.7, hard=True,
             tail=False, grad=True),
        # held-out loss over an odd vocabulary, the teacher's remaining mass counted
        dict(name="distill-eval-8192", op="distill", N=8192, V=50021, dt="bf16", k=32, temp=1.0, alpha=1.0, hard=False,
             tail=True, grad=False),
        # the lookup of one decode step
        dict(name="lookup-256", op="lookup", N=256, V=32768, d=768, dt="bf16"),
        # the lookup of the benchmark's 32 x 2,048 prompt tokens
        dict(name="lookup-65536", op="lookup", N=65536, V=32768, d=768, dt="bf16"),
        # the table's gradient over the same tokens, into a float32 master gradient
        dict(name="table-grad-65536", op="table_grad", N=65536, V=32768, d=768, dt="bf16", gdt="f32"),
        # a small odd model's table gradient
        dict(name="table-grad-5000", op="table_grad", N=5000, V=50021, d=330, dt="f32", gdt="f32"),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rules", "choose", "distill", "lookup", "table_grad"])
    dt = rng.choice(["f32", "bf16"])
    V = rng.choice([32768, _spread(rng, 500, 131072)])
    if op in ("rules", "choose"):
        S = _spread(rng, 1, max(1, min(512, 256 * 32768 // V)))
        c = dict(op=op, S=S, V=V, dt=dt, hist=_spread(rng, 1, 4096), bias=rng.choice([0, _spread(rng, 1, 64)]),
                 mask=rng.random() < 0.5)
        if op == "choose":
            c.update(temp=rng.choice([0.0, round(rng.uniform(0.4, 1.5), 2)]),
                     top_k=rng.choice([0, _spread(rng, 1, 1000)]), top_p=rng.choice([1.0, round(rng.uniform(0.5, 0.99), 3)]))
        return c
    if op == "distill":
        return dict(op=op, N=_spread(rng, 16, max(16, min(16384, 16384 * 32768 // V))), V=V, dt=dt,
                    k=_spread(rng, 1, 128), temp=rng.choice([1.0, round(rng.uniform(0.7, 4.0), 2)]),
                    alpha=round(rng.uniform(0.1, 1.0), 2), hard=rng.random() < 0.5, tail=rng.random() < 0.5,
                    grad=rng.random() < 0.7)
    d = rng.choice([768, 1536, _spread(rng, 33, 1536)])
    c = dict(op=op, N=_spread(rng, 1, min(65536, 65536 * 768 // d)), V=V if op == "lookup" else min(V, 65536), d=d, dt=dt)
    if op == "table_grad":
        c["gdt"] = rng.choice(["f32", dt])
    return c


def _zipf_cdf(V, device):
    w = torch.arange(1, V + 1, device=device, dtype=torch.float64) ** -1.1
    return torch.cumsum(w / w.sum(), 0)


def _zipf(shape, V, g):
    u = torch.rand(shape, generator=g, device="cuda", dtype=torch.float64)
    return torch.searchsorted(_zipf_cdf(V, "cuda"), u).clamp_(max=V - 1).to(torch.int32)


def _logits(N, V, dt, g):
    """Logits of a language model: a bell of width 2.5 whose centre falls with the token's rank."""
    x = torch.randn(N, V, generator=g, device="cuda", dtype=dt if N * V > 1 << 25 else torch.float32)
    x.mul_(2.5).sub_((0.3 * torch.log(torch.arange(1, V + 1, device="cuda"))).to(x.dtype))
    return x.to(dt)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, V, dt = case["op"], case["V"], DT[case["dt"]]

    def uniform(n, lo, hi):
        return lo + (hi - lo) * torch.rand(n, generator=g, device="cuda")

    def whole(shape, lo, hi):
        return torch.randint(lo, hi, shape if isinstance(shape, tuple) else (shape,), generator=g, device="cuda",
                             dtype=torch.int32)

    if op in ("rules", "choose"):
        S, L = case["S"], case["hist"]
        st = {"case": case, "logits": _logits(S, V, dt, g), "history": _zipf((S, L), V, g),
              "history_len": whole(S, (L + 1) // 2, L + 1), "repetition": uniform(S, 1.0, 1.4),
              "frequency": uniform(S, 0.0, 0.5), "presence": uniform(S, 0.0, 0.5)}
        st["prompt_len"] = st["history_len"] // 2
        st["history"].masked_fill_(torch.arange(L, device="cuda") >= st["history_len"][:, None], -1)
        if case["bias"]:
            st["bias_ids"] = whole((S, case["bias"]), 0, V)
            st["bias_values"] = uniform((S, case["bias"]), -4.0, 4.0)
        if case["mask"]:
            # grammar states shared by the streams: one of digits (a few tokens), one of most tokens, one finished
            # (nothing is allowed), some half open; -1 for a stream without a grammar
            W = -(-V // 32)
            st["mask"] = whole((8, W), -2 ** 31, 2 ** 31 - 1)
            st["mask"][0] = 0
            st["mask"][0, : max(1, W // 64)] = -1
            st["mask"][1] |= whole(W, -2 ** 31, 2 ** 31 - 1) | whole(W, -2 ** 31, 2 ** 31 - 1)
            st["mask"][7] = 0
            st["mask_row"] = whole(S, -2, 7).clamp_(min=-1)
            if S >= 8:
                st["mask_row"][S // 2] = 7
        if op == "choose":
            T = case["temp"]
            st["temperature"] = torch.full((S,), T, device="cuda") * uniform(S, 0.9, 1.1)
            st["top_k"] = torch.full((S,), case["top_k"], dtype=torch.int32, device="cuda")
            st["top_p"] = torch.full((S,), case["top_p"], device="cuda")
            if S >= 16 and T > 0:
                st["temperature"][::16] = 0.0  # a few streams of the batch are greedy
            st["u"] = torch.rand(S, generator=g, device="cuda")
        return st
    if op == "distill":
        N, k = case["N"], min(case["k"], V // 4)
        st = {"case": case, "logits": _logits(N, V, dt, g)}
        # distinct ids in every row: an arithmetic progression modulo V
        step = whole((N, 1), 1, V // k)
        ids = (whole((N, 1), 0, V) + step * torch.arange(k, device="cuda", dtype=torch.int32)) % V
        tl = 2.0 * torch.randn(N, k, generator=g, device="cuda").sort(1, descending=True).values + 4.0
        ragged = torch.arange(k, device="cuda") >= whole((N, 1), (k + 1) // 2, 4 * k + 1)  # some rows have fewer entries
        st["teacher_ids"] = ids.masked_fill(ragged, -1).contiguous()
        st["teacher_logits"] = tl.contiguous()
        if case["tail"]:
            z = (tl / case["temp"]).masked_fill(ragged, -math.inf)
            st["teacher_lse"] = torch.logsumexp(z, 1) + uniform(N, 0.02, 0.7)
        st["targets"] = None
        if case["hard"]:
            st["targets"] = _zipf(N, V, g).masked_fill_(torch.rand(N, generator=g, device="cuda") < 0.03, -1)
        st["row_weight"] = (torch.rand(N, generator=g, device="cuda") > 0.05).float()
        return st
    N, d = case["N"], case["d"]
    st = {"case": case, "ids": _zipf(N, V, g), "scale": math.sqrt(d)}
    if op == "lookup":
        st["table"] = (0.02 * torch.randn(V, d, generator=g, device="cuda")).to(dt)
    else:
        st["dout"] = torch.randn(N, d, generator=g, device="cuda").to(dt)
    return st


RULES = ("history", "history_len", "prompt_len", "repetition", "frequency", "presence", "bias_ids", "bias_values",
         "mask", "mask_row")


def _ruled(st, x):
    """The rules on x (S, V), in x's type: the plain form."""
    S, V = x.shape
    L = st["history"].shape[1]
    at = torch.arange(L, device=x.device)
    seen = (at < st["history_len"][:, None]) & (st["history"] >= 0)
    tok = torch.where(seen, st["history"], V).long()
    new = torch.where(seen & (at >= st["prompt_len"][:, None]), st["history"], V).long()
    one = torch.ones_like(tok, dtype=torch.int32)
    c = torch.zeros(S, V + 1, dtype=torch.int32, device=x.device).scatter_add_(1, tok, one)[:, :V]
    n = torch.zeros(S, V + 1, dtype=torch.int32, device=x.device).scatter_add_(1, new, one)[:, :V]
    r = st["repetition"][:, None].to(x.dtype)
    x = torch.where(c > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - st["frequency"][:, None].to(x.dtype) * n
    x = torch.where(n > 0, x - st["presence"][:, None].to(x.dtype), x)
    if "bias_ids" in st:
        b = torch.zeros(S, V, dtype=x.dtype, device=x.device)
        x = x + b.scatter_add_(1, st["bias_ids"].long(), st["bias_values"].to(x.dtype))
    if "mask" in st:
        v = torch.arange(V, device=x.device)
        bits = (st["mask"][:, v // 32] >> (v % 32).to(torch.int32)) & 1
        row = st["mask_row"].long()
        allowed = (bits[row.clamp(min=0)] == 1) | (row < 0)[:, None]
        x = x.masked_fill(~allowed, -math.inf)
    return x


def _choose(st):
    y = _ruled(st, st["logits"].float())
    S, V = y.shape
    m = y.amax(1, keepdim=True)
    T = st["temperature"][:, None]
    greedy = T == 0
    t = torch.where(y == m, torch.zeros_like(y), (y - m) / torch.where(greedy, torch.ones_like(T), T))
    w = torch.round(torch.exp(t) * UNIT).to(torch.int64)
    ys, order = torch.sort(y, dim=1, descending=True, stable=True)
    ws = w.gather(1, order)
    k = st["top_k"][:, None].long()
    rank = torch.arange(V, device=y.device)
    ws = torch.where((rank < k) | (k <= 0) | greedy, ws, 0)
    before = torch.cumsum(ws, 1) - ws
    W = ws.sum(1, keepdim=True)
    cut = torch.ceil(st["top_p"][:, None].double() * W.double()).to(torch.int64).clamp(min=1)
    cut = torch.where((st["top_p"][:, None] >= 1) | greedy, W, cut)
    ws = torch.where(before < cut, ws, 0)
    kept = torch.zeros_like(w).scatter_(1, order, ws)
    K = kept.sum(1, keepdim=True)
    r = torch.minimum(torch.floor(st["u"][:, None].double() * K.double()).to(torch.int64), K - 1)
    ids = (torch.cumsum(kept, 1) <= r).sum(1, keepdim=True)
    ids = torch.where(greedy, order[:, :1], ids)
    lp = t.gather(1, ids) - torch.log(K.float() / UNIT)
    none = m == -math.inf
    return torch.where(none, -1, ids)[:, 0].to(torch.int32), torch.where(none, m, lp)[:, 0]


def _distill(st):
    c = st["case"]
    T, a, tail = c["temp"], c["alpha"], "teacher_lse" in st
    s = st["logits"].float()
    ids, w = st["teacher_ids"], st["row_weight"]
    ok = (ids >= 0) & (st["teacher_logits"] > -math.inf)
    at = ids.clamp(min=0).long()
    z = (st["teacher_logits"] / T).masked_fill(~ok, -math.inf)
    if tail:
        logp = z - st["teacher_lse"][:, None]
    else:
        mz = z.amax(1, keepdim=True)
        logp = z - (mz + torch.log(torch.exp(z - mz).sum(1, keepdim=True)))
    p = torch.where(ok, torch.exp(logp), 0.0)
    some = ok.any(1)
    zs = s / T
    m = zs.amax(1, keepdim=True)
    e = torch.exp(zs - m)
    tot = e.sum(1, keepdim=True)
    logq = zs.gather(1, at) - m - torch.log(tot)
    soft = torch.where(ok & (p > 0), p * (logp - logq), 0.0).sum(1)
    if tail:
        rest = e.scatter(1, torch.where(ok, at, at[:, :1]), 0.0)  # the listed tokens' terms taken out
        qr = rest.sum(1) / tot[:, 0]
        pr = (1.0 - p.sum(1)).clamp(min=0.0)
        soft = soft + torch.where(some & (pr > 0), pr * (torch.log(pr) - torch.log(qr)), 0.0)
    soft = torch.where(some, soft, 0.0) * (T * T)
    loss = a * soft
    tgt = st["targets"]
    if tgt is not None:
        hit = tgt >= 0
        th = tgt.clamp(min=0).long()[:, None]
        m1 = s.amax(1, keepdim=True)
        e1 = torch.exp(s - m1)
        tot1 = e1.sum(1, keepdim=True)
        loss = loss + (1 - a) * torch.where(hit, (m1 + torch.log(tot1) - s.gather(1, th))[:, 0], 0.0)
    loss = torch.where(w > 0, w * loss, 0.0)
    if not c["grad"]:
        return {"loss": loss}
    mass = p.sum(1) + pr if tail else some.float()  # the teacher's whole mass: 1, or 0 where the row has no entry
    grad = e.mul_(a * T / tot) * (some * mass)[:, None]
    if tail:
        f = torch.where(pr > 0, 1.0 - pr / (qr * mass), 1.0)[:, None]
        took = torch.zeros_like(grad).scatter_(1, torch.where(ok, at, at[:, :1]), 1.0)
        grad = torch.where(took > 0, grad, grad * f)
    grad.scatter_add_(1, at, -(a * T) * p)
    if tgt is not None:
        e1.mul_((1 - a) / tot1 * hit.float()[:, None])
        grad = grad + e1
        grad.scatter_add_(1, th, -(1 - a) * hit.float()[:, None])
    return {"loss": loss, "dlogits": grad.mul_(w[:, None]).to(st["logits"].dtype)}


def run(state):
    c = state["case"]
    if own:
        import sdmchat_b200 as S
        if c["op"] in ("rules", "choose"):
            rules = S.LogitRules(**{n: state[n] for n in RULES if n in state})
            if c["op"] == "rules":
                return S.process_logits(state["logits"], rules)
            return S.sample_logits(state["logits"], rules, u=state["u"], temperature=state["temperature"],
                                   top_k=state["top_k"], top_p=state["top_p"])
        if c["op"] == "distill":
            args = dict(targets=state["targets"], temperature=c["temp"], alpha=c["alpha"],
                        row_weight=state["row_weight"], teacher_lse=state.get("teacher_lse"))
            if c["grad"]:
                loss, dlogits = S.distill_loss_and_grad(state["logits"], state["teacher_ids"],
                                                        state["teacher_logits"], **args)
                return {"loss": loss, "dlogits": dlogits}
            return {"loss": S.distill_loss(state["logits"], state["teacher_ids"], state["teacher_logits"],
                                           reduction="none", **args)}
        if c["op"] == "lookup":
            return S.embed_tokens(state["ids"], state["table"], scale=state["scale"])
        return S.embed_grad(state["ids"], state["dout"], c["V"], scale=state["scale"], dtype=DT[c["gdt"]])
    if c["op"] == "rules":
        return _ruled(state, state["logits"].float()).to(state["logits"].dtype)
    if c["op"] == "choose":
        return _choose(state)
    if c["op"] == "distill":
        return _distill(state)
    if c["op"] == "lookup":
        return (state["table"][state["ids"].long()].float() * state["scale"]).to(state["table"].dtype)
    dout = state["dout"].float() * state["scale"]
    grad = torch.zeros(c["V"], c["d"], device=dout.device).index_add_(0, state["ids"].long(), dout)
    return grad.to(DT[c["gdt"]])


def _distinct(N, V):
    """The table rows that N Zipf tokens are expected to touch."""
    w = np.arange(1, V + 1, dtype=np.float64) ** -1.1
    return float(-np.expm1(N * np.log1p(-w / w.sum())).sum())


def work(case):
    es = 2 if case["dt"] == "bf16" else 4
    V = case["V"]
    if case["op"] in ("rules", "choose"):
        S = case["S"]
        side = S * (case["hist"] * 3 + case["bias"] * 8 + 24) + (8 * V // 8 if case["mask"] else 0)
        if case["op"] == "rules":
            return {"bytes": 2 * S * V * es + side, "flops": 5 * S * V}
        return {"bytes": S * V * es + side + 24 * S, "flops": 8 * S * V}
    if case["op"] == "distill":
        N = case["N"]
        return {"bytes": N * V * es * (2 if case["grad"] else 1) + N * (case["k"] * 8 + 16),
                "flops": N * V * (4 + 4 * case["hard"]) * (2 if case["grad"] else 1)}
    N, d = case["N"], case["d"]
    if case["op"] == "lookup":
        return {"bytes": N * 4 + N * d * es + _distinct(N, V) * d * es, "flops": N * d}
    return {"bytes": N * 4 + N * d * es + V * d * (2 if case["gdt"] == "bf16" else 4), "flops": 2 * N * d}


def _exact_row(st, i, V):
    """Row i of the rules in 64 bits, token by token of its history."""
    x = st["logits"][i].double().cpu().numpy().copy()
    n, p0 = int(st["history_len"][i]), int(st["prompt_len"][i])
    h = st["history"][i, :n].cpu().numpy()
    seen = np.unique(h[h >= 0])
    r, f, p = (float(st[q][i]) for q in ("repetition", "frequency", "presence"))
    x[seen] = np.where(x[seen] > 0, x[seen] / r, x[seen] * r)
    made = h[p0:]
    tok, times = np.unique(made[made >= 0], return_counts=True)
    x[tok] -= f * times + p
    if "bias_ids" in st:
        np.add.at(x, st["bias_ids"][i].cpu().numpy(), st["bias_values"][i].double().cpu().numpy())
    if "mask" in st and int(st["mask_row"][i]) >= 0:
        words = st["mask"][int(st["mask_row"][i])].cpu().numpy().astype(np.uint32)
        bits = np.unpackbits(words.view(np.uint8), bitorder="little")[:V]
        x[bits == 0] = -np.inf
    return x


def _exact_choice(st, i, x):
    m = x.max()
    if m == -np.inf:
        return -np.inf
    T = float(st["temperature"][i])
    z = (x - m) / (T or 1.0)
    w = np.exp(z)
    if T == 0:
        return -math.log(w.sum())
    w = np.rint(w * UNIT)
    order = np.argsort(-x, kind="stable")
    k, p = int(st["top_k"][i]), float(st["top_p"][i])
    if 0 < k < x.size:
        order = order[:k]
    if p < 1:
        run_ = np.cumsum(w[order])
        order = order[(run_ - w[order]) < max(1.0, math.ceil(p * run_[-1]))]
    keep = np.sort(order)
    run_ = np.cumsum(w[keep])
    at = keep[min(int(np.searchsorted(run_, float(st["u"][i]) * run_[-1], side="right")), keep.size - 1)]
    return z[at] - math.log(run_[-1] / UNIT)


def exact(case, seed):
    st = prepare(case, seed)
    op, V = case["op"], case["V"]
    if op in ("rules", "choose"):
        rows = [_exact_row(st, i, V) for i in range(case["S"])]
        if op == "rules":
            return torch.from_numpy(np.stack(rows))
        return (None, torch.tensor([_exact_choice(st, i, x) for i, x in enumerate(rows)], dtype=torch.float64))
    if op == "lookup":
        return st["table"].double()[st["ids"].long()] * st["scale"]
    if op == "table_grad":
        order = torch.argsort(st["ids"], stable=True)
        run_ = torch.zeros(V, case["d"], dtype=torch.float64, device="cuda")
        return run_.index_add_(0, st["ids"][order].long(), st["dout"].double()[order]) * st["scale"]
    T, a, N = case["temp"], case["alpha"], case["N"]
    loss = torch.zeros(N, dtype=torch.float64, device="cuda")
    grad = torch.zeros(N, V, dtype=torch.float64, device="cuda") if case["grad"] else None
    for lo in range(0, N, 1024):
        hi = min(N, lo + 1024)
        s = st["logits"][lo:hi].double()
        ids, w = st["teacher_ids"][lo:hi].long(), st["row_weight"][lo:hi].double()
        row, col = (ids >= 0).nonzero(as_tuple=True)
        z = torch.full(ids.shape, -math.inf, dtype=torch.float64, device="cuda")
        z[row, col] = st["teacher_logits"][lo:hi].double()[row, col] / T
        norm = st["teacher_lse"][lo:hi].double() if case["tail"] else torch.logsumexp(z, 1)
        P = torch.zeros_like(s)
        P[row, ids[row, col]] = torch.exp(z[row, col] - norm[row])
        listed_ = torch.zeros_like(s, dtype=torch.bool)
        listed_[row, ids[row, col]] = True
        lq = torch.log_softmax(s / T, 1)
        part = torch.where(P > 0, P * (torch.log(P) - lq), 0.0).sum(1)
        G = P.sum(1, keepdim=True) * torch.exp(lq) - P
        if case["tail"]:
            some = listed_.any(1)
            pr = torch.where(some, (1 - P.sum(1)).clamp(min=0), 0.0)
            lr = torch.logsumexp(lq.masked_fill(listed_, -math.inf), 1)
            part = part + torch.where(pr > 0, pr * (torch.log(pr) - lr), 0.0)
            q = torch.exp(lq) * some[:, None]
            G = q * (P.sum(1) + pr)[:, None] - torch.where(listed_, P, q * (pr / torch.exp(lr))[:, None])
        each = a * T * T * part
        G = a * T * G
        if st["targets"] is not None:
            t = st["targets"][lo:hi].long()
            at = (t >= 0).nonzero()[:, 0]
            l1 = torch.log_softmax(s, 1)
            each[at] -= (1 - a) * l1[at, t[at]]
            one = torch.exp(l1) * (t >= 0)[:, None]
            one[at, t[at]] -= 1
            G = G + (1 - a) * one
        loss[lo:hi] = w * each
        if grad is not None:
            grad[lo:hi] = w[:, None] * G
    return {"loss": loss, "dlogits": grad} if case["grad"] else {"loss": loss}
