"""The vocabulary-end operators (process_logits, sample_logits, distill_loss, embed_tokens and their gradients) on the
GPU against plain 64-bit implementations written here, at the sizes and values where they can go wrong: odd
vocabularies and strides, rows that a mask empties, infinities and NaN, empty and repeated histories, ties, teacher
entries that are missing or repeated, tokens that occur thousands of times.

Tolerances are bounds on rounding: u = 2^-24 per float32 operation, h = 2^-8 for one rounding to bfloat16 (twice the
half step, so that a float32 error on a rounding boundary is covered); two values that are each rounded can be a whole
step, 2 h, apart."""
import math

import numpy as np
import pytest
import torch

import sdmchat_b200 as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
U, H = 2.0 ** -24, 2.0 ** -8
F32, BF16 = torch.float32, torch.bfloat16


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def np64(t):
    return t.detach().double().cpu().numpy()


# ------------------------------------------------------------------------------------------------ rules on logits
def make_rules(rows, V, L, nb, masks, seed, prompt=True):
    g = gen(seed)
    r = S.LogitRules()
    if L:
        r.history = torch.randint(-1, max(2, min(V, 40)), (rows, L), generator=g, device=DEV, dtype=torch.int32)
        r.history[:, ::5] = V  # outside: skipped
        r.history_len = torch.randint(0, L + 1, (rows,), generator=g, device=DEV, dtype=torch.int32)
        if prompt:
            r.prompt_len = torch.randint(0, L + 1, (rows,), generator=g, device=DEV, dtype=torch.int32)
        r.repetition = 1 + torch.rand(rows, generator=g, device=DEV)
        r.frequency = torch.rand(rows, generator=g, device=DEV)
        r.presence = 0.25
    if nb:
        r.bias_ids = torch.randint(-1, max(2, min(V, 8)), (rows, nb), generator=g, device=DEV, dtype=torch.int32)
        r.bias_values = torch.randn(rows, nb, generator=g, device=DEV)
    if masks:
        r.mask = torch.randint(-2 ** 31, 2 ** 31 - 1, (masks, -(-V // 32)), generator=g, device=DEV, dtype=torch.int32)
        r.mask[0] = 0
        r.mask_row = torch.arange(rows, device=DEV, dtype=torch.int32) % (masks + 1) - 1
    return r


def ruled64(x, r, row, V):
    """(values, magnitude for the rounding bound) of one row."""
    x = x.copy()
    mag = np.abs(x)
    if r.history is not None:
        h = r.history[row].cpu().numpy()
        n = len(h) if r.history_len is None else int(r.history_len[row])
        p = 0 if r.prompt_len is None else min(int(r.prompt_len[row]), n)
        rep, frq, prs = (float(v[row]) if torch.is_tensor(v) else v for v in (r.repetition, r.frequency, r.presence))
        seen = sorted({t for t in h[:n] if 0 <= t < V})
        for t in seen:
            x[t] = x[t] / rep if x[t] > 0 else x[t] * rep
            k = int((h[p:n] == t).sum())
            if k:
                x[t] = x[t] - frq * k - prs
            mag[t] = max(mag[t], abs(x[t])) * 2 + frq * k + prs
    if r.bias_ids is not None:
        for t, b in zip(r.bias_ids[row].tolist(), r.bias_values[row].tolist()):
            if 0 <= t < V:
                x[t] += b
                mag[t] += abs(b)
    if r.mask is not None:
        m = int(r.mask_row[row]) if r.mask_row is not None else (0 if r.mask.shape[0] == 1 else row)
        if 0 <= m < r.mask.shape[0]:
            words = r.mask[m].cpu().numpy().view(np.uint32)
            for t in range(V):
                if not (words[t // 32] >> (t % 32)) & 1:
                    x[t] = -np.inf
    return x, mag


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("rows,V,L,nb,masks", [(1, 1, 3, 1, 0), (3, 31, 0, 0, 2), (2, 33, 7, 3, 1), (5, 1000, 64, 0, 4),
                                               (4, 2053, 700, 9, 3), (2, 32768, 2048, 16, 2), (3, 50021, 1, 0, 0)])
def test_process_logits(cuda_ok, dt, rows, V, L, nb, masks):
    r = make_rules(rows, V, L, nb, masks, rows + V)
    x = (3 * torch.randn(rows, V, generator=gen(V), device=DEV)).to(dt)
    before = x.clone()
    y = S.process_logits(x, r)
    assert torch.equal(x, before) and y.dtype == dt
    for i in range(rows):
        want, mag = ruled64(np64(x)[i], r, i, V)
        got = np64(y)[i]
        dead = np.isneginf(want)
        np.testing.assert_array_equal(np.isneginf(got), dead)
        tol = 8 * nb * U * mag + 8 * U * mag + (H * np.abs(want) if dt == BF16 else 0)
        assert (np.abs(got[~dead] - want[~dead]) <= tol[~dead]).all()
    z = x.clone()
    assert S.process_logits(z, r, out=z) is z and torch.equal(z, y)  # in place


def test_process_logits_strides_and_values(cuda_ok):
    V = 517
    base = torch.randn(4, 640, generator=gen(1), device=DEV).to(BF16)
    for lead in (0, 1, 3, 5):  # rows that begin at every kind of address, a stride wider than the row
        x = base[:, lead:lead + V]
        r = make_rules(4, V, 50, 2, 3, 7)
        out = torch.zeros(4, 700, device=DEV, dtype=BF16)
        got = S.process_logits(x, r, out=out[:, 9:9 + V])
        assert torch.equal(got, S.process_logits(x.contiguous(), r))
        assert out[:, :9].abs().sum() == 0 and out[:, 9 + V:].abs().sum() == 0
    # masked places hold anything; infinities and NaN elsewhere stay what they are
    x = torch.tensor([[float("nan"), math.inf, -math.inf, torch.finfo(F32).min, 1.0, float("nan")]], device=DEV)
    mask = torch.tensor([[0b011110]], device=DEV, dtype=torch.int32)
    y = S.process_logits(x, S.LogitRules(mask=mask))[0].tolist()
    assert y[0] == -math.inf and y[1] == math.inf and y[2] == -math.inf and y[5] == -math.inf and y[4] == 1.0
    y = S.process_logits(x)[0]
    assert torch.isnan(y[0]) and torch.isnan(y[5]) and torch.equal(y[1:5], x[0, 1:5])
    # one mask for all rows, one mask per row, no rows
    x = torch.randn(3, 40, generator=gen(2), device=DEV)
    one = torch.tensor([[-1, 0]], device=DEV, dtype=torch.int32)
    assert torch.isneginf(S.process_logits(x, S.LogitRules(mask=one))[:, 32:]).all()
    each = torch.tensor([[0, 0], [-1, -1], [1, 0]], device=DEV, dtype=torch.int32)
    assert torch.isneginf(S.process_logits(x, S.LogitRules(mask=each))).sum(1).tolist() == [40, 0, 39]
    assert S.process_logits(x[:0]).shape == (0, 40)


# -------------------------------------------------------------------------------------------------- token choice
def kept64(x, T, k, p):
    """Kept tokens (ascending) and their masses."""
    w = np.where(x == x.max(), 1.0, np.exp(np.where(x == x.max(), 0.0, x - x.max()) / T))
    order = np.argsort(-x, kind="stable")
    if 0 < k < len(x):
        order = order[:k]
    if p < 1:
        c = np.cumsum(w[order])
        order = order[c - w[order] < p * c[-1]]
    keep = np.sort(order)
    return keep, w[keep]


def clear_p(x, T, k, share):
    """A top_p near `share` that lies in the middle of a kept token's mass, away from rounding."""
    keep, w = kept64(x, T, k, 1.0)
    w = np.sort(w)[::-1]
    c = np.cumsum(w)
    i = int(np.searchsorted(c, share * c[-1]))
    return (c[i] - 0.5 * w[i]) / c[-1]


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("rows,V,k,share,T", [(1, 1, 0, 1.0, 1.0), (6, 7, 3, 1.0, 0.7), (5, 100, 0, 0.6, 1.3),
                                              (7, 1000, 50, 0.8, 0.5), (3, 4099, 0, 1.0, 1.0), (160, 2000, 200, 0.9, 1.0),
                                              (4, 32768, 0, 0.7, 0.8), (2, 50021, 1000, 0.95, 1.0),
                                              (1, 200003, 40, 0.9, 1.0), (300, 37, 5, 1.0, 2.0)])
def test_sample_logits(cuda_ok, dt, rows, V, k, share, T):
    """u in the middle of a token's share of the kept mass has to give that token."""
    x = (4 * torch.randn(rows, V, generator=gen(V + rows), device=DEV)).to(dt)
    rng = np.random.default_rng(V)
    xs = np64(x)
    p = [1.0 if share >= 1 else clear_p(xs[i], T, k, share) for i in range(rows)]
    u, want, lp = [], [], []
    for i in range(rows):
        keep, w = kept64(xs[i], T, k, p[i])
        c = np.cumsum(w)
        heavy = np.flatnonzero(w > 1e-4 * c[-1])  # shares that float32 masses resolve
        j = int(rng.choice(heavy))
        u.append((c[j] - 0.5 * w[j]) / c[-1])
        want.append(int(keep[j]))
        lp.append(math.log(w[j] / c[-1]))
    d = lambda v: torch.tensor(v, device=DEV, dtype=F32)  # noqa: E731
    ids, got = S.sample_logits(x, u=d(u), temperature=T, top_k=k, top_p=d(p) if share < 1 else 1.0)
    assert ids.tolist() == want
    # t = (x - m) / T has two roundings of |t|, the mass three more, their sum's logarithm its own
    tol = 16 * U * (1 + np.abs(lp))
    assert (np.abs(np64(got) - lp) <= tol).all()
    ids, got = S.sample_logits(x, temperature=0.0)  # greedy: the lowest index of the largest
    assert ids.tolist() == [int(np.argmax(r)) for r in xs]
    want_lp = [-math.log(np.exp(r - r.max()).sum()) for r in xs]
    assert np.allclose(np64(got), want_lp, rtol=16 * U, atol=16 * U)


@pytest.mark.parametrize("crowd,far", [(100, 0), (700, 0), (1024, 0), (1025, 0), (100, 800), (30, 1100)])
@pytest.mark.parametrize("k,share", [(300, 1.0), (0, 0.6), (500, 0.45), (0, 0.95)])
@pytest.mark.parametrize("rows", [2, 200])
def test_sample_crowded_cut(cuda_ok, crowd, far, k, share, rows):
    """The cut among many tokens whose logits are close or tied, and among tokens whose masses are 0."""
    V, g = 3000, gen(crowd + far)
    x = torch.full((rows, V), -math.inf, device=DEV)
    for i in range(rows):
        at = torch.randperm(V, generator=g, device=DEV)
        steps = torch.randint(0, 64, (crowd,), generator=g, device=DEV)
        x[i, at[:crowd]] = -5.02 - steps / 1024.0  # ties among them
        x[i, at[crowd:crowd + far]] = -40.0 - torch.rand(far, generator=g, device=DEV)
        x[i, at[crowd + far]] = 0.0
    rng = np.random.default_rng(crowd)
    xs = np64(x)
    p = [1.0 if share >= 1 else clear_p(xs[i], 1.0, k, share) for i in range(rows)]
    u, want, lp = [], [], []
    for i in range(rows):
        keep, w = kept64(xs[i], 1.0, k, p[i])
        c = np.cumsum(w)
        j = int(rng.choice(np.flatnonzero(w > 1e-4 * c[-1])))
        u.append((c[j] - 0.5 * w[j]) / c[-1])
        want.append(int(keep[j]))
        lp.append(math.log(w[j] / c[-1]))
    d = lambda v: torch.tensor(v, device=DEV, dtype=F32)  # noqa: E731
    ids, got = S.sample_logits(x, u=d(u), top_k=k, top_p=d(p) if share < 1 else 1.0)
    assert ids.tolist() == want
    assert (np.abs(np64(got) - lp) <= 16 * U * (1 + np.abs(lp))).all()


def test_sample_ties_and_ends(cuda_ok):
    V = 3000
    x = torch.zeros(4, V, device=DEV)
    d = lambda v: torch.tensor(v, device=DEV, dtype=F32)  # noqa: E731
    # all tied: the lowest indices are kept, so u spreads over them
    ids, lp = S.sample_logits(x, u=d([0.0, 0.999999, 0.5, 0.1]), top_k=10)
    assert ids.tolist() == [0, 9, 5, 1] and torch.allclose(lp, d([math.log(0.1)] * 4), atol=1e-6)
    ids, _ = S.sample_logits(x, u=d([0.0, 0.999999, 0.5, 0.1]), top_p=0.5)
    assert ids.tolist() == [0, V // 2 - 1, V // 4, 150]
    # a tie on the cut, some of it kept: 5 of the 100 tokens at 0, after 3 above
    x = torch.full((4, V), -50.0, device=DEV)
    x[:, 100:200] = 0.0
    x[:, [7, 1500, 2900]] = math.log(2.0)
    keep = [7] + list(range(100, 105)) + [1500, 2900]
    u = [(sum(2 if t in (7, 1500, 2900) else 1 for t in keep[:j]) + 0.5) / 11 for j in (0, 3, 5, 7)]
    ids, _ = S.sample_logits(x, u=d(u), top_k=8)
    assert ids.tolist() == [7, 102, 104, 2900]
    # u at and beyond its ends, a temperature that leaves one token, one that levels all
    x = torch.randn(4, V, generator=gen(5), device=DEV)
    ids, _ = S.sample_logits(x, u=d([0.0, 1.0, 2.0, -1.0]))
    assert ids.tolist() == [0, V - 1, V - 1, 0]
    ids, _ = S.sample_logits(x, u=d([0.3] * 4), temperature=d([1e-6, 1e-30, 0.0, -1.0]))
    assert torch.equal(ids.long(), x.argmax(1))
    ids, _ = S.sample_logits(x, u=d([0.0, 0.25, 0.5, 0.75]), temperature=1e30)
    assert ids.tolist() == [0, V // 4, V // 2, 3 * V // 4]
    # tiny and zero top_p keep one token; top_k 1 too
    for kw in (dict(top_p=0.0), dict(top_p=1e-7), dict(top_p=-1.0), dict(top_k=1)):
        ids, lp = S.sample_logits(x, u=d([0.9] * 4), **kw)
        assert torch.equal(ids.long(), x.argmax(1)) and lp.abs().max() == 0
    # -0 and +0 are one value: index order decides
    x = torch.full((1, 64), -1.0, device=DEV)
    x[0, 9], x[0, 20] = -0.0, 0.0
    assert S.sample_logits(x, temperature=0.0)[0].item() == 9
    assert S.sample_logits(x, u=d([0.9]), top_k=1)[0].item() == 9


def test_sample_masked_and_special(cuda_ok):
    d = lambda v: torch.tensor(v, device=DEV, dtype=F32)  # noqa: E731
    inf, nan = math.inf, math.nan
    x = d([[-inf, -inf, -inf, -inf], [nan, nan, nan, nan], [nan, 2.0, nan, -inf], [1.0, inf, inf, 0.0],
           [torch.finfo(F32).min] * 4])
    for kw in (dict(temperature=0.0), dict(u=d([0.6] * 5)), dict(u=d([0.6] * 5), top_k=3, top_p=0.9)):
        ids, lp = S.sample_logits(x, **kw)
        greedy = "u" not in kw
        assert ids[:3].tolist() == [-1, -1, 1] and lp[:3].tolist() == [-inf, -inf, 0.0]
        assert ids[3].item() == (1 if greedy else 2) and lp[3].item() == pytest.approx(-math.log(2), abs=1e-6)
        n = 3 if "top_k" in kw else 4
        assert ids[4].item() == (0 if greedy else int(0.6 * n))
    # a mask that leaves one token, and one that leaves none, under every kind of choice
    V = 5000
    x = torch.randn(2, V, generator=gen(3), device=DEV)
    mask = torch.zeros(2, -(-V // 32), device=DEV, dtype=torch.int32)
    mask[0, 4321 // 32] = 1 << (4321 % 32)
    for kw in (dict(temperature=0.0), dict(u=d([0.99, 0.5])), dict(u=d([0.0, 0.5]), top_k=5, top_p=0.3)):
        ids, lp = S.sample_logits(x, S.LogitRules(mask=mask), **kw)
        assert ids.tolist() == [4321, -1] and lp.tolist() == [0.0, -inf]
    assert S.sample_logits(x[:0], temperature=0.0)[0].shape == (0,)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_sample_agrees_with_processed_logits(cuda_ok, dt):
    """Choosing under rules is choosing from the processed logits (float32: bf16 logits are widened first)."""
    rows, V = 9, 3001
    r = make_rules(rows, V, 80, 4, 3, 11)
    x = (3 * torch.randn(rows, V, generator=gen(12), device=DEV)).to(dt)
    u = torch.rand(rows, generator=gen(13), device=DEV)
    y = S.process_logits(x.float(), r)
    for kw in (dict(temperature=0.0), dict(u=u), dict(u=u, temperature=0.7, top_k=20, top_p=0.9)):
        a, b = S.sample_logits(x, r, **kw), S.sample_logits(y, **kw)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        wide = torch.zeros(rows, V + 6, device=DEV, dtype=dt)
        wide[:, 3:V + 3] = x
        c = S.sample_logits(wide[:, 3:V + 3], r, **kw)
        assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


def test_sample_follows_the_distribution(cuda_ok):
    """Evenly spaced u reproduce the probabilities to within one draw per token."""
    n, V = 4000, 50
    x = torch.randn(1, V, generator=gen(4), device=DEV)
    u = (torch.arange(n, device=DEV) + 0.5) / n
    ids, _ = S.sample_logits(x.expand(n, V).contiguous(), u=u, temperature=0.9)
    want = torch.softmax(x[0].double() / 0.9, 0) * n
    assert (torch.bincount(ids.long(), minlength=V) - want).abs().max() <= 1.01


# -------------------------------------------------------------------------------------------------- distillation
def distill64(x, ids, tl, tg, w, T, a, lse):
    """(loss, gradient, magnitudes for the rounding bounds) of one row in 64 bits."""
    V = len(x)
    z = x / T
    lq = z - (z.max() + np.log(np.exp(z - z.max()).sum()))
    l1 = x - (x.max() + np.log(np.exp(x - x.max()).sum()))
    g, mag = np.zeros(V), np.zeros(V)
    ok = [j for j in range(len(ids)) if 0 <= ids[j] < V and tl[j] > -np.inf]
    loss, lm = 0.0, 0.0
    if ok:
        zt = np.array([tl[j] / T for j in ok])
        lp = zt - (zt.max() + np.log(np.exp(zt - zt.max()).sum()) if lse is None else lse)
        p = np.exp(lp)
        at = np.array([ids[j] for j in ok])
        soft = float((p * (lp - lq[at])).sum())
        lm = float((p * (np.abs(lp) + np.abs(lq[at]) + 1)).sum())
        pr = 0.0
        listed = np.zeros(V, bool)
        listed[at] = True
        if lse is not None:
            pr = max(0.0, 1 - p.sum())
        q = np.exp(lq)
        gs = (p.sum() + pr) * q
        gm = gs.copy()
        if pr > 0:
            qr = q[~listed].sum()
            soft += pr * (math.log(pr) - math.log(qr))
            lm += (p.sum() + 1) * (abs(math.log(pr)) + abs(math.log(qr)) + 1)  # pr = 1 - P carries P's error
            gs[~listed] -= pr * q[~listed] / qr
            gm[~listed] += (pr + 1) * q[~listed] / qr
        np.add.at(gs, at, -p)
        np.add.at(gm, at, p)
        loss += a * T * T * soft
        lm *= a * T * T
        g += a * T * gs
        mag += a * T * gm
    if 0 <= tg < V:
        loss -= (1 - a) * l1[tg]
        lm += (1 - a) * (abs(l1[tg]) + 1)
        q = np.exp(l1)
        g += (1 - a) * q
        mag += (1 - a) * q
        g[tg] -= 1 - a
        mag[tg] += 1 - a
    return w * loss, w * g, w * lm, w * mag


# float32 error of a probability: exp of a difference d (|d| * 2 u for its roundings, up to |d| = 40 where the
# probability still counts), 4 u for the exponential, the sum and the quotient
PERR = 100 * U


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("N,V,k,T,a,hard,tail", [(1, 1, 1, 1.0, 1.0, False, False), (3, 17, 5, 2.0, 0.5, True, True),
                                                 (5, 1000, 8, 1.0, 0.7, True, False), (4, 2053, 64, 0.7, 1.0, False, True),
                                                 (200, 311, 16, 3.0, 0.3, True, True), (2, 32768, 100, 2.0, 0.5, True, False),
                                                 (3, 50021, 512, 1.0, 0.9, True, True), (1, 131073, 33, 1.5, 0.5, True, True),
                                                 (2, 262144, 4, 1.0, 0.0, True, False), (600, 517, 20, 2.0, 0.6, True, True),
                                                 (150, 9001, 30, 2.0, 0.5, True, False), (600, 24007, 7, 1.7, 0.5, True, True),
                                                 (593, 1024, 128, 1.0, 1.0, False, False), (601, 2053, 129, 0.8, 0.5, True, False)])
def test_distill(cuda_ok, dt, N, V, k, T, a, hard, tail):
    g = gen(V + k)
    x = (3 * torch.randn(N, V, generator=g, device=DEV)).to(dt)
    ids = torch.stack([torch.randperm(V, generator=g, device=DEV)[:k] if V >= k else
                       torch.randint(0, V, (k,), generator=g, device=DEV) for _ in range(N)]).to(torch.int32)
    tl = 2 * torch.randn(N, k, generator=g, device=DEV)
    if k >= 5:
        ids[0, 1] = ids[0, 3]      # listed twice
        ids[-1, 2], ids[-1, 4] = -1, V  # unused
        tl[0, 0] = -math.inf       # probability 0: unused
    if N >= 3:
        ids[1] = -1                # no teacher at all
    tg = torch.randint(0, V, (N,), generator=g, device=DEV, dtype=torch.int32) if hard else None
    if hard and N >= 3:
        tg[2], tg[0] = -1, ids[0, -1]  # no target; a target that the teacher lists
    w = torch.rand(N, generator=g, device=DEV)
    if N > 3:
        w[3] = 0.0
        x[3, 0] = math.nan         # a row of weight 0 is not read
    lse = None
    if tail:
        zt = (tl / T).masked_fill((ids < 0) | (ids >= V), -math.inf)
        lse = torch.logsumexp(zt, 1).nan_to_num(neginf=0.0) + 0.3
    loss, grad = S.distill_loss_and_grad(x, ids, tl, tg, T, a, w, lse, grad_scale=0.5)
    only = S.distill_loss(x, ids, tl, tg, T, a, w, lse, reduction="none")
    assert grad.dtype == dt and grad.shape == x.shape
    xs, tls, grads = np64(x), np64(tl), np64(grad)
    for i in range(N):
        if float(w[i]) == 0:
            assert loss[i] == 0 and only[i] == 0 and torch.count_nonzero(grad[i]) == 0
            continue
        wl, wg, lm, mag = distill64(xs[i], ids[i].tolist(), tls[i], int(tg[i]) if hard else -1, float(w[i]),
                                    T, a, None if lse is None else float(lse[i]))
        assert abs(float(loss[i]) - wl) <= PERR * lm + 1e-30, (i, float(loss[i]), wl)
        assert abs(float(only[i]) - wl) <= PERR * lm + 1e-30, (i, float(only[i]), wl)  # the loss without a gradient
        got = grads[i]
        tol = 0.5 * PERR * mag + (H * np.abs(0.5 * wg) if dt == BF16 else 0) + 1e-37
        assert (np.abs(got - 0.5 * wg) <= tol).all(), (i, np.abs(got - 0.5 * wg).max())
    z = x.clone()
    l2, g2 = S.distill_loss_and_grad(z, ids, tl, tg, T, a, w, lse, grad_scale=0.5, out=z)  # over the logits
    assert g2 is z and torch.equal(l2, loss) and torch.equal(z, grad)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("N,V,k,T,a,hard,tail", [(3, 17, 5, 4.0, 0.5, True, True), (200, 2053, 16, 4.0, 0.3, True, False),
                                                 (150, 9001, 30, 4.0, 0.5, True, True), (2, 50021, 300, 4.0, 0.5, True, True),
                                                 (600, 24007, 7, 2.0, 0.5, True, False), (600, 22001, 7, 4.0, 0.5, True, True),
                                                 (600, 26003, 128, 2.0, 0.5, True, True), (593, 33005, 7, 4.0, 0.4, True, True),
                                                 (300, 24007, 7, 2.0, 0.5, True, True)])
def test_distill_powers(cuda_ok, dt, N, V, k, T, a, hard, tail):
    """At T = 2 and 4 the exponential at 1 is a power of the one at T: its error, 4 u for the exponential, grows by the
    same power (16 u, and 2 u for the squarings), which PERR's 16 u beyond the 80 u of the difference's roundings hold
    with that of the sum."""
    test_distill(cuda_ok, dt, N, V, k, T, a, hard, tail)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("N,V", [(3, 40), (600, 24003), (600, 28001), (2, 50021)])
@pytest.mark.parametrize("T", [1.0, 2.0, 0.5, 3.0])
def test_distill_rows_at_the_ends_of_the_range(cuda_ok, dt, N, V, T):
    """A row all at the type's lowest value is level; a row with one token at its highest has all mass there."""
    if dt == F32 and V > 20000:
        V //= 2
    x = torch.full((N, V), torch.finfo(dt).min, device=DEV, dtype=dt)
    x[1] = 0.0
    x[1, 7] = torch.finfo(dt).max
    ids = torch.tensor([[3, 7]] * N, device=DEV, dtype=torch.int32)
    tl, tg = torch.zeros(N, 2, device=DEV), torch.full((N,), 7, device=DEV, dtype=torch.int32)
    ids[1], tl[1] = torch.tensor([7, -1], device=DEV), 0.0
    lse = torch.full((N,), math.log(4.0), device=DEV)  # half the teacher's mass on the two
    for tail in (None, lse):
        loss, grad = S.distill_loss_and_grad(x, ids, tl, tg, T, 0.5, None, tail)
        only = S.distill_loss(x, ids, tl, tg, T, 0.5, None, tail, reduction="none")
        for i in {0, N - 1} - {1}:
            soft = math.log(V) - math.log(2) if tail is None else \
                0.5 * (math.log(V) - math.log(4)) + 0.5 * (math.log(0.5) - math.log((V - 2) / V))
            want = 0.5 * T * T * soft + 0.5 * math.log(V)
            mag = 0.5 * T * T * (2 * math.log(V) + 4) + 0.5 * (math.log(V) + 1)
            assert abs(float(loss[i]) - want) <= PERR * mag and abs(float(only[i]) - want) <= PERR * mag
            p, rest = (0.5, 1 / V) if tail is None else (0.25, 1 / V - 0.5 / (V - 2))
            g = grad[i].double().cpu().numpy()
            h = H if dt == BF16 else 0
            want7, want3 = 0.5 * T * (1 / V - p) + 0.5 * (1 / V - 1), 0.5 * T * (1 / V - p) + 0.5 / V
            want0 = 0.5 * T * rest + 0.5 / V
            m0 = 0.5 * T * (1 / V + 0.5 / V) + 0.5 / V
            assert abs(g[7] - want7) <= PERR * (T + 1) + h * abs(want7) and abs(g[3] - want3) <= PERR * T + h * abs(want3)
            others = np.delete(g, [3, 7])
            assert (np.abs(others - want0) <= PERR * 2 * m0 + h * abs(want0)).all()
        if tail is None:
            assert abs(float(loss[1])) <= PERR and abs(float(only[1])) <= PERR and grad[1].abs().max() <= PERR


def test_distill_powers_of_excluded_tokens(cuda_ok):
    """Logits of -infinity and far below the largest, where the exponential at 1 is 0 and the one at T is not."""
    for T in (2.0, 4.0):
        for V in (40, 24000):
            x = torch.zeros(600, V, device=DEV)
            x[:, 3], x[:, 4], x[:, 5] = -math.inf, -200.0, torch.finfo(F32).min
            ids = torch.full((600, 1), 0, device=DEV, dtype=torch.int32)
            tl, tg = torch.zeros(600, 1, device=DEV), torch.full((600,), 1, device=DEV, dtype=torch.int32)
            for dt in (F32, BF16):
                loss, grad = S.distill_loss_and_grad(x.to(dt), ids, tl, tg, T, 0.5)
                only = S.distill_loss(x.to(dt), ids, tl, tg, T, 0.5, reduction="none")
                far = math.exp(-200.0 / T)
                q, q1 = 1 / (V - 3 + far), 1 / (V - 3)
                want = 0.5 * T * T * math.log(1 / q) + 0.5 * math.log(1 / q1)
                mag = 0.5 * T * T * (math.log(1 / q) + 1) + 0.5 * (math.log(1 / q1) + 1)
                assert (loss.double() - want).abs().max() <= PERR * mag and (only.double() - want).abs().max() <= PERR * mag
                assert (grad[:, 3] == 0).all() and (grad[:, 5] == 0).all()
                g4, g6 = 0.5 * T * q * far, 0.5 * T * q + 0.5 * q1
                h = H if dt == BF16 else 0
                assert ((grad[:, 4].double() - g4).abs() <= (4 * PERR + h) * g4 + 1e-37).all()  # |d| up to 100 there
                assert ((grad[:, 6].double() - g6).abs() <= (PERR + h) * g6).all()


@pytest.mark.parametrize("dt,V", [(F32, 11000), (BF16, 22000), (F32, 14003), (BF16, 30005)])
def test_distill_many_rows(cuda_ok, dt, V):
    """Rows enough that every block has many, and half of them without weight, so that one half of a block runs ahead
    of the other: every row against torch in 64 bits."""
    N, k, a = 3000, 9, 0.5  # 44 and 56 to 60 KB a row: a block per row, and persistent blocks
    g = gen(77)
    x = (3 * torch.randn(N, V, generator=g, device=DEV)).to(dt)
    ids = torch.randint(-1, V, (N, k), generator=g, device=DEV, dtype=torch.int32)
    tl = torch.randn(N, k, generator=g, device=DEV)
    tg = torch.randint(-1, V, (N,), generator=g, device=DEV, dtype=torch.int32)
    w = (torch.rand(N, generator=g, device=DEV) > 0.5).float()
    w[::5] = 0.0
    for T in (1.0, 2.0, 4.0):
        loss, grad = S.distill_loss_and_grad(x, ids, tl, tg, T, a, w)
        xd, wd = x.double(), w.double()
        lq, l1 = torch.log_softmax(xd / T, 1), torch.log_softmax(xd, 1)
        ok, some = ids >= 0, (ids >= 0).any(1)
        lp = torch.log_softmax((tl.double() / T).masked_fill(~ok, -math.inf), 1)
        p = torch.where(ok, lp.exp(), 0.0).nan_to_num()
        at = ids.clamp(min=0).long()
        lqa = lq.gather(1, at)
        soft = torch.where(ok, p * (lp - lqa), 0.0).sum(1)
        mag = torch.where(ok, p * (lp.abs() + lqa.abs() + 1), 0.0).sum(1) * a * T * T
        G, M = lq.exp() * some[:, None], lq.exp() * some[:, None]
        G, M = G.scatter_add(1, at, -p) * a * T, M.scatter_add(1, at, p) * a * T
        hit, t = tg >= 0, tg.clamp(min=0).long()[:, None]
        one = (1 - a) * hit[:, None].double()
        lt = l1.gather(1, t)[:, 0]
        want = wd * (a * T * T * soft - (1 - a) * torch.where(hit, lt, 0.0))
        mag = mag + (1 - a) * torch.where(hit, lt.abs() + 1, 0.0)
        G = wd[:, None] * (G + one * l1.exp()).scatter_add(1, t, -one)
        M = wd[:, None] * (M + one * l1.exp()).scatter_add(1, t, one)
        assert ((loss - want).abs() <= PERR * mag + 1e-30).all()
        assert ((grad.double() - G).abs() <= PERR * M + (H * G.abs() if dt == BF16 else 0) + 1e-37).all()


def test_distill_strides_and_values(cuda_ok):
    N, V, k = 4, 517, 6
    g = gen(9)
    ids = torch.randint(0, V, (N, k), generator=g, device=DEV, dtype=torch.int32)
    tl = torch.randn(N, k, generator=g, device=DEV)
    base = torch.randn(N, 640, generator=g, device=DEV).to(BF16)
    for lead in (0, 1, 5):
        x = base[:, lead:lead + V]
        out = torch.zeros(N, 700, device=DEV, dtype=BF16)
        l0, g0 = S.distill_loss_and_grad(x.contiguous(), ids, tl, temperature=2.0)
        l1, g1 = S.distill_loss_and_grad(x, ids, tl, temperature=2.0, out=out[:, 3:3 + V])
        assert out[:, :3].abs().sum() == 0 and out[:, 3 + V:].abs().sum() == 0
        # an odd start puts other elements into a thread's share: sums differ by their order only
        assert torch.allclose(g0.float(), g1.float(), rtol=2 * H, atol=PERR)
        assert torch.allclose(l0, l1, rtol=PERR, atol=PERR)
    # a student that excludes a token the teacher wants: infinite loss, the gradient pulls the token up
    x = torch.randn(2, 40, generator=g, device=DEV)
    x[0, 5] = -math.inf
    ids = torch.tensor([[5, 6], [5, 6]], device=DEV, dtype=torch.int32)
    tl = torch.zeros(2, 2, device=DEV)
    loss, grad = S.distill_loss_and_grad(x, ids, tl)
    assert loss[0] == math.inf and abs(grad[0, 5] + 0.5) <= PERR and torch.isfinite(grad).all() and torch.isfinite(loss[1])
    # the type's lowest value is a number like another
    x[0, 5] = torch.finfo(F32).min
    loss, grad = S.distill_loss_and_grad(x, ids, tl)
    assert abs(grad[0, 5] + 0.5) <= PERR and torch.isfinite(grad).all() and not torch.isnan(loss).any()
    # NaN in a row stays in the row
    x[0, 7] = math.nan
    loss, grad = S.distill_loss_and_grad(x, ids, tl)
    assert torch.isnan(loss[0]) and torch.isfinite(loss[1]) and torch.isfinite(grad[1]).all()
    assert S.distill_loss_and_grad(x[:0], ids[:0], tl[:0])[1].shape == (0, 40)


@pytest.mark.parametrize("tail", [False, True])
def test_distill_gradient_against_differences(cuda_ok, tail):
    """<gradient, d> against (loss(x + e d) - loss(x - e d)) / 2e along directions of entries +-1.  The third
    derivative of a softmax's log-sum at T is a third central moment, at most 8 / T^3 here, of up to two sums (all
    tokens and the unlisted ones), so the truncation is at most 2 e^2 8 / 6 (soft T^2 / T^3, hard 1)."""
    N, V, k, T, a, e = 6, 700, 10, 1.5, 0.6, 2.0 ** -6
    g = gen(21)
    x = torch.randn(N, V, generator=g, device=DEV)
    ids = torch.stack([torch.randperm(V, generator=g, device=DEV)[:k] for _ in range(N)]).to(torch.int32)
    tl = torch.randn(N, k, generator=g, device=DEV)
    tg = torch.randint(0, V, (N,), generator=g, device=DEV, dtype=torch.int32)
    lse = torch.logsumexp(tl / T, 1) + 0.4 if tail else None
    loss, grad = S.distill_loss_and_grad(x, ids, tl, tg, T, a, None, lse)
    for s in range(4):
        d = torch.randint(0, 2, (N, V), generator=gen(30 + s), device=DEV).float() * 2 - 1
        up = S.distill_loss(x + e * d, ids, tl, tg, T, a, None, lse, reduction="none").double()
        dn = S.distill_loss(x - e * d, ids, tl, tg, T, a, None, lse, reduction="none").double()
        want = (up - dn) / (2 * e)
        got = (grad.double() * d).sum(1)
        tol = 2 * 8 / 6 * e * e + PERR * 2 * loss.abs().max() / (2 * e)
        assert ((got - want).abs() <= tol).all()


def test_distill_autograd(cuda_ok):
    N, V, k = 5, 300, 4
    g = gen(41)
    ids = torch.randint(0, V, (N, k), generator=g, device=DEV, dtype=torch.int32)
    tl = torch.randn(N, k, generator=g, device=DEV)
    tg = torch.randint(0, V, (N,), generator=g, device=DEV)
    x0 = torch.randn(N, V, generator=g, device=DEV)
    loss0, grad0 = S.distill_loss_and_grad(x0, ids, tl, tg, 2.0, 0.5)
    c = torch.rand(N, generator=g, device=DEV)
    for red, head, want in (("sum", lambda v: v, grad0), ("mean", lambda v: v, grad0 / N), ("sum", lambda v: 3 * v, 3 * grad0),
                            ("none", lambda v: (v * c).sum(), grad0 * c[:, None]), ("none", lambda v: v.sum(), grad0)):
        x = x0.clone().requires_grad_()
        loss = S.distill_loss(x, ids, tl, tg, 2.0, 0.5, reduction=red)
        assert torch.allclose(loss, {"sum": loss0.sum(), "mean": loss0.mean(), "none": loss0}[red], rtol=8 * U * N)
        head(loss).backward()
        assert torch.allclose(x.grad, want, rtol=8 * U, atol=U)
    with torch.no_grad():
        assert not S.distill_loss(x, ids, tl, tg).requires_grad


# --------------------------------------------------------------------------------------------------- token table
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("N,V,d", [(1, 1, 1), (7, 10, 33), (300, 50, 64), (64, 1000, 330), (1000, 37, 768), (5, 40, 1536)])
def test_embed_tokens(cuda_ok, dt, N, V, d):
    ids = torch.randint(0, V, (N,), generator=gen(N), device=DEV)
    E = torch.randn(V, d, generator=gen(d), device=DEV).to(dt)
    out = S.embed_tokens(ids, E, scale=1.7)
    want = (E[ids].float() * 1.7).to(dt)  # one product, rounded once: exact
    assert torch.equal(out, want)
    bad = torch.zeros(1, device=DEV, dtype=torch.int32)
    ids = torch.tensor([[0, -1], [V, V - 1]], device=DEV)
    out = S.embed_tokens(ids, E, bad=bad)
    assert out.shape == (2, 2, d) and bad.item() == 1 and torch.equal(out[0, 0], E[0]) and torch.equal(out[1, 1], E[V - 1])
    assert out[0, 1].abs().sum() == 0 and out[1, 0].abs().sum() == 0
    assert S.embed_tokens(ids[:0], E).shape == (0, 2, d)


def grad64(ids, dout, V, scale, skip):
    n, a, c = np.zeros((V, dout.shape[1])), np.zeros((V, dout.shape[1])), np.zeros((V, 1))
    for i, t in enumerate(ids):
        if 0 <= t < V and t != skip:
            n[t] += dout[i]
            a[t] += np.abs(dout[i])
            c[t] += 1
    return scale * n, scale * a, c


@pytest.mark.parametrize("dt,gdt", [(F32, F32), (BF16, F32), (BF16, BF16), (F32, BF16)])
@pytest.mark.parametrize("N,V,d,kind", [(0, 5, 8, "any"), (1, 1, 1, "any"), (1, 200, 768, "any"), (33, 1, 16, "any"),
                                        (31, 3, 24, "any"), (500, 40, 33, "any"), (3000, 2000, 64, "zipf"),
                                        (5000, 300, 330, "zipf"), (4096, 130, 258, "runs"), (2000, 70000, 12, "any"),
                                        (1037, 9, 768, "one"), (700, 140000, 8, "any"), (3, 1000000, 2, "any"), (300, 5, 20, "one"),
                                        (250, 70, 6, "one"), (65536, 1000, 8, "zipf"), (65537, 40000, 4, "any"),
                                        (70001, 300, 8, "zipf"), (80000, 12, 5, "one")])
def test_embed_grad(cuda_ok, dt, gdt, N, V, d, kind):
    rng = np.random.default_rng(N + V)
    if kind == "zipf":
        ids = np.minimum(rng.zipf(1.1, N) - 1, V - 1)
    elif kind == "runs":
        ids = np.repeat(rng.permutation(V), -(-N // V))[:N]  # long runs that end inside a piece
    elif kind == "one":
        ids = np.full(N, V // 2)
    else:
        ids = rng.integers(-1, V + 1, N)  # some outside the table
    t = torch.from_numpy(np.asarray(ids, np.int64)).to(DEV)
    dout = torch.randn(N, d, generator=gen(N + d), device=DEV).to(dt)
    skip = 0 if V > 3 and kind == "any" else None
    got = S.embed_grad(t, dout, V, scale=0.5, padding_id=skip, dtype=gdt)
    want, mag, cnt = grad64(ids, np64(dout), V, 0.5, -1 if skip is None else skip)
    tol = (cnt + 2) * U * mag + (H * np.abs(want) if gdt == BF16 else 0)
    assert got.dtype == gdt and (np.abs(np64(got) - want) <= tol).all()
    assert torch.equal(got, S.embed_grad(t, dout, V, scale=0.5, padding_id=skip, dtype=gdt))  # the same bits
    # onto an old gradient; from rows of a wider buffer that start off a 16-byte boundary
    old = torch.randn(V, d, generator=gen(3), device=DEV).to(gdt)
    wide = torch.zeros(N, d + 5, device=DEV, dtype=dt)
    wide[:, 1:d + 1] = dout
    acc = S.embed_grad(t, wide[:, 1:d + 1], V, scale=0.5, padding_id=skip, out=old.clone())
    w2 = want + np64(old)
    tol = (cnt + 3) * U * (mag + np.abs(np64(old))) + (H * np.abs(w2) if gdt == BF16 else 0)
    assert (np.abs(np64(acc) - w2) <= tol).all()


def test_embed_autograd(cuda_ok):
    """d/dE <embed(E), c> is linear in E: the gradient's product with E is the value itself."""
    V, d = 100, 48
    E = torch.randn(V, d, generator=gen(1), device=DEV).requires_grad_()
    ids = torch.randint(0, V, (6, 50), generator=gen(2), device=DEV)
    c = torch.randn(6, 50, d, generator=gen(3), device=DEV)
    val = (S.embed_tokens(ids, E, scale=2.0, padding_id=7) * c).sum()
    val.backward()
    keep = (ids != 7)[..., None]
    want = (2.0 * E.detach().double()[ids] * c.double() * keep).sum()
    got = (E.grad.double() * E.detach().double()).sum()
    assert abs(got - want) <= 20 * U * (2.0 * E.detach().double()[ids] * c.double()).abs().sum()
    assert E.grad[7].abs().sum() == 0


def test_offsets_beyond_32_bits(cuda_ok):
    """Rows that lie beyond 2^31 elements give what they give by themselves."""
    V, k = 32768, 5
    N = 2 ** 31 // V + 40
    x = torch.randn(N, V, generator=gen(1), device=DEV, dtype=BF16)
    last = slice(N - 7, N)
    ids = torch.randint(0, V, (N, k), generator=gen(2), device=DEV, dtype=torch.int32)
    tl = torch.randn(N, k, generator=gen(3), device=DEV)
    r = S.LogitRules(bias_ids=ids, bias_values=tl)
    y = S.process_logits(x, r)
    assert torch.equal(y[last], S.process_logits(x[last].clone(), S.LogitRules(bias_ids=ids[last], bias_values=tl[last])))
    del y
    want = S.sample_logits(x[last].clone(), temperature=0.0)[0]
    assert torch.equal(S.sample_logits(x, temperature=0.0)[0][last], want)
    l2, g2 = S.distill_loss_and_grad(x[last].clone(), ids[last], tl[last], temperature=1.5)
    l0 = S.distill_loss(x, ids, tl, temperature=1.5, reduction="none")[last]
    l1, g1 = S.distill_loss_and_grad(x, ids, tl, temperature=1.5, out=x)
    assert torch.allclose(l0, l2, rtol=PERR) and torch.allclose(l1[last], l2, rtol=PERR)
    assert torch.allclose(g1[last].float(), g2.float(), rtol=2 * H, atol=PERR)
    del x, g1
    d = 768
    N = 2 ** 31 // d + 40
    dout = torch.randn(N, d, generator=gen(4), device=DEV, dtype=BF16)
    tok = torch.zeros(N, dtype=torch.int32, device=DEV)
    tok[-3:] = 7
    tok[5] = 9
    got = S.embed_grad(tok, dout, 20)
    want = dout[-3:].float()
    assert torch.equal(got[7], want[0] + want[1] + want[2]) and torch.equal(got[9], dout[5].float())
    table = torch.randn(20, d, generator=gen(5), device=DEV).to(BF16)
    del dout
    assert torch.equal(S.embed_tokens(tok, table)[-1], table[7])


# ------------------------------------------------------------------------------------------------------- streams
def test_calls_run_on_the_current_stream(cuda_ok):
    """Each operator on a side stream, right behind work there that makes its input."""
    side = torch.cuda.Stream()
    N, V, d = 64, 4096, 256
    E = torch.randn(V, d, generator=gen(1), device=DEV)
    big = torch.randn(4096, 4096, generator=gen(2), device=DEV)
    ids = torch.randint(0, V, (N,), generator=gen(3), device=DEV, dtype=torch.int32)
    tl = torch.randn(N, 4, generator=gen(4), device=DEV)
    src = torch.randn(N, V, generator=gen(5), device=DEV)
    want = (S.process_logits(src), S.sample_logits(src, temperature=0.0)[0],
            S.distill_loss_and_grad(src, ids[:, None].expand(N, 4), tl)[1], S.embed_grad(ids, src[:, :d], V),
            S.embed_tokens(ids, E))
    torch.cuda.synchronize()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            big = big @ big * 1e-3
        x = src + 0 * big[:N, :1].nan_to_num(0, 0, 0)
        got = (S.process_logits(x), S.sample_logits(x, temperature=0.0)[0],
               S.distill_loss_and_grad(x, ids[:, None].expand(N, 4), tl)[1], S.embed_grad(ids, x[:, :d], V),
               S.embed_tokens(ids, E))
    side.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


# ----------------------------------------------------------------------------------------------- the path together
def small_model(V=500):
    torch.manual_seed(3)
    m = S.build_onesdm("onesdm_allsdm", V, dict(d=64, layers=2, mlp_f=176, heads=4, n_sub=8, d_a=8, k=4, chunk=16))
    with torch.no_grad():
        for p in m.parameters():
            if p.dim() >= 2 and float(p.abs().max()) == 0:
                torch.nn.init.normal_(p, std=0.3)
        m.emb.weight.mul_(20)
    return m.to_bf16_stream().to(DEV)


def test_generate_greedy_under_rules_that_change_nothing(cuda_ok):
    m = small_model()
    prompt = torch.randint(0, 500, (3, 20), generator=gen(1), device=DEV)
    with torch.no_grad():
        want = m.generate(prompt, 8)
        got, lp = m.generate(prompt, 8, rules=S.LogitRules(), return_logprobs=True)
        assert torch.equal(got, want) and (lp <= 0).all() and torch.isfinite(lp).all()
        assert torch.equal(m.generate(prompt, 8, rules=S.LogitRules(), use_graph=False), want)
        assert torch.equal(m.generate(prompt, 1, rules=S.LogitRules()), want[:, :1])


def test_generate_sampled(cuda_ok):
    m = small_model()
    S_, T, n, V = 5, 12, 16, 500
    prompt = torch.randint(0, V, (S_, T), generator=gen(2), device=DEV)
    u = torch.rand(S_, n, generator=gen(3), device=DEV)
    allowed = torch.zeros(2, -(-V // 32), dtype=torch.int32, device=DEV)
    allowed[0, 3] = -1  # tokens 96 .. 127
    row = torch.tensor([-1, 0, 0, 1, -1], device=DEV)
    rules = S.LogitRules(presence=1e4, mask=allowed, mask_row=row)
    kw = dict(rules=rules, u=u, temperature=0.8, top_k=40, top_p=0.9, return_logprobs=True)
    with torch.no_grad():
        a, la = m.generate(prompt, n, **kw)
        b, lb = m.generate(prompt, n, use_graph=False, **kw)
    assert torch.equal(a, b) and torch.equal(la, lb)  # a graph's steps are the same steps
    for i in (0, 1, 2, 4):
        assert len(set(a[i].tolist())) == n  # the presence penalty forbids a token twice
    assert ((a[1:3] >= 96) & (a[1:3] < 128)).all()
    assert (a[3] == -1).all() and torch.isneginf(la[3]).all()  # its mask allows nothing
    # step by step by hand: prefix logits, the same rules and numbers
    with torch.no_grad():
        logits = m(torch.cat([prompt, a[:, :4].clamp(min=0)], 1))[:, -1]
    hist = torch.cat([prompt, a[:, :4]], 1)
    r = S.LogitRules(history=hist, prompt_len=torch.full((S_,), T, device=DEV), presence=1e4, mask=allowed, mask_row=row)
    ids, _ = S.sample_logits(logits, r, u=u[:, 4], temperature=0.8, top_k=40, top_p=0.9)
    # decode and prefix logits differ by bf16 rounding, which may move a draw near a boundary: most agree
    assert (ids.long() == a[:, 4]).sum() >= S_ - 1


def test_distil_example(cuda_ok):
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "distil_on_policy.py")
    spec = importlib.util.spec_from_file_location("distil_on_policy", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    losses = mod.main(["--steps", "25", "--vocab", "512", "--d", "64", "--batch", "8", "--prompt", "8", "--new", "8"])
    assert all(np.isfinite(losses)) and np.mean(losses[-5:]) < 0.8 * np.mean(losses[:5])
