"""Distillation where logits leave the range that one base can serve: rows partly masked with finite lowest values,
rows that lie far from zero as a whole, and students whose listed tokens lead all others by more than an exponential
spans.  The loss alone, the loss with its gradient and 64 bits have to agree, in every kernel (blocks and clusters of
blocks per row, persistent blocks, the loss alone).

Tolerances are those of the operator's other tests: a probability is off by 100 u of its own value (|d| * 2 u for the
roundings of an exponent d of magnitude up to 40, 4 u for the exponential, the rest for sums and quotients), a
logarithm by 100 u of its magnitude, one rounding to bfloat16 by 2^-8 of the value."""
import math

import pytest
import torch

import sdmchat_b200 as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
U, H = 2.0 ** -24, 2.0 ** -8
PERR = 100 * U
F32, BF16 = torch.float32, torch.bfloat16


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def reference(x, ids, tl, tg, T, a, lse):
    """(loss, gradient, their magnitudes for the rounding bounds) of all rows in 64 bits; distinct entries per row."""
    x, tl = x.double(), tl.double()
    N, V = x.shape
    ok, at = ids >= 0, ids.clamp(min=0).long()
    some = ok.any(1)
    zt = (tl / T).masked_fill(~ok, -math.inf)
    norm = torch.logsumexp(zt, 1) if lse is None else lse.double()
    lp = torch.where(ok, zt - torch.where(some, norm, 0.0)[:, None], 0.0)
    p = torch.where(ok, lp.exp(), 0.0)
    P = p.sum(1)
    lq = torch.log_softmax(x / T, 1)
    lqa = lq.gather(1, at)
    part = torch.where(ok, p * (lp - lqa), 0.0).sum(1)
    lm = torch.where(ok, p * (lp.abs() + lqa.abs() + 1), 0.0).sum(1)
    pr = torch.zeros_like(P)
    q = lq.exp() * some[:, None]
    listed = torch.zeros(N, V + 1, dtype=torch.bool, device=x.device)
    listed.scatter_(1, torch.where(ok, at, V), True)
    listed = listed[:, :V]
    G = torch.zeros_like(x)
    M = torch.zeros_like(x)
    if lse is not None:
        pr = torch.where(some, (1 - P).clamp(min=0), 0.0)
        lr = torch.logsumexp(lq.masked_fill(listed, -math.inf), 1)  # log of the student's mass that is not listed
        part = part + torch.where(pr > 0, pr * (pr.clamp(min=1e-300).log() - lr), 0.0)
        lm = lm + torch.where(pr > 0, (P + 1) * (pr.clamp(min=1e-300).log().abs() + lr.abs() + 1), 0.0)
        share = torch.softmax((x / T).masked_fill(listed, -math.inf), 1) * (pr > 0)[:, None]
        G, M = G - pr[:, None] * share, M + (pr + 1)[:, None] * share
    mass = (P + pr)[:, None]
    G, M = G + mass * q, M + mass * q
    G, M = G.scatter_add(1, at, -p), M.scatter_add(1, at, p)
    loss, lm, G, M = a * T * T * part, a * T * T * lm, a * T * G, a * T * M
    if tg is not None:
        hit, t = tg >= 0, tg.clamp(min=0).long()[:, None]
        l1 = torch.log_softmax(x, 1)
        lt = torch.where(hit, l1.gather(1, t)[:, 0], 0.0)
        one = (1 - a) * hit[:, None].double()
        loss, lm = loss - (1 - a) * lt, lm + (1 - a) * hit * (lt.abs() + 1)
        G, M = G + one * l1.exp(), M + one * l1.exp()
        G, M = G.scatter_add(1, t, -one), M.scatter_add(1, t, one)
    return loss, G, lm, M


def check(x, ids, tl, tg, T, a, lse, with_loss=True):
    loss, grad = S.distill_loss_and_grad(x, ids, tl, tg, T, a, None, lse)
    only = S.distill_loss(x, ids, tl, tg, T, a, None, lse, reduction="none")
    want, G, lm, M = reference(x, ids, tl, tg, T, a, lse)
    bad = ~((only - want).abs() <= PERR * lm + 1e-30) & with_loss
    assert not bad.any(), ("loss alone", bad.nonzero()[:5].tolist(), only[bad][:5], want[bad][:5])
    bad = ~((loss - want).abs() <= PERR * lm + 1e-30) & with_loss
    assert not bad.any(), ("loss", bad.nonzero()[:5].tolist(), loss[bad][:5], want[bad][:5])
    tol = PERR * M + (H * G.abs() if x.dtype == BF16 else 0) + 1e-37
    bad = ~((grad.double() - G).abs() <= tol)
    assert not bad.any(), ("gradient", bad.nonzero()[:5].tolist(), grad[bad][:5], G[bad][:5])
    over = x.clone()  # over the logits
    again = S.distill_loss_and_grad(over, ids, tl, tg, T, a, None, lse, out=over)
    assert torch.equal(again[0], loss) and torch.equal(over, grad)
    # rows at every kind of address, the gradient's at another
    N, V = x.shape
    wide, out = torch.zeros(N, V + 9, device=DEV, dtype=x.dtype), torch.zeros(N, V + 6, device=DEV, dtype=x.dtype)
    wide[:, 3:V + 3] = x
    S.distill_loss_and_grad(wide[:, 3:V + 3], ids, tl, tg, T, a, None, lse, out=out[:, 5:V + 5])
    bad = ~((out[:, 5:V + 5].double() - G).abs() <= tol)
    assert not bad.any(), ("gradient off 16 bytes", bad.nonzero()[:5].tolist())
    assert (out[:, :5] == 0).all() and (out[:, V + 5:] == 0).all()


# rows and vocabularies: a cluster of eight blocks per row, of two to four, a block per row, persistent blocks
SHAPES = [(12, 1000), (12, 50021), (48, 2053), (240, 2053), (624, 517), (624, 14003), (624, 28001)]


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("N,V", SHAPES)
@pytest.mark.parametrize("T", [0.5, 1.0, 1.5, 2.0, 4.0])
def test_rows_far_from_zero(cuda_ok, dt, N, V, T):
    """Whole rows at or around one value of every magnitude."""
    g = gen(N + V + 1)
    k = 5
    base = torch.tensor([-1e30, -1e10, -1e20, 1e10, -3e9, 3e5, -6e5, 8e5, -1e6, 3e6, -1e7, 1e30], device=DEV)
    at = base[torch.arange(N, device=DEV) % 12][:, None]
    spread = torch.where(at.abs() < 2e7, torch.randn(N, V, generator=g, device=DEV) * 2, 0.0)
    x = (at + spread).to(dt)
    x[::5, 3] *= 1 + 2.0 ** -6  # one token of some rows apart
    ids = torch.stack([torch.randperm(V, generator=g, device=DEV)[:k] for _ in range(N)]).to(torch.int32)
    hot = x.argmax(1).to(torch.int32)
    lead = x.max(1).values > x.min(1).values  # rows that are not level: the teacher lists tokens near the largest
    near = (x >= x.max(1, keepdim=True).values - 20).float()
    ids = torch.where(lead[:, None], torch.multinomial(near, 1).to(torch.int32), ids)
    ids[lead, 1:] = -1
    tg = torch.where(lead, hot, ids[:, 0])
    tl = torch.randn(N, k, generator=g, device=DEV)
    for hard in (False, True):
        check(x, ids, tl, tg if hard else None, T, 0.6, None)
    # the rest of the teacher's mass, where a token that is not listed shares it with the largest
    level = ~lead
    lse = torch.logsumexp((tl / T).masked_fill(ids < 0, -math.inf), 1) + 0.3
    for hard in (False, True):
        check(x[level], ids[level], tl[level], tg[level] if hard else None, T, 0.6, lse[level])


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("N,V", SHAPES)
@pytest.mark.parametrize("T", [0.5, 1.0, 1.5, 2.0, 4.0])
def test_partly_masked_rows(cuda_ok, dt, N, V, T):
    """1, 8, 64 and most of a row's tokens are ordinary, at its beginning, its end, side by side inside or anywhere;
    the others hold a mask's finite lowest value."""
    g = gen(N + V)
    k = 5
    x = torch.empty(N, V, device=DEV)
    ids = torch.full((N, k), -1, device=DEV, dtype=torch.int32)
    tg = torch.empty(N, device=DEV, dtype=torch.int32)
    one = torch.zeros(N, device=DEV, dtype=torch.bool)
    lowest = [torch.finfo(dt).min, -1e30, -1e20, -1e10]
    order = torch.randperm(48 * (1 + N // 48), generator=g, device=DEV).tolist()
    for i in range(N):
        c = order[i] % 48
        n = (1, 8, 64, V - 100)[c % 4]
        start = {0: 0, 1: V - n, 2: (V - n) // 2 // 8 * 8}.get(c // 4 % 3, 0)
        at = torch.arange(start, start + n, device=DEV)
        if c % 7 == 3:
            at = torch.randperm(V, generator=g, device=DEV)[:n]
        x[i] = lowest[c // 12]
        x[i, at] = 2 * torch.randn(n, generator=g, device=DEV)
        some = at[torch.randperm(n, generator=g, device=DEV)[:k]]
        m = min(k, n)
        ids[i, :m] = some[:m].to(torch.int32)
        tg[i] = at[n // 2]
        one[i] = n == 1
    x = x.to(dt)
    tl = torch.randn(N, k, generator=g, device=DEV)
    for hard in (False, True):
        for tail in (False, True):
            e = ids.masked_fill(one[:, None], -1) if tail else ids  # the rest of the mass needs a token to go to
            lse = None
            if tail:
                lse = torch.logsumexp((tl / T).masked_fill(e < 0, -math.inf), 1).nan_to_num(neginf=0.0) + 0.3
            check(x, e, tl, tg if hard else None, T, 0.6, lse)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("N,V", SHAPES)
@pytest.mark.parametrize("T", [0.7, 1.0, 1.5, 2.0, 4.0])
def test_listed_tokens_lead(cuda_ok, dt, N, V, T):
    """The teacher's remaining mass where the student gives the tokens that are not listed next to nothing."""
    g = gen(N + V + 2)
    k = 5
    x = torch.randn(N, V, generator=g, device=DEV)
    ids = torch.stack([torch.randperm(V, generator=g, device=DEV)[:k] for _ in range(N)]).to(torch.int32)
    gap = torch.tensor([0.0, 20.0, 50.0, 61.0, 86.0, 100.0, 150.0, 300.0, 600.0, 1e4], device=DEV)
    gap = gap[torch.arange(N, device=DEV) % 10]
    far = torch.tensor([0.0, -1e6, 0.0], device=DEV)[torch.arange(N, device=DEV) % 3]  # rows far from zero among them
    x.scatter_(1, ids[:, :3].long(), gap[:, None] + torch.randn(N, 3, generator=g, device=DEV))
    x = (x + far[:, None]).to(dt)
    tl = torch.randn(N, k, generator=g, device=DEV)
    tg = torch.randint(0, V, (N,), generator=g, device=DEV, dtype=torch.int32)
    tg = torch.where(torch.arange(N, device=DEV) % 2 == 0, ids[:, 0], tg)
    lse = torch.logsumexp(tl / T, 1) + 0.3
    for hard in (False, True):
        check(x, ids, tl, tg if hard else None, T, 0.6, lse)
    # the others at a mask's finite lowest value (finfo.min times 1 / T and log2(e) is beyond float32: the loss is infinite)
    others = torch.ones(N, V, device=DEV, dtype=torch.bool).scatter_(1, ids.long(), False)
    for low in (-1e10, -1e20, torch.finfo(dt).min):
        y = torch.randn(N, V, generator=g, device=DEV).masked_fill(others, low).to(dt)
        tg = torch.where(torch.arange(N, device=DEV) % 2 == 0, ids[:, 0], -1)
        for hard in (False, True):
            check(y, ids, tl, tg if hard else None, T, 0.6, lse, with_loss=low > -1e30)
    # nothing but listed tokens is possible: the loss is infinite, and the others, at -infinity, have no gradient
    listed = torch.zeros(N, V, device=DEV, dtype=torch.bool).scatter_(1, ids.long(), True)
    y = x.masked_fill(~listed, -math.inf)
    loss, grad = S.distill_loss_and_grad(y, ids, tl, None, T, 0.6, None, lse)
    only = S.distill_loss(y, ids, tl, None, T, 0.6, None, lse, reduction="none")
    assert torch.isposinf(loss).all() and torch.isposinf(only).all()
    assert torch.isfinite(grad).all() and (grad[~listed] == 0).all()


@pytest.mark.parametrize("dt,V,T", [(BF16, 32768, 2.0), (BF16, 20000, 2.0), (F32, 8192, 1.5)])
def test_rows_without_weight_are_not_read(cuda_ok, dt, V, T):
    """Of rows without weight only the gradient's zeros move: half the bytes of a copy of the logits, which takes the
    memory 8,192 rows of 40 KB and more long enough to be measured."""
    N = 8192 * 32768 // V
    x = torch.zeros(N, V, device=DEV, dtype=dt)
    ids, tl = torch.zeros(N, 4, device=DEV, dtype=torch.int32), torch.zeros(N, 4, device=DEV)
    w, out = torch.zeros(N, device=DEV), torch.ones_like(x)

    def best(f):
        t = []
        for _ in range(8):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            f()
            b.record()
            b.synchronize()
            t.append(a.elapsed_time(b))
        return min(t)

    tg = torch.zeros(N, device=DEV, dtype=torch.int32)
    mine = best(lambda: S.distill_loss_and_grad(x, ids, tl, tg, T, 0.5, w, out=out))
    assert torch.count_nonzero(out) == 0
    copy = best(lambda: out.copy_(x))
    assert mine < 0.85 * copy, (mine, copy)
