"""Arguments at the ends of their ranges: the vocabulary-end operators on the GPU against plain computations."""
import math

import pytest
import torch

import sdmchat_b200 as S

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("V", [50, 3000, 40000])
@pytest.mark.parametrize("rows", [2, 200])
@pytest.mark.parametrize("T", [3e38, math.inf])
def test_temperature_without_end(cuda_ok, V, rows, T):
    """All tokens that are not at -infinity are alike: u picks among the kept ones by their number."""
    g = torch.Generator(device=DEV).manual_seed(V)
    x = torch.randn(rows, V, generator=g, device=DEV)
    x[:, ::3] = -math.inf
    u = torch.rand(rows, generator=g, device=DEV)
    n = V - len(range(0, V, 3))
    for kw in ({}, dict(top_k=5), dict(top_k=n // 2), dict(top_p=0.5), dict(top_k=20, top_p=0.375)):
        k = kw.get("top_k", n)
        m = math.ceil(k * kw.get("top_p", 1.0))
        for temperature in (T, torch.full((rows,), T, device=DEV)):
            ids, lp = S.sample_logits(x, u=u, temperature=temperature, **kw)
            assert torch.allclose(lp, torch.full_like(lp, -math.log(m)), atol=16 * 2.0 ** -24 * (1 + math.log(m)))
            keep = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :m].sort(1).values
            at = (u.double() * m).long().clamp(max=m - 1)
            assert torch.equal(ids.long(), keep.gather(1, at[:, None])[:, 0])


def test_host_threads_at_different_sizes(cuda_ok):
    """Two host threads launch the same kernel on streams of their own, one over a vocabulary that takes little shared
    memory and one over one that takes much: no launch may be refused.  The calls are made at the C entry point, so
    that the threads meet in it."""
    import threading

    from sdmchat_b200 import _lib
    lib = _lib.lib()
    greedy = _lib.ChoiceParams(top_p_all=1.0)

    def work(V, seed, results):
        x = torch.randn(1, V, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)
        ids = torch.full((1,), -7, device=DEV, dtype=torch.int32)
        torch.cuda.synchronize()
        st = torch.cuda.Stream()
        args = (None, greedy, _lib.ptr(x), V, 1, V, 0, _lib.ptr(ids), None, _lib.c_void_p(st.cuda_stream))
        refused = sum(lib.sdm_logits_choose(*args) != 0 for _ in range(20000))
        st.synchronize()
        results.append((refused, int(ids.item()) == int(x.argmax())))

    results = []
    threads = [threading.Thread(target=work, args=(V, V, results)) for V in (70000, 200000)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert results == [(0, True), (0, True)], results


def test_ids_beyond_32_bits(cuda_ok):
    """Ids that a 64-bit tensor holds and 32 bits do not are outside every table."""
    far = [2 ** 32 + 5, -2 ** 32 + 5, 2 ** 31 + 5]
    ids = torch.tensor(far + [3], device=DEV)
    table = torch.randn(10, 4, device=DEV)
    bad = torch.zeros(1, device=DEV, dtype=torch.int32)
    out = S.embed_tokens(ids, table, bad=bad)
    assert bad.item() == 1 and (out[:3] == 0).all() and torch.equal(out[3], table[3])
    grad = S.embed_grad(ids, torch.ones(4, 4, device=DEV), 10)
    assert grad.sum() == 4 and (grad[3] == 1).all()
    for skip in (2 ** 32 + 3, -2 ** 32 + 3, 10, -1):  # no token of the table: nothing is skipped
        assert torch.equal(S.embed_grad(ids, torch.ones(4, 4, device=DEV), 10, padding_id=skip), grad)
    x = torch.randn(1, 10, device=DEV)
    far = torch.tensor([far], device=DEV)
    assert torch.equal(S.process_logits(x, S.LogitRules(history=far, presence=1.0)), x)
    assert torch.equal(S.process_logits(x, S.LogitRules(bias_ids=far, bias_values=torch.ones(1, 3, device=DEV))), x)
    tl = torch.zeros(1, 3, device=DEV)
    loss, dx = S.distill_loss_and_grad(x, far, tl, targets=far[:, 0], alpha=0.5)
    assert loss.item() == 0 and (dx == 0).all()
    ids, _ = S.sample_logits(x, u=torch.tensor([0.999], device=DEV), top_k=torch.tensor([2 ** 32 + 1], device=DEV))
    assert ids.item() == S.sample_logits(x, u=torch.tensor([0.999], device=DEV))[0].item()


def test_outputs_in_place_are_seen_by_autograd(cuda_ok):
    """A tensor that a graph saved and an operator then wrote over makes the backward pass raise, as torch's own do."""
    ids = torch.zeros(3, 2, device=DEV, dtype=torch.int32)
    tl = torch.zeros(3, 2, device=DEV)
    tok = torch.zeros(4, device=DEV, dtype=torch.int32)
    for write in (lambda x: S.process_logits(x, out=x), lambda x: S.distill_loss_and_grad(x, ids, tl, out=x),
                  lambda x: S.embed_grad(tok, torch.ones(4, 8, device=DEV), 3, out=x)):
        leaf = torch.randn(3, 8, device=DEV, requires_grad=True)
        x = leaf * 2
        y = (x * x).sum()  # saves x
        write(x.detach())
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
        with torch.inference_mode():  # whose tensors' versions nobody reads
            write(torch.randn(3, 8, device=DEV))
