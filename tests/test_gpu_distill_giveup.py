"""The persistent distillation kernel under a wait limit of a nanosecond: waits that do not find their row or buffer at
once give up.  The kernel has to end, sdm_device_status to tell whether a wait gave up, rows that were not finished to
have a NaN loss, and the next call under the default limit to be right."""
import pytest
import torch

import sdmchat_b200 as S
from sdmchat_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
SDM_OK, SDM_ERR_TIMEOUT = 0, 4


@pytest.mark.parametrize("dt,V", [(torch.float32, 14003), (torch.bfloat16, 30005)])
@pytest.mark.parametrize("tail", [False, True])
def test_waits_that_give_up(cuda_ok, dt, V, tail):
    N, k = 2000, 9
    g = torch.Generator(device=DEV).manual_seed(V)
    x = (3 * torch.randn(N, V, generator=g, device=DEV)).to(dt)
    ids = torch.stack([torch.randperm(V, generator=g, device=DEV)[:k] for _ in range(N)]).to(torch.int32)
    tl = torch.randn(N, k, generator=g, device=DEV)
    tg = torch.randint(-1, V, (N,), generator=g, device=DEV, dtype=torch.int32)
    w = (torch.rand(N, generator=g, device=DEV) > 0.3).float()
    lse = torch.logsumexp(tl / 2, 1) + 0.3 if tail else None
    lib, st = _lib.lib(), _lib.stream_ptr()
    want, dwant = S.distill_loss_and_grad(x, ids, tl, tg, 2.0, 0.5, w, lse)
    assert lib.sdm_device_status(st) == SDM_OK
    _lib.check(lib.sdm_set_wait_limit_ns(1), "sdm_set_wait_limit_ns")
    try:
        loss, grad = S.distill_loss_and_grad(x, ids, tl, tg, 2.0, 0.5, w, lse)
        status = lib.sdm_device_status(st)  # synchronises: the kernel has ended
    finally:
        _lib.check(lib.sdm_set_wait_limit_ns(0), "sdm_set_wait_limit_ns")
    assert status in (SDM_OK, SDM_ERR_TIMEOUT) and lib.sdm_device_status(st) == SDM_OK
    done = ~torch.isnan(loss)
    assert torch.equal(loss[done], want[done]) and torch.equal(grad[done], dwant[done])
    assert done.all() or status == SDM_ERR_TIMEOUT
    print(int(done.sum()), "of", N, "rows finished, status", status)
    loss, grad = S.distill_loss_and_grad(x, ids, tl, tg, 2.0, 0.5, w, lse)
    assert torch.equal(loss, want) and torch.equal(grad, dwant) and lib.sdm_device_status(st) == SDM_OK
