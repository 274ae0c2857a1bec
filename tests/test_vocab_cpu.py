"""Refusals of the vocabulary-end operators, without a GPU: the C entry points' status codes (nothing is launched) and
the Python checks in front of them."""
import ctypes

import pytest
import torch

import sdmchat_b200 as S
from sdmchat_b200 import _lib

FAKE = ctypes.c_void_p(0x10000)  # never dereferenced: every call below is rejected before a launch
OK, ARG, SHAPE, WORKSPACE = 0, 1, 2, 6


def rules(**kw):
    return _lib.LogitRules(**{"repetition_all": 1.0, **kw})


def test_process_refuses():
    f = _lib.lib().sdm_logits_process

    def call(r=None, x=FAKE, ld=100, rows=3, V=100, dt=0, out=ctypes.c_void_p(0x80000), ld_out=100):
        return f(r, x, ld, rows, V, dt, out, ld_out, None)

    assert call(x=None) == ARG and call(out=None) == ARG and call(dt=2) == ARG
    assert call(x=ctypes.c_void_p(0x10002)) == ARG  # a float32 pointer off its alignment
    assert call(rows=-1) == SHAPE and call(V=0) == SHAPE and call(ld=99) == SHAPE and call(ld_out=99) == SHAPE
    assert call(out=FAKE, ld=128) == ARG  # in place with another stride
    assert call(rows=1 << 40) == SHAPE
    assert call(rules(history=0x10000, history_n=4, history_ld=3)) == SHAPE
    assert call(rules(history_len=0x10000)) == ARG and call(rules(prompt_len=0x10000)) == ARG
    assert call(rules(bias_ids=0x10000, bias_n=1)) == ARG and call(rules(bias_values=0x10000, bias_n=1)) == ARG
    assert call(rules(bias_ids=0x10000, bias_values=0x10000, bias_n=1025)) == SHAPE
    assert call(rules(mask=0x10000)) == SHAPE and call(rules(mask=0x10000, mask_rows=2)) == SHAPE
    assert call(rules(mask_row=0x10000)) == ARG
    assert call(rows=0, x=None, out=None) == OK


def test_choose_refuses():
    f = _lib.lib().sdm_logits_choose
    greedy = _lib.ChoiceParams(top_p_all=1.0)

    def call(r=None, c=greedy, x=FAKE, ld=100, rows=3, V=100, dt=1, ids=FAKE):
        return f(r, c, x, ld, rows, V, dt, ids, None, None)

    assert call(c=None) == ARG and call(x=None) == ARG and call(ids=None) == ARG and call(dt=7) == ARG
    assert call(V=(1 << 18) + 1, ld=1 << 19) == SHAPE and call(ld=99) == SHAPE and call(rows=1 << 31) == SHAPE
    assert call(c=_lib.ChoiceParams(temperature_all=1.0)) == ARG  # no u
    assert call(c=_lib.ChoiceParams(temperature=0x10000)) == ARG
    assert call(c=_lib.ChoiceParams(temperature_all=-1.0, u=0x10000)) == ARG
    assert call(c=_lib.ChoiceParams(temperature_all=float("nan"), u=0x10000)) == ARG
    assert call(rows=0, x=None, ids=None) == OK


def test_distill_refuses():
    f = _lib.lib().sdm_distill

    def call(x=FAKE, ld=100, N=3, V=100, dt=1, ids=FAKE, tl=FAKE, k=4, T=1.0, a=0.5, gs=1.0, loss=FAKE, g=None, ldg=0):
        return f(x, ld, N, V, dt, ids, tl, k, None, None, None, T, a, gs, loss, g, ldg, None)

    assert call(x=None) == ARG and call(ids=None) == ARG and call(tl=None) == ARG and call(loss=None) == ARG
    assert call(dt=5) == ARG and call(x=ctypes.c_void_p(0x10001)) == ARG
    for T in (0.0, -1.0, float("inf"), float("nan")):
        assert call(T=T) == ARG
    assert call(a=float("inf")) == ARG and call(gs=float("nan")) == ARG
    assert call(k=0) == SHAPE and call(k=513) == SHAPE and call(V=(1 << 18) + 1, ld=1 << 19) == SHAPE
    assert call(ld=99) == SHAPE and call(g=ctypes.c_void_p(0x80000), ldg=99) == SHAPE
    assert call(g=FAKE, ld=128, ldg=100) == ARG
    assert call(N=0, x=None, ids=None, tl=None, loss=None) == OK
    s = _lib.lib().sdm_scale_rows
    assert s(None, 10, 2, 10, 0, FAKE, 0, None) == ARG and s(FAKE, 10, 2, 10, 0, None, 0, None) == ARG
    assert s(FAKE, 10, 2, 10, 0, FAKE, 2, None) == ARG and s(FAKE, 9, 2, 10, 0, FAKE, 1, None) == SHAPE


def test_table_refuses():
    lib = _lib.lib()
    assert lib.sdm_embed_scaled(FAKE, None, 4, 8, 10, 1.0, 0, FAKE, None, None) == ARG
    assert lib.sdm_embed_scaled(FAKE, FAKE, 4, 8, 10, 1.0, 3, FAKE, None, None) == ARG
    assert lib.sdm_embed_scaled(FAKE, FAKE, 4, 0, 10, 1.0, 0, FAKE, None, None) == SHAPE
    need = lib.sdm_embed_grad_workspace_size(1000, 64, 500)
    assert need >= 1000 * 4 + 2 * 500 * 4 + 2 * 32 * 64 * 4

    def call(ids=FAKE, dout=FAKE, ld=64, N=1000, d=64, V=500, dt=0, gdt=0, g=FAKE, ws=FAKE, nb=need):
        return lib.sdm_embed_grad(ids, dout, ld, N, d, V, 1.0, -1, dt, gdt, 0, g, ws, nb, None)

    assert call(ids=None) == ARG and call(dout=None) == ARG and call(g=None) == ARG
    assert call(dt=2) == ARG and call(gdt=2) == ARG and call(ws=ctypes.c_void_p(0x10008)) == ARG
    assert call(ld=63) == SHAPE and call(d=0) == SHAPE and call(V=(1 << 24) + 1) == SHAPE and call(N=-1) == SHAPE
    assert call(nb=need - 1) == WORKSPACE and call(ws=None) == WORKSPACE
    assert lib.sdm_embed_grad_workspace_size(-1, 64, 500) == 0


def test_python_checks_need_device_tensors():
    x = torch.zeros(2, 10)
    i = torch.zeros(2, 3, dtype=torch.int32)
    for f in (lambda: S.process_logits(x), lambda: S.sample_logits(x, temperature=0.0),
              lambda: S.distill_loss(x, i, torch.zeros(2, 3)), lambda: S.embed_tokens(i, x),
              lambda: S.embed_grad(i, torch.zeros(2, 3, 4), 10)):
        with pytest.raises(ValueError):
            f()
    with pytest.raises(ValueError):
        S.distill_loss(x, i, torch.zeros(2, 3), reduction="max")


def test_packed_structs_are_the_declared_ones():
    from sdmchat_b200 import vocab as W
    assert W._RULES.size == ctypes.sizeof(_lib.LogitRules) and W._CHOICE.size == ctypes.sizeof(_lib.ChoiceParams)
    vals = list(range(1, 18))
    r = _lib.LogitRules.from_buffer_copy(W._RULES.pack(*vals))
    assert [getattr(r, n) for n, _ in r._fields_] == vals
    c = _lib.ChoiceParams.from_buffer_copy(W._CHOICE.pack(*vals[:7]))
    assert [getattr(c, n) for n, _ in c._fields_] == vals[:7]


def test_python_checks_of_rules():
    """Shapes, types and pairs are looked at before any pointer is taken (host tensors stand in)."""
    i, f = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3)
    for kw in (dict(history=i[:2]), dict(history=i.float()), dict(history_len=i[:, 0]), dict(prompt_len=i[:, 0]),
               dict(bias_ids=i), dict(bias_values=torch.zeros(3, 4)), dict(bias_ids=i, bias_values=torch.zeros(3, 5)),
               dict(mask=torch.zeros(1, 3, dtype=torch.int32)), dict(mask=torch.zeros(2, 4, dtype=torch.int32)),
               dict(mask_row=i[:, 0]), dict(repetition=f[:2]), dict(frequency=i)):
        with pytest.raises((ValueError, TypeError)):
            S.LogitRules(**kw)._struct(3, 100, -1, [])
