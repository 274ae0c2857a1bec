"""The vocabulary end of a language model on libsdm_b200: rules on logits and the choice of a token (serving), the
distillation loss and the token table's lookup with their gradients (training).

Tensors are on a CUDA device, in float32 or bfloat16 (ids int32; other integer types are converted); every call runs
on the current stream of its tensors' device.  `distill_loss` and `embed_tokens` record autograd; the other functions
are forward only.  There is no CPU or PyTorch fallback.
"""
import dataclasses
from typing import Optional, Union

import torch

from . import _lib as L_
from ._lib import check, lib, ptr, stream_ptr, workspace, dtype_code

Per = Union[float, torch.Tensor]  # one value for all rows, or one per row


def _device(t, name):
    if not t.is_cuda:
        raise ValueError(f"{name}: libsdm_b200 takes device tensors only")
    return t.device


def _on(t, dev, name, dtype, shape):
    """t as a contiguous tensor of dtype on dev with the given shape (None: any size)."""
    if t is None:
        return None
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, the logits or ids on {dev}")
    if t.dim() != len(shape) or any(w is not None and n != w for n, w in zip(t.shape, shape)):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, wanted {tuple('any' if w is None else w for w in shape)}")
    if dtype == torch.int32 and (t.dtype.is_floating_point or t.dtype.is_complex):
        raise TypeError(f"{name} holds whole numbers, not {t.dtype}")
    return t.detach().to(dtype).contiguous()


def _rows(t, name):
    """t (N, V) with contiguous rows, and its row stride."""
    if t.dim() != 2:
        raise ValueError(f"{name} is 2-D (rows, vocabulary), not {t.dim()}-D")
    dtype_code(t.dtype)
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t, (t.stride(0) if t.shape[0] > 1 else t.shape[1])


def _out_rows(out, like, name):
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
        raise ValueError(f"{name} has the shape, dtype and device of the logits")
    if out.shape[1] > 1 and out.stride(1) != 1 or out.shape[0] > 1 and out.stride(0) < out.shape[1]:
        raise ValueError(f"{name} needs contiguous rows that do not overlap")
    if out.data_ptr() != like.data_ptr() and out.untyped_storage().data_ptr() == like.untyped_storage().data_ptr():
        span = lambda t: (t.data_ptr(), t.data_ptr() + ((t.shape[0] - 1) * t.stride(0) + t.shape[1]) * t.element_size())  # noqa: E731
        (a0, a1), (b0, b1) = span(out), span(like)
        if a0 < b1 and b0 < a1:
            raise ValueError(f"{name} overlaps the logits without being them")
    return out


def _per(v, dev, name, dtype, S):
    """(tensor or None, value for all rows) of a per-row parameter."""
    if isinstance(v, torch.Tensor):
        return _on(v, dev, name, dtype, (S,)), 0
    return None, v


@dataclasses.dataclass
class LogitRules:
    """What a serving loop knows about each of S rows of logits (struct sdm_logit_rules; everything is optional).

    history (S, L): the row's tokens so far, prompt first, padded with -1 or cut by history_len (S); prompt_len (S):
    where the generated ones begin (default 0: all were generated).  A token of the history has its logit divided
    (positive) or multiplied (else) by `repetition`; one generated g times loses frequency * g and `presence`.
    bias_ids, bias_values (S, n): added to the logits of those tokens (-1: unused entry).  mask (G, ceil(V / 32))
    int32: bit v % 32 of word v / 32 allows token v; row s is under mask mask_row[s] (-1: none), or under mask s
    (mask 0 if there is one) without mask_row.  Others become -infinity."""
    history: Optional[torch.Tensor] = None
    history_len: Optional[torch.Tensor] = None
    prompt_len: Optional[torch.Tensor] = None
    repetition: Per = 1.0
    frequency: Per = 0.0
    presence: Per = 0.0
    bias_ids: Optional[torch.Tensor] = None
    bias_values: Optional[torch.Tensor] = None
    mask: Optional[torch.Tensor] = None
    mask_row: Optional[torch.Tensor] = None

    def _struct(self, S, V, dev):
        """(sdm_logit_rules, the tensors it points to)."""
        i32, f32 = torch.int32, torch.float32
        hist = _on(self.history, dev, "history", i32, (S, None))
        hl = _on(self.history_len, dev, "history_len", i32, (S,))
        pl = _on(self.prompt_len, dev, "prompt_len", i32, (S,))
        if hist is None and (hl is not None or pl is not None):
            raise ValueError("history_len and prompt_len need a history")
        if hist is not None and hist.shape[1] == 0:
            hist = hl = pl = None
        if (self.bias_ids is None) != (self.bias_values is None):
            raise ValueError("bias_ids and bias_values come together")
        bi = _on(self.bias_ids, dev, "bias_ids", i32, (S, None))
        bv = _on(self.bias_values, dev, "bias_values", f32, (S, None if bi is None else bi.shape[1]))
        mask = _on(self.mask, dev, "mask", i32, (None, -(-V // 32)))
        mr = _on(self.mask_row, dev, "mask_row", i32, (S,))
        if mask is None and mr is not None:
            raise ValueError("mask_row needs a mask")
        if mask is not None and mr is None and mask.shape[0] not in (1, S):
            raise ValueError(f"{mask.shape[0]} masks for {S} rows need mask_row")
        rep, rep_all = _per(self.repetition, dev, "repetition", f32, S)
        frq, frq_all = _per(self.frequency, dev, "frequency", f32, S)
        prs, prs_all = _per(self.presence, dev, "presence", f32, S)
        keep = (hist, hl, pl, rep, frq, prs, bi, bv, mask, mr)
        r = L_.LogitRules(
            history=ptr(hist), history_ld=0 if hist is None else hist.shape[1],
            history_n=0 if hist is None else hist.shape[1], history_len=ptr(hl), prompt_len=ptr(pl),
            repetition=ptr(rep), frequency=ptr(frq), presence=ptr(prs), repetition_all=rep_all,
            frequency_all=frq_all, presence_all=prs_all, bias_ids=ptr(bi), bias_values=ptr(bv),
            bias_n=0 if bi is None else bi.shape[1], mask=ptr(mask), mask_rows=0 if mask is None else mask.shape[0],
            mask_row=ptr(mr))
        return r, keep


def process_logits(logits, rules=None, out=None):
    """The rules on logits (S, V), in their dtype (rounded once): penalties, biases, then the mask (sdm_logits_process).
    out: where to write (the logits themselves are allowed), else a new tensor."""
    dev = _device(logits, "logits")
    x, ld = _rows(logits.detach(), "logits")
    S, V = x.shape
    out = torch.empty(S, V, dtype=x.dtype, device=dev) if out is None else _out_rows(out, logits, "out")
    r, keep = (rules or LogitRules())._struct(S, V, dev)
    with torch.cuda.device(dev):
        check(lib().sdm_logits_process(r, ptr(x), ld, S, V, dtype_code(x.dtype), ptr(out),
                                       out.stride(0) if S > 1 else V, stream_ptr(dev)), "sdm_logits_process")
    return out


def sample_logits(logits, rules=None, u=None, temperature: Per = 1.0, top_k: Union[int, torch.Tensor] = 0,
                  top_p: Per = 1.0):
    """One token per row of logits (S, V) under the rules: ids (S,) int32 and log-probabilities (S,) float32 under the
    distribution drawn from (sdm_logits_choose).  u (S,) in [0, 1) picks the token: with the kept tokens in index
    order, the first whose running probability exceeds it.  temperature 0 takes the largest logit (u may be None if
    that is so for all rows).  A row that allows no token gives -1 and -infinity."""
    dev = _device(logits, "logits")
    x, ld = _rows(logits.detach(), "logits")
    S, V = x.shape
    r, keep = (rules or LogitRules())._struct(S, V, dev)
    f32 = torch.float32
    tt, t_all = _per(temperature, dev, "temperature", f32, S)
    tk, k_all = _per(top_k, dev, "top_k", torch.int32, S)
    tp, p_all = _per(top_p, dev, "top_p", f32, S)
    u = _on(u, dev, "u", f32, (S,))
    if u is None and (tt is not None or t_all != 0):
        raise ValueError("sampling needs u, one number in [0, 1) per row")
    c = L_.ChoiceParams(temperature=ptr(tt), top_k=ptr(tk), top_p=ptr(tp), u=ptr(u), temperature_all=t_all,
                        top_p_all=p_all, top_k_all=k_all)
    ids = torch.empty(S, dtype=torch.int32, device=dev)
    lp = torch.empty(S, dtype=f32, device=dev)
    with torch.cuda.device(dev):
        check(lib().sdm_logits_choose(r, c, ptr(x), ld, S, V, dtype_code(x.dtype), ptr(ids), ptr(lp),
                                      stream_ptr(dev)), "sdm_logits_choose")
    return ids, lp


# -------------------------------------------------------------------------------------------------- distillation
def _distill(logits, teacher_ids, teacher_logits, targets, temperature, alpha, row_weight, teacher_lse, grad_scale,
             want_grad, out=None):
    dev = _device(logits, "logits")
    x, ld = _rows(logits.detach(), "logits")
    N, V = x.shape
    ids = _on(teacher_ids, dev, "teacher_ids", torch.int32, (N, None))
    tl = _on(teacher_logits, dev, "teacher_logits", torch.float32, (N, ids.shape[1]))
    tg = _on(targets, dev, "targets", torch.int32, (N,))
    w = _on(row_weight, dev, "row_weight", torch.float32, (N,))
    lse = _on(teacher_lse, dev, "teacher_lse", torch.float32, (N,))
    loss = torch.empty(N, dtype=torch.float32, device=dev)
    grad = None
    if want_grad:
        grad = torch.empty(N, V, dtype=x.dtype, device=dev) if out is None else _out_rows(out, logits, "out")
    with torch.cuda.device(dev):
        check(lib().sdm_distill(ptr(x), ld, N, V, dtype_code(x.dtype), ptr(ids), ptr(tl), ids.shape[1], ptr(lse),
                                ptr(tg), ptr(w), temperature, alpha, grad_scale, ptr(loss), ptr(grad),
                                0 if grad is None else (grad.stride(0) if N > 1 else V), stream_ptr(dev)), "sdm_distill")
    return loss, grad


def distill_loss_and_grad(logits, teacher_ids, teacher_logits, targets=None, temperature=1.0, alpha=1.0,
                          row_weight=None, teacher_lse=None, grad_scale=1.0, out=None):
    """Per-row distillation losses (N,) float32 and grad_scale times their sum's gradient by the logits, in the
    logits' dtype, from one pass over the logits.  out: where the gradient goes (the logits themselves are allowed).
    See distill_loss for the rest."""
    return _distill(logits, teacher_ids, teacher_logits, targets, temperature, alpha, row_weight, teacher_lse,
                    grad_scale, True, out)


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, args, scale):
        loss, grad = _distill(logits, *args, scale, True)
        ctx.save_for_backward(grad)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        (grad,) = ctx.saved_tensors
        N, V = grad.shape
        one = N > 0 and g.stride(0) == 0  # a sum's or mean's factor: one number for all rows
        g = (g[:1] if one else g).float().contiguous()
        if ctx.needs_input_grad[0] and N > 0:
            if getattr(ctx, "used", False):
                raise RuntimeError("the gradient was formed with the loss and handed out by the first backward pass")
            ctx.used = True
            with torch.cuda.device(grad.device):
                check(lib().sdm_scale_rows(ptr(grad), V, N, V, dtype_code(grad.dtype), ptr(g), 0 if one else 1,
                                           stream_ptr(grad.device)), "sdm_scale_rows")
        return grad, None, None


def distill_loss(logits, teacher_ids, teacher_logits, targets=None, temperature=1.0, alpha=1.0, row_weight=None,
                 teacher_lse=None, reduction="mean"):
    """Distillation of a student's logits (N, V) from a teacher's k top logits per row (sdm_distill):
    row_weight * (alpha * T^2 * KL(p | softmax(logits / T)) + (1 - alpha) * cross-entropy against targets).

    teacher_ids, teacher_logits (N, k): the teacher's tokens and their logits; an id outside the vocabulary (-1) or a
    logit of -infinity is an unused entry.  p is their softmax at T; with teacher_lse (N,), the teacher's log-sum-exp
    at T over its whole vocabulary, p is exact and the mass of the tokens not listed counts as one event.  targets
    (N,), -1 for none.  row_weight (N,): a row of weight 0 is not read.  reduction: "none" (N,), "sum", or "mean" (the
    sum over N).

    Differentiable by the logits: with autograd recording, the gradient is formed with the loss in the same pass over
    the logits and kept for the backward pass, which is free for "sum" and "mean" used as the loss itself; it can be
    run once."""
    if reduction not in ("none", "sum", "mean"):
        raise ValueError(f"reduction is none, sum or mean, not {reduction!r}")
    args = (teacher_ids, teacher_logits, targets, temperature, alpha, row_weight, teacher_lse)
    N = logits.shape[0]
    scale = 1.0 / N if reduction == "mean" and N > 0 else 1.0
    if torch.is_grad_enabled() and logits.requires_grad:
        loss = _DistillLoss.apply(logits, args, scale)
        return loss if reduction == "none" else _ScaledSum.apply(loss, scale)
    loss, _ = _distill(logits, *args, 1.0, False)
    return loss if reduction == "none" else loss.sum() * scale


class _ScaledSum(torch.autograd.Function):
    """scale * sum(loss) over rows whose gradient already holds the scale."""

    @staticmethod
    def forward(ctx, loss, scale):
        ctx.n = loss.shape[0]
        return loss.sum() * scale

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        return g.expand(ctx.n), None


# ------------------------------------------------------------------------------------------------- token table
def _ids32(ids):
    _device(ids, "ids")
    if ids.dtype.is_floating_point or ids.dtype.is_complex or ids.dtype == torch.bool:
        raise TypeError(f"ids are whole numbers, not {ids.dtype}")
    return ids.detach().to(torch.int32).contiguous()


def embed_grad(ids, dout, num_rows, scale=1.0, padding_id=None, dtype=torch.float32, out=None):
    """The token table's gradient (num_rows, d): scale times the sum of dout (..., d) over the positions of each id
    (sdm_embed_grad).  ids outside the table and padding_id are skipped.  out: a gradient (num_rows, d), float32 or
    bfloat16, to add to; else a new one of `dtype`.  The same inputs give the same bits."""
    i32 = _ids32(ids)
    dev = i32.device
    if dout.device != dev or dout.shape[:-1] != ids.shape:
        raise ValueError(f"dout {tuple(dout.shape)} on {dout.device} does not go with ids {tuple(ids.shape)} on {dev}")
    d = dout.shape[-1]
    N = i32.numel()
    g = dout.detach()
    if g.dim() != 2 or g.stride(1) != 1 or g.stride(0) < d:
        g = g.reshape(N, d).contiguous()
    if out is not None and (out.shape != (num_rows, d) or not out.is_contiguous() or out.device != dev):
        raise ValueError(f"out is a contiguous ({num_rows}, {d}) tensor on {dev}")
    grad = torch.empty(num_rows, d, dtype=dtype, device=dev) if out is None else out
    ws = workspace(lib().sdm_embed_grad_workspace_size(N, d, num_rows), dev)
    with torch.cuda.device(dev):
        check(lib().sdm_embed_grad(ptr(i32), ptr(g), g.stride(0) if N > 1 else d, N, d, num_rows, scale,
                                   -1 if padding_id is None else padding_id, dtype_code(g.dtype),
                                   dtype_code(grad.dtype), int(out is not None), ptr(grad), ptr(ws), ws.numel(),
                                   stream_ptr(dev)), "sdm_embed_grad")
    return grad


def _embed(i32, table, scale, bad):
    V, d = table.shape
    out = torch.empty(*i32.shape, d, dtype=table.dtype, device=table.device)
    with torch.cuda.device(table.device):
        check(lib().sdm_embed_scaled(ptr(i32), ptr(table), i32.numel(), d, V, scale, dtype_code(table.dtype), ptr(out),
                                     ptr(bad), stream_ptr(table.device)), "sdm_embed_scaled")
    return out


class _EmbedTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, i32, scale, padding_id, bad):
        ctx.save_for_backward(i32)
        ctx.args = (table.shape[0], scale, padding_id, table.dtype)
        return _embed(i32, table.detach().contiguous(), scale, bad)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        (i32,) = ctx.saved_tensors
        V, scale, padding_id, dt = ctx.args
        return embed_grad(i32, g, V, scale, padding_id, dtype=dt), None, None, None, None


def embed_tokens(ids, table, scale=1.0, padding_id=None, bad=None):
    """scale * table[ids] in the table's dtype (sdm_embed_scaled), differentiable by the table (padding_id's row gets
    no gradient).  An id outside the table gives a zero row and sets bad (a device int32 tensor of one element)."""
    i32 = _ids32(ids)
    if table.dim() != 2:
        raise ValueError(f"the table is 2-D (tokens, d), not {table.dim()}-D")
    if table.device != i32.device:
        raise ValueError(f"ids are on {i32.device}, the table on {table.device}")
    if bad is not None and (bad.dtype != torch.int32 or bad.device != i32.device):
        raise ValueError("bad is an int32 tensor on the ids' device")
    if torch.is_grad_enabled() and table.requires_grad:
        return _EmbedTokens.apply(table, i32, scale, padding_id, bad)
    return _embed(i32, table.detach().contiguous(), scale, bad)
