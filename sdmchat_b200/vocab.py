"""The vocabulary end of a language model on libsdm_b200: rules on logits and the choice of a token (serving), the
distillation loss and the token table's lookup with their gradients (training).

Tensors are on a CUDA device, in float32 or bfloat16 (ids int32; other integer types are converted, numbers that int32
does not hold to ones outside every table); every call runs on the current stream of its tensors' device.
`distill_loss` and `embed_tokens` record autograd; the other functions are forward only.  There is no CPU or PyTorch
fallback.  Distillation's device-side waits are bounded: rows left over by one that gave up have a NaN loss, and
sdm_device_status reports it.
"""
import contextlib
import dataclasses
import struct
from typing import Optional, Union

import torch

from . import _lib as L_
from ._lib import check, lib, workspace, dtype_code

Per = Union[float, torch.Tensor]  # one value for all rows, or one per row
I32, F32 = torch.int32, torch.float32
I32_MAX = 2 ** 31 - 1
_WIDE = (torch.int64, torch.uint32, torch.uint64)  # integer types with numbers that int32 does not hold
_NOTHING = contextlib.nullcontext()
# sdm_logit_rules and sdm_choice_params as C lays them out (a call at one stream is bound by the host: packing a struct
# this way takes a fifth of setting its fields one by one)
_RULES = struct.Struct("@PqiPPPPPfffPPiPiP")
_CHOICE = struct.Struct("@PPPPffi0P")


def _ix(t, name):
    """Device index of a CUDA tensor."""
    ix = t.get_device()
    if ix < 0:
        raise ValueError(f"{name}: libsdm_b200 takes device tensors only")
    return ix


def _stream(ix):
    return torch._C._cuda_getCurrentRawStream(ix)


def _guard(ix):
    """Makes device ix current for a launch."""
    return _NOTHING if torch.cuda.current_device() == ix else torch.cuda.device(ix)


def _narrow(t):
    """Whole numbers t as contiguous int32.  What int32 does not hold becomes -1 or 2^31 - 1, so that an id outside a
    table stays outside."""
    t = t.detach()
    if t.dtype in _WIDE:
        t = t.to(torch.int64).clamp(-1, I32_MAX)
    return t.to(I32).contiguous()


def _at(t, ix, name, dtype, shape, keep, bits=False):
    """Pointer of t (None: 0) as a contiguous tensor of dtype on device ix with the given shape (None: any size).  A
    converted copy goes into `keep`, which lives until the launch.  bits: int32 words whose bits count."""
    if t is None:
        return 0
    if t.dtype is dtype and t.get_device() == ix and t.shape == shape and t.is_contiguous():
        return t.data_ptr()
    if t.get_device() != ix:
        raise ValueError(f"{name} is on {t.device}, the logits or ids are on device {ix}")
    if t.dim() != len(shape) or any(w is not None and n != w for n, w in zip(t.shape, shape)):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, wanted {tuple('any' if w is None else w for w in shape)}")
    if dtype is I32 and (t.dtype.is_floating_point or t.dtype.is_complex):
        raise TypeError(f"{name} holds whole numbers, not {t.dtype}")
    t = _narrow(t) if dtype is I32 and not bits else t.detach().to(dtype).contiguous()
    keep.append(t)
    return t.data_ptr()


def _per(v, ix, name, dtype, S, keep):
    """(pointer, value for all rows) of a per-row parameter."""
    if isinstance(v, torch.Tensor):
        return _at(v, ix, name, dtype, (S,), keep), 0
    return 0, v


def _rows(t, name):
    """t (N, V) with contiguous rows, and its row stride."""
    if t.dim() != 2:
        raise ValueError(f"{name} is 2-D (rows, vocabulary), not {t.dim()}-D")
    N, V = t.shape
    if V > I32_MAX:
        raise ValueError(f"{name}: {V} tokens are more than the library counts")
    if t.is_contiguous():
        return t, V
    if V > 1 and t.stride(1) != 1 or N > 1 and t.stride(0) < V:
        return t.contiguous(), V
    return t, (t.stride(0) if N > 1 else V)


def _out_rows(out, like, name):
    """Row stride of an output for `like`'s rows."""
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
        raise ValueError(f"{name} has the shape, dtype and device of the logits")
    N, V = out.shape
    if V > 1 and out.stride(1) != 1 or N > 1 and out.stride(0) < V:
        raise ValueError(f"{name} needs contiguous rows that do not overlap")

    def span(t):
        return t.data_ptr(), t.data_ptr() + ((N - 1) * t.stride(0) + (V - 1) * t.stride(1) + 1) * t.element_size()

    (a0, a1), (b0, b1) = span(out), span(like)
    apart = False  # side by side in the rows of one buffer
    if N > 1 and out.stride() == like.stride():
        ld, width = out.stride(0) * out.element_size(), V * out.element_size()
        apart = width <= (a0 - b0) % ld <= ld - width
    if a0 < b1 and b0 < a1 and not apart and (a0 != b0 or out.stride() != like.stride()) and N * V > 0:
        raise ValueError(f"{name} overlaps the logits without being them")
    return out.stride(0) if N > 1 else V


def _written(t):
    """Tells autograd that the library wrote to a tensor of the caller's: what was saved of its old values is stale."""
    torch.autograd.graph.increment_version(t)
    return t


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

    def _struct(self, S, V, ix, keep):
        """sdm_logit_rules for S rows over V tokens on device ix."""
        hist, bi, bv, mask = self.history, self.bias_ids, self.bias_values, self.mask
        L = nb = G = 0
        hp = hlp = plp = bip = bvp = mp = 0
        if hist is not None:
            L = hist.shape[-1]
            hp = _at(hist, ix, "history", I32, (S, L), keep)
            hlp = _at(self.history_len, ix, "history_len", I32, (S,), keep)
            plp = _at(self.prompt_len, ix, "prompt_len", I32, (S,), keep)
            if L == 0:
                hp = hlp = plp = 0
        elif self.history_len is not None or self.prompt_len is not None:
            raise ValueError("history_len and prompt_len need a history")
        if bi is not None and bv is not None:
            nb = bi.shape[-1]
            bip = _at(bi, ix, "bias_ids", I32, (S, nb), keep)
            bvp = _at(bv, ix, "bias_values", F32, (S, nb), keep)
        elif bi is not None or bv is not None:
            raise ValueError("bias_ids and bias_values come together")
        mrp = _at(self.mask_row, ix, "mask_row", I32, (S,), keep)
        if mask is not None:
            G = mask.shape[0]
            mp = _at(mask, ix, "mask", I32, (G, -(-V // 32)), keep, bits=True)
            if not mrp and G != 1 and G != S:
                raise ValueError(f"{G} masks for {S} rows need mask_row")
        elif mrp:
            raise ValueError("mask_row needs a mask")
        rp, ra = _per(self.repetition, ix, "repetition", F32, S, keep)
        fp, fa = _per(self.frequency, ix, "frequency", F32, S, keep)
        pp, pa = _per(self.presence, ix, "presence", F32, S, keep)
        return L_.LogitRules.from_buffer_copy(
            _RULES.pack(hp, L, L, hlp, plp, rp, fp, pp, ra, fa, pa, bip, bvp, nb, mp, G, mrp))


def process_logits(logits, rules=None, out=None):
    """The rules on logits (S, V), in their dtype (rounded once): penalties, biases, then the mask (sdm_logits_process).
    out: where to write (the logits themselves are allowed), else a new tensor."""
    ix = _ix(logits, "logits")
    code = dtype_code(logits.dtype)
    x, ld = _rows(logits, "logits")
    S, V = x.shape
    own = out is None
    if own:
        out, ld_out = torch.empty(S, V, dtype=x.dtype, device=x.device), V
    else:
        ld_out = _out_rows(out, logits, "out")
    keep = []
    r = None if rules is None else rules._struct(S, V, ix, keep)
    with _guard(ix):
        check(lib().sdm_logits_process(r, x.data_ptr(), ld, S, V, code, out.data_ptr(), ld_out, _stream(ix)),
              "sdm_logits_process")
    return out if own else _written(out)


def sample_logits(logits, rules=None, u=None, temperature: Per = 1.0, top_k: Union[int, torch.Tensor] = 0,
                  top_p: Per = 1.0):
    """One token per row of logits (S, V) under the rules: ids (S,) int32 and log-probabilities (S,) float32 under the
    distribution drawn from (sdm_logits_choose).  u (S,) in [0, 1) picks the token: with the kept tokens in index
    order, the first whose running probability exceeds it.  temperature 0 takes the largest logit (u may be None if
    that is so for all rows).  A row that allows no token gives -1 and -infinity."""
    ix = _ix(logits, "logits")
    code = dtype_code(logits.dtype)
    x, ld = _rows(logits, "logits")
    S, V = x.shape
    keep = []
    r = None if rules is None else rules._struct(S, V, ix, keep)
    tp, ta = _per(temperature, ix, "temperature", F32, S, keep)
    kp, ka = _per(top_k, ix, "top_k", I32, S, keep)
    pp, pa = _per(top_p, ix, "top_p", F32, S, keep)
    if u is None and (tp or ta != 0):
        raise ValueError("sampling needs u, one number in [0, 1) per row")
    up = _at(u, ix, "u", F32, (S,), keep)
    c = L_.ChoiceParams.from_buffer_copy(_CHOICE.pack(tp, kp, pp, up, ta, pa, ka))
    ids = torch.empty(S, dtype=I32, device=x.device)
    lp = torch.empty(S, dtype=F32, device=x.device)
    with _guard(ix):
        check(lib().sdm_logits_choose(r, c, x.data_ptr(), ld, S, V, code, ids.data_ptr(), lp.data_ptr(), _stream(ix)),
              "sdm_logits_choose")
    return ids, lp


# -------------------------------------------------------------------------------------------------- distillation
def _distill(logits, teacher_ids, teacher_logits, targets, temperature, alpha, row_weight, teacher_lse, grad_scale,
             want_grad, out=None):
    ix = _ix(logits, "logits")
    code = dtype_code(logits.dtype)
    x, ld = _rows(logits, "logits")
    N, V = x.shape
    k = teacher_ids.shape[-1]
    keep = []
    idp = _at(teacher_ids, ix, "teacher_ids", I32, (N, k), keep)
    tlp = _at(teacher_logits, ix, "teacher_logits", F32, (N, k), keep)
    tgp = _at(targets, ix, "targets", I32, (N,), keep)
    wp = _at(row_weight, ix, "row_weight", F32, (N,), keep)
    lsep = _at(teacher_lse, ix, "teacher_lse", F32, (N,), keep)
    loss = torch.empty(N, dtype=F32, device=x.device)
    grad, gp, ldg = None, 0, 0
    if want_grad:
        if out is None:
            grad, ldg = torch.empty(N, V, dtype=x.dtype, device=x.device), V
        else:
            grad, ldg = out, _out_rows(out, logits, "out")
        gp = grad.data_ptr()
    with _guard(ix):
        check(lib().sdm_distill(x.data_ptr(), ld, N, V, code, idp, tlp, k, lsep, tgp, wp, temperature, alpha,
                                grad_scale, loss.data_ptr(), gp, ldg, _stream(ix)), "sdm_distill")
    if out is not None:
        _written(out)
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
            ix = grad.get_device()
            with _guard(ix):
                check(lib().sdm_scale_rows(grad.data_ptr(), V, N, V, dtype_code(grad.dtype), g.data_ptr(),
                                           0 if one else 1, _stream(ix)), "sdm_scale_rows")
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
    the logits and kept in their dtype for the backward pass, which is free for "sum" and "mean" used as the loss itself;
    another factor multiplies it there, in bfloat16 with a second rounding.  The backward pass can be run once.
    Teacher, targets and weights get no gradient."""
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
    if ids.dtype is I32 and ids.is_contiguous():
        return ids
    if ids.dtype.is_floating_point or ids.dtype.is_complex or ids.dtype is torch.bool:
        raise TypeError(f"ids are whole numbers, not {ids.dtype}")
    return _narrow(ids)


def embed_grad(ids, dout, num_rows, scale=1.0, padding_id=None, dtype=torch.float32, out=None):
    """The token table's gradient (num_rows, d): scale times the sum of dout (..., d) over the positions of each id
    (sdm_embed_grad).  ids outside the table and padding_id are skipped.  out: a gradient (num_rows, d), float32 or
    bfloat16, to add to; else a new one of `dtype`.  The same inputs give the same bits."""
    ix = _ix(ids, "ids")
    i32 = _ids32(ids)
    if dout.get_device() != ix or dout.shape[:-1] != ids.shape:
        raise ValueError(f"dout {tuple(dout.shape)} on {dout.device} does not go with ids {tuple(ids.shape)} on {ids.device}")
    d = dout.shape[-1]
    N = i32.numel()
    if dout.is_contiguous():
        ld = d
    elif dout.dim() == 2 and dout.stride(1) == 1 and dout.stride(0) >= d:
        ld = dout.stride(0) if N > 1 else d
    else:
        dout, ld = dout.contiguous(), d
    if out is None:
        grad = torch.empty(num_rows, d, dtype=dtype, device=i32.device)
    else:
        if out.shape != (num_rows, d) or not out.is_contiguous() or out.get_device() != ix:
            raise ValueError(f"out is a contiguous ({num_rows}, {d}) tensor on {ids.device}")
        grad = out
    if not 0 < num_rows <= I32_MAX or d > I32_MAX:
        raise ValueError(f"a table of {num_rows} x {d} is more than the library counts")
    skip = padding_id if padding_id is not None and 0 <= padding_id < num_rows else -1
    nbytes = lib().sdm_embed_grad_workspace_size(N, d, num_rows)
    ws = workspace(nbytes, i32.device)
    with _guard(ix):
        check(lib().sdm_embed_grad(i32.data_ptr(), dout.data_ptr(), ld, N, d, num_rows, scale,
                                   skip, dtype_code(dout.dtype), dtype_code(grad.dtype), int(out is not None),
                                   grad.data_ptr(), ws.data_ptr(), nbytes, _stream(ix)), "sdm_embed_grad")
    return grad if out is None else _written(out)


def _embed(i32, table, scale, bad):
    V, d = table.shape
    if max(V, d) > I32_MAX:
        raise ValueError(f"a table of {V} x {d} is more than the library counts")
    ix = i32.get_device()
    out = torch.empty(*i32.shape, d, dtype=table.dtype, device=table.device)
    with _guard(ix):
        check(lib().sdm_embed_scaled(i32.data_ptr(), table.data_ptr(), i32.numel(), d, V, scale,
                                     dtype_code(table.dtype), out.data_ptr(), 0 if bad is None else bad.data_ptr(),
                                     _stream(ix)), "sdm_embed_scaled")
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
    ix = _ix(ids, "ids")
    i32 = _ids32(ids)
    if table.dim() != 2:
        raise ValueError(f"the table is 2-D (tokens, d), not {table.dim()}-D")
    if table.get_device() != ix:
        raise ValueError(f"ids are on {ids.device}, the table is on {table.device}")
    if bad is not None and (bad.dtype is not I32 or bad.get_device() != ix):
        raise ValueError("bad is an int32 tensor on the ids' device")
    if table.requires_grad and torch.is_grad_enabled():
        return _EmbedTokens.apply(table, i32, scale, padding_id, bad)
    return _embed(i32, table if table.is_contiguous() else table.contiguous(), scale, bad)
