"""Layers of a decoder as functions: `embedding` (the token table's lookup with a factor, its gradient by sorted tokens) and
`gated_linear` (both products of a gated feed-forward block, the activation and their product in one kernel).

They are ordinary autograd nodes, for the parts of a model that run beside a runner's stages or without one.  In a model that is
compiled for a runner a call is one node of the captured graph (`torch.ops.pfeife_amd`), which the stages' lowering knows
(`executor/lowering.py`)."""
import math
from typing import Tuple

import torch

from .hip import ACT_GELU, ACT_GELU_TANH, ACT_RELU, ACT_SILU
from .loss import _CODE, _LOGITS, _NoContext, _at, _call, _dual, _has_tangent, _need, _once, _recorded, _table

ACTS = {"silu": ACT_SILU, "gelu": ACT_GELU, "gelu_tanh": ACT_GELU_TANH, "relu": ACT_RELU}
KEPT = {"16bit": 1, "8bit": 2}


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, args, want=True):
        ids, scale, padding = args
        vocab, dim = weight.shape
        out = torch.empty(ids.shape + (dim,), dtype=weight.dtype, device=weight.device)
        _call(weight, "pf_embedding_scaled_fwd", weight.data_ptr(), _CODE[weight.dtype], ids.data_ptr(), out.data_ptr(), ids.numel(), dim, vocab, scale)
        if want:
            ctx.save_for_backward(ids)
            ctx.cfg = vocab, scale, padding
        return out

    @_once
    def backward(ctx, dout):
        ids, = ctx.saved_tensors
        return _table_gradient(dout, ids, *ctx.cfg), None


def _table_gradient(dout, ids, vocab, scale, padding):
    dim, n, dtype = dout.shape[-1], ids.numel(), _CODE[dout.dtype]
    dout = dout.contiguous()
    dw = torch.empty((vocab, dim), dtype=dout.dtype, device=dout.device)
    need = _need(dout, "pf_embedding_sorted_workspace", n, dim)
    work = torch.empty((need,), dtype=torch.uint8, device=dout.device) if need else None
    _call(dout, "pf_embedding_sorted_bwd", dout.data_ptr(), dtype, ids.data_ptr(), dw.data_ptr(), dtype, n, dim, vocab, padding, scale, 0, _at(work))
    return dw


def embedding(ids, weight, *, scale=1.0, padding_idx=None):
    """scale * weight[ids], with a dense gradient that is summed in fp32, in an order that the ids alone decide.

    ids int64 [...], weight [rows, width] (fp32, fp16 or bf16).  -> [..., width] in the weight's type.  padding_idx: a row that learns nothing
    (negative: counted from the end).  Ids outside the table give NaN and take no part in the gradient.  The gradient's work is dealt
    out by the tokens, so a token that fills half of a batch costs no more than others.  There are no second and no forward-mode
    derivatives.  A backward pass is captured into a graph, as any of torch's, only while no autograd graph made outside the capture holds
    the same leaves."""
    if torch.compiler.is_compiling() or _recorded():
        return torch.ops.pfeife_amd.embedding.default(ids, weight, float(scale), _table_row(weight, padding_idx))
    return _embedding(ids, weight, scale, padding_idx)


def _embedding(ids, weight, scale, padding_idx):
    if not torch.is_tensor(ids) or not torch.is_tensor(weight):
        raise RuntimeError("embedding: ids and weight are tensors")
    _table(weight, "embedding")
    padding = _check_embedding(ids, weight, scale, padding_idx)
    if _dual._current_level >= 0 and _has_tangent(weight):
        raise RuntimeError("embedding: there is no forward-mode derivative")
    wants = torch.is_grad_enabled() and weight.requires_grad
    if wants and (ids.numel() > 1 << 27 or weight.shape[0] >= (1 << 27) - 1 or weight.shape[1] > 65535 * 64):
        raise RuntimeError("embedding: too many ids, rows or columns for a gradient")
    weight = weight.contiguous()
    args = (ids.contiguous(), float(scale), padding)
    if wants:
        return _EmbeddingFn.apply(weight, args)
    return _EmbeddingFn.forward(_NoContext, weight, args, False)


def _table_row(weight, padding_idx):
    """-1: none"""
    rows = weight.shape[0]
    if padding_idx is not None and (not isinstance(padding_idx, int) or not -rows <= padding_idx < rows):
        raise RuntimeError("embedding: padding_idx is a row of the table (got %r)" % (padding_idx,))
    return -1 if padding_idx is None else padding_idx % rows


def _check_embedding(ids, weight, scale, padding_idx):
    who = "embedding"
    if weight.dtype not in _LOGITS or weight.dim() != 2 or weight.shape[0] == 0 or weight.shape[1] == 0:
        raise RuntimeError("%s: weight is [rows, width] in fp32, fp16 or bf16 (got %s %s)" % (who, weight.dtype, tuple(weight.shape)))
    if ids.dtype != torch.int64 or ids.device != weight.device:
        raise RuntimeError("%s: ids are int64 on %s (got %s on %s)" % (who, weight.device, ids.dtype, ids.device))
    if not isinstance(scale, (int, float)) or not math.isfinite(scale):
        raise RuntimeError("%s: scale is a finite number" % who)
    return _table_row(weight, padding_idx)


class _GatedLinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, args, want=True):
        act, keep = args
        y, kept = _gated_forward(x, weight, act, keep if want else 0)
        if want:
            ctx.save_for_backward(x, weight, kept)
            ctx.cfg = act, keep
        return y

    @_once
    def backward(ctx, dy):
        return *_gated_gradients(dy, *ctx.saved_tensors, *ctx.cfg, *ctx.needs_input_grad[:2]), None


def _gated_forward(x, weight, act, keep):
    """-> (y, what the backward pass starts from; None: nothing)"""
    rows, D = x.shape
    ffn, dtype, dev = weight.shape[0] // 2, _CODE[x.dtype], x.device
    at, w = x.data_ptr(), weight.data_ptr()
    kept = None
    if keep:
        kept = torch.empty((_need(x, "pf_gated_linear_kept", dtype, rows, ffn, keep),), dtype=torch.uint8, device=dev)
    need = _need(x, "pf_gated_linear_workspace", at, w, dtype, rows, D, ffn, keep, 0)
    work = torch.empty((need,), dtype=torch.uint8, device=dev) if need else None
    y = torch.empty((rows, ffn), dtype=x.dtype, device=dev)
    _call(x, "pf_gated_linear_fwd", at, dtype, rows, D, w, ffn, act, keep, y.data_ptr(), _at(kept), _at(work))
    return y, kept


def _gated_gradients(dy, x, weight, kept, act, keep, want_x, want_weight):
    rows, D = x.shape
    ffn, dtype, dev = weight.shape[0] // 2, _CODE[x.dtype], x.device
    at, w = x.data_ptr(), weight.data_ptr()
    work = torch.empty((_need(x, "pf_gated_linear_workspace", at, w, dtype, rows, D, ffn, keep, 1),), dtype=torch.uint8, device=dev)
    dx = torch.empty((rows, D), dtype=x.dtype, device=dev) if want_x else None
    dw = torch.empty((2 * ffn, D), dtype=x.dtype, device=dev) if want_weight else None
    dy = dy.contiguous()
    _call(x, "pf_gated_linear_bwd", at, dtype, rows, D, w, ffn, act, keep, kept.data_ptr(), dy.data_ptr(), _at(dx), _at(dw), work.data_ptr())
    return dx, dw


def gated_linear(x, weight, *, act="silu", kept="16bit"):
    """act(x @ gate.T) * (x @ up.T), the first half of a gated feed-forward block.

    x [..., D] and weight [2 F, D] (fp32, fp16 or bf16, the same type): the gate's F rows, then the other matrix'.  -> [..., F].  act is
    "silu", "gelu" (the erf form), "gelu_tanh" or "relu".  kept: what the backward pass finds of the two products, "16bit": rounded to
    the operands' type (fp32 operands: as they are), "8bit" (16-bit operands): e4m3 codes, 16 neighbouring columns under one power
    of two, in 17/32 of the memory; the result itself is the same.  The gradient flows to x and weight.  There are no second and no
    forward-mode derivatives.  A backward pass is captured into a graph, as any of torch's, only while no autograd graph made outside the
    capture holds the same leaves."""
    if torch.compiler.is_compiling() or _recorded():
        return torch.ops.pfeife_amd.gated_linear.default(x, weight, act, kept)
    return _gated_linear(x, weight, act, kept)


def _gated_linear(x, weight, act, kept):
    if not torch.is_tensor(x) or not torch.is_tensor(weight):
        raise RuntimeError("gated_linear: x and weight are tensors")
    _table(x, "gated_linear")
    _check_gated(x, weight, act, kept)
    if _dual._current_level >= 0 and _has_tangent(x, weight):
        raise RuntimeError("gated_linear: there is no forward-mode derivative")
    if x.dtype == torch.float32 and kept == "8bit":
        raise RuntimeError("gated_linear: kept is '16bit', or for 16-bit operands '8bit' (got %r for %s)" % (kept, x.dtype))
    shape = x.shape
    rows = (x if len(shape) == 2 else x.reshape(math.prod(shape[:-1]), shape[-1])).contiguous()
    weight = weight.contiguous()
    args = (ACTS[act], KEPT[kept])
    if torch.is_grad_enabled() and (rows.requires_grad or weight.requires_grad):
        y = _GatedLinearFn.apply(rows, weight, args)
    else:
        y = _GatedLinearFn.forward(_NoContext, rows, weight, args, False)
    return y if len(shape) == 2 else y.reshape(shape[:-1] + y.shape[1:])


def _check_gated(x, weight, act, kept):
    """(Not whether 8 bits go with the operands' type: a runner's stages compute in one of their own.)"""
    who = "gated_linear"
    if x.dtype not in _LOGITS or weight.dtype != x.dtype:
        raise RuntimeError("%s: x and weight are both fp32, fp16 or bf16 (got %s and %s)" % (who, x.dtype, weight.dtype))
    shape, of = x.shape, weight.shape
    if len(shape) < 1 or shape[-1] == 0:
        raise RuntimeError("%s: x is [..., width] (got %s)" % (who, tuple(shape)))
    if len(of) != 2 or of[1] != shape[-1] or of[0] == 0 or of[0] % 2 or weight.device != x.device:
        raise RuntimeError("%s: weight is [2 * columns, %d] on %s (got %s on %s)" % (who, shape[-1], x.device, tuple(of), weight.device))
    if act not in ACTS:
        raise RuntimeError("%s: act is one of %s (got %r)" % (who, ", ".join(ACTS), act))
    if kept not in KEPT:
        raise RuntimeError("%s: kept is '16bit', or for 16-bit operands '8bit' (got %r for %s)" % (who, kept, x.dtype))


# A call inside a graph that is being captured is a node of it, and so is its backward pass where that is traced as well.  What their results look
# like is all that capturing asks; a runner's stages run the forward nodes by their lowering, and whatever else runs a captured graph (the compiler's
# other backends) runs the functions above.
@torch.library.custom_op("pfeife_amd::embedding", mutates_args=())
def _embedding_op(ids: torch.Tensor, weight: torch.Tensor, scale: float, padding_idx: int) -> torch.Tensor:
    return _embedding(ids, weight.detach(), scale, None if padding_idx < 0 else padding_idx)


@_embedding_op.register_fake
def _(ids, weight, scale, padding_idx):
    _check_embedding(ids, weight, scale, None if padding_idx < 0 else padding_idx)
    return weight.new_empty(tuple(ids.shape) + (weight.shape[1],))


@torch.library.custom_op("pfeife_amd::embedding_backward", mutates_args=())
def _embedding_backward_op(grad: torch.Tensor, ids: torch.Tensor, rows: int, scale: float, padding_idx: int) -> torch.Tensor:
    _table(grad, "embedding")
    return _table_gradient(grad, ids.contiguous(), rows, scale, padding_idx)


@_embedding_backward_op.register_fake
def _(grad, ids, rows, scale, padding_idx):
    return grad.new_empty((rows, grad.shape[-1]))


@torch.library.custom_op("pfeife_amd::gated_linear", mutates_args=())
def _gated_linear_op(x: torch.Tensor, weight: torch.Tensor, act: str, kept: str) -> torch.Tensor:
    return _gated_linear(x.detach(), weight.detach(), act, kept)      # (nothing is kept: the backward pass forms both products again)


@_gated_linear_op.register_fake
def _(x, weight, act, kept):
    _check_gated(x, weight, act, kept)
    return x.new_empty(tuple(x.shape[:-1]) + (weight.shape[0] // 2,))


# An operator of the graph hands over one result, so both products are formed again here (rounded as kept says, as where they are kept); what is not wanted
# is empty
@torch.library.custom_op("pfeife_amd::gated_linear_backward", mutates_args=())
def _gated_linear_backward_op(grad: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, act: str, kept: str, want_x: bool,
                              want_weight: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    _table(x, "gated_linear")
    rows, weight = x.reshape(math.prod(x.shape[:-1]), x.shape[-1]).contiguous(), weight.contiguous()
    _, held = _gated_forward(rows, weight, ACTS[act], KEPT[kept])
    dx, dw = _gated_gradients(grad, rows, weight, held, ACTS[act], KEPT[kept], want_x, want_weight)
    return dx.reshape(x.shape) if want_x else x.new_empty(0), dw if want_weight else weight.new_empty(0)


@_gated_linear_backward_op.register_fake
def _(grad, x, weight, act, kept, want_x, want_weight):
    return x.new_empty(x.shape if want_x else 0), weight.new_empty(weight.shape if want_weight else 0)


def _save_embedding(ctx, inputs, output):
    ids, weight, scale, padding = inputs
    ctx.save_for_backward(ids)
    ctx.rest = weight.shape[0], scale, padding


def _embedding_backward(ctx, grad):
    ids, = ctx.saved_tensors
    return None, torch.ops.pfeife_amd.embedding_backward.default(grad, ids, *ctx.rest), None, None


def _save_gated_linear(ctx, inputs, output):
    ctx.save_for_backward(*inputs[:2])
    ctx.rest = inputs[2:]


def _gated_linear_backward(ctx, grad):
    want = ctx.needs_input_grad[:2]
    grads = torch.ops.pfeife_amd.gated_linear_backward.default(grad, *ctx.saved_tensors, *ctx.rest, *want)
    return *(g if w else None for g, w in zip(grads, want)), None, None


_embedding_op.register_autograd(_embedding_backward, setup_context=_save_embedding)
_gated_linear_op.register_autograd(_gated_linear_backward, setup_context=_save_gated_linear)
