"""Layers of a decoder as functions: `embedding` (the token table's lookup with a factor, its gradient by sorted tokens) and
`gated_linear` (both products of a gated feed-forward block, the activation and their product in one kernel).

They are ordinary autograd nodes, for the parts of a model that run beside a runner's stages or without one; the stages' own are
lowered from the captured graph (`executor/lowering.py`)."""
import math

import torch

from .hip import ACT_GELU, ACT_GELU_TANH, ACT_RELU, ACT_SILU
from .loss import _CODE, _LOGITS, _NoContext, _at, _call, _dual, _has_tangent, _need, _once, _table

_ACTS = {"silu": ACT_SILU, "gelu": ACT_GELU, "gelu_tanh": ACT_GELU_TANH, "relu": ACT_RELU}
_KEPT = {"16bit": 1, "8bit": 2}


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
        vocab, scale, padding = ctx.cfg
        dim, n, dtype = dout.shape[-1], ids.numel(), _CODE[dout.dtype]
        dout = dout.contiguous()
        dw = torch.empty((vocab, dim), dtype=dout.dtype, device=dout.device)
        need = _need(dout, "pf_embedding_sorted_workspace", n, dim)
        work = torch.empty((need,), dtype=torch.uint8, device=dout.device) if need else None
        _call(dout, "pf_embedding_sorted_bwd", dout.data_ptr(), dtype, ids.data_ptr(), dw.data_ptr(), dtype, n, dim, vocab, padding, scale, 0, _at(work))
        return dw, None


def embedding(ids, weight, *, scale=1.0, padding_idx=None):
    """scale * weight[ids], with a dense gradient that is summed in fp32, in an order that the ids alone decide.

    ids int64 [...], weight [rows, width] (fp32, fp16 or bf16).  -> [..., width] in the weight's type.  padding_idx: a row that learns nothing
    (negative: counted from the end).  Ids outside the table give NaN and take no part in the gradient.  The gradient's work is dealt
    out by the tokens, so a token that fills half of a batch costs no more than others.  There are no second and no forward-mode
    derivatives.  A backward pass is captured into a graph, as any of torch's, only while no autograd graph made outside the capture holds
    the same leaves."""
    who = "embedding"
    if not torch.is_tensor(ids) or not torch.is_tensor(weight):
        raise RuntimeError("%s: ids and weight are tensors" % who)
    _table(weight, who)
    if weight.dtype not in _LOGITS or weight.dim() != 2 or weight.shape[0] == 0 or weight.shape[1] == 0:
        raise RuntimeError("%s: weight is [rows, width] in fp32, fp16 or bf16 (got %s %s)" % (who, weight.dtype, tuple(weight.shape)))
    if ids.dtype != torch.int64 or ids.get_device() != weight.get_device():
        raise RuntimeError("%s: ids are int64 on %s (got %s on %s)" % (who, weight.device, ids.dtype, ids.device))
    if not isinstance(scale, (int, float)) or not math.isfinite(scale):
        raise RuntimeError("%s: scale is a finite number" % who)
    rows = weight.shape[0]
    if padding_idx is not None and (not isinstance(padding_idx, int) or not -rows <= padding_idx < rows):
        raise RuntimeError("%s: padding_idx is a row of the table (got %r)" % (who, padding_idx))
    if _dual._current_level >= 0 and _has_tangent(weight):
        raise RuntimeError("%s: there is no forward-mode derivative" % who)
    weight = weight.contiguous()
    args = (ids.contiguous(), float(scale), -1 if padding_idx is None else padding_idx % rows)
    if torch.is_grad_enabled() and weight.requires_grad:
        return _EmbeddingFn.apply(weight, args)
    return _EmbeddingFn.forward(_NoContext, weight, args, False)


class _GatedLinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, args, want=True):
        act, keep = args
        keep = keep if want else 0
        rows, D = x.shape
        ffn, dtype, dev = weight.shape[0] // 2, _CODE[x.dtype], x.device
        at, w = x.data_ptr(), weight.data_ptr()
        kept = None
        if want:
            kept = torch.empty((_need(x, "pf_gated_linear_kept", dtype, rows, ffn, keep),), dtype=torch.uint8, device=dev)
        need = _need(x, "pf_gated_linear_workspace", at, w, dtype, rows, D, ffn, keep, 0)
        work = torch.empty((need,), dtype=torch.uint8, device=dev) if need else None
        y = torch.empty((rows, ffn), dtype=x.dtype, device=dev)
        _call(x, "pf_gated_linear_fwd", at, dtype, rows, D, w, ffn, act, keep, y.data_ptr(), _at(kept), _at(work))
        if want:
            ctx.save_for_backward(x, weight, kept)
            ctx.cfg = act, keep
        return y

    @_once
    def backward(ctx, dy):
        x, weight, kept = ctx.saved_tensors
        act, keep = ctx.cfg
        rows, D = x.shape
        ffn, dtype, dev = weight.shape[0] // 2, _CODE[x.dtype], x.device
        at, w = x.data_ptr(), weight.data_ptr()
        work = torch.empty((_need(x, "pf_gated_linear_workspace", at, w, dtype, rows, D, ffn, keep, 1),), dtype=torch.uint8, device=dev)
        dx = torch.empty((rows, D), dtype=x.dtype, device=dev) if ctx.needs_input_grad[0] else None
        dw = torch.empty((2 * ffn, D), dtype=x.dtype, device=dev) if ctx.needs_input_grad[1] else None
        dy = dy.contiguous()
        _call(x, "pf_gated_linear_bwd", at, dtype, rows, D, w, ffn, act, keep, kept.data_ptr(), dy.data_ptr(), _at(dx), _at(dw), work.data_ptr())
        return dx, dw, None


def gated_linear(x, weight, *, act="silu", kept="16bit"):
    """act(x @ gate.T) * (x @ up.T), the first half of a gated feed-forward block.

    x [..., D] and weight [2 F, D] (fp32, fp16 or bf16, the same type): the gate's F rows, then the other matrix'.  -> [..., F].  act is
    "silu", "gelu" (the erf form), "gelu_tanh" or "relu".  kept: what the backward pass finds of the two products, "16bit": rounded to
    the operands' type (fp32 operands: as they are), "8bit" (16-bit operands): e4m3 codes, 16 neighbouring columns under one power
    of two, in 17/32 of the memory; the result itself is the same.  The gradient flows to x and weight.  There are no second and no
    forward-mode derivatives.  A backward pass is captured into a graph, as any of torch's, only while no autograd graph made outside the
    capture holds the same leaves."""
    who = "gated_linear"
    if not torch.is_tensor(x) or not torch.is_tensor(weight):
        raise RuntimeError("%s: x and weight are tensors" % who)
    _table(x, who)
    if x.dtype not in _LOGITS or weight.dtype != x.dtype:
        raise RuntimeError("%s: x and weight are both fp32, fp16 or bf16 (got %s and %s)" % (who, x.dtype, weight.dtype))
    if x.dim() < 1 or x.shape[-1] == 0:
        raise RuntimeError("%s: x is [..., width] (got %s)" % (who, tuple(x.shape)))
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1] or weight.shape[0] == 0 or weight.shape[0] % 2 or weight.get_device() != x.get_device():
        raise RuntimeError("%s: weight is [2 * columns, %d] on %s (got %s on %s)" % (who, x.shape[-1], x.device, tuple(weight.shape), weight.device))
    if act not in _ACTS:
        raise RuntimeError("%s: act is one of %s (got %r)" % (who, ", ".join(_ACTS), act))
    if kept not in _KEPT or (kept == "8bit" and x.dtype == torch.float32):
        raise RuntimeError("%s: kept is '16bit', or for 16-bit operands '8bit' (got %r for %s)" % (who, kept, x.dtype))
    if _dual._current_level >= 0 and _has_tangent(x, weight):
        raise RuntimeError("%s: there is no forward-mode derivative" % who)
    rows = x.reshape(math.prod(x.shape[:-1]), x.shape[-1]).contiguous()
    weight = weight.contiguous()
    args = (_ACTS[act], _KEPT[kept])
    if torch.is_grad_enabled() and (rows.requires_grad or weight.requires_grad):
        y = _GatedLinearFn.apply(rows, weight, args)
    else:
        y = _GatedLinearFn.forward(_NoContext, rows, weight, args, False)
    return y.reshape(x.shape[:-1] + y.shape[1:])
