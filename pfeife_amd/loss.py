"""Loss wrappers with the reference's signatures (`forward(input, target, model=None)`,
pfeife/loss.py:4-70).

`CrossEntropyLoss` / `HFCrossEntropyLoss` are the mean-reduced cross entropy of
nn.CrossEntropyLoss computed by the pf_cross_entropy_fwd/bwd kernels when the
logits live on the GPU; `SumLoss` uses pf_sum_fwd.  The wrappers are ordinary
autograd nodes, so user code keeps calling `loss.backward()`.

`linear_cross_entropy` is the cross entropy of a decoder's head from the last hidden state, without the logits in memory.

For fine-tuning a language model: `token_logprobs` (log-probabilities of given tokens),
`preference_loss` (paired log ratios against a reference model) and `policy_loss` (clipped
ratio with a KL term), each straight from the logits, and `PreferenceLoss` / `PolicyLoss`.
"""
import functools
import math
from types import SimpleNamespace

import torch
import torch.autograd.forward_ad as forward_ad
import torch.nn as nn


def _kernels_for(t):
    if t.device.type != "cuda":
        raise RuntimeError("pfeife_amd.loss: the HIP loss kernels need GPU tensors (got %s)" % t.device)
    from .hip import HipKernels

    k = getattr(_kernels_for, "_k", None)
    if k is None:
        k = _kernels_for._k = HipKernels(t.device.index)
    return k


_scratch = {}


def _scratch_buffer(name, shape, dtype, device):
    """Per-shape work buffers of the loss kernels, allocated once: every micro-batch's loss is
    evaluated on the same stream in turn, and each buffer's last reader (the backward kernel, or the
    copy of the gradient into the stage's own buffer) is enqueued before the next micro-batch's
    writer, so a training loop makes no allocator call and no fill here."""
    key = (name, tuple(shape), dtype, str(device))
    t = _scratch.get(key)
    if t is None:
        if len(_scratch) > 64:
            _scratch.clear()
        t = _scratch[key] = torch.empty(shape, dtype=dtype, device=device)
    return t


class _CrossEntropyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, target, ignore_index):
        k = _kernels_for(logits)
        logits = logits.contiguous()
        target = target.contiguous()
        rows, classes = logits.shape
        row_loss = _scratch_buffer("row_loss", (rows,), torch.float32, logits.device)
        # saved for backward: per call, a second loss may be evaluated before the first one's backward
        row_lse = torch.empty(rows, dtype=torch.float32, device=logits.device)
        loss = torch.empty(2, dtype=torch.float32, device=logits.device)   # {mean loss, 1 / counted rows}
        k.run("cross_entropy_fwd", logits, target, row_loss, row_lse, loss, rows, classes, ignore_index)
        ctx.save_for_backward(logits, target, row_lse, loss)
        ctx.ignore_index = ignore_index
        return loss[0]      # a view of this call's own result pair: no copy kernel

    @staticmethod
    def backward(ctx, grad_out):
        logits, target, row_lse, loss = ctx.saved_tensors
        k = _kernels_for(logits)
        rows, classes = logits.shape
        dlogits = _scratch_buffer("dlogits", logits.shape, logits.dtype, logits.device)
        g = grad_out.detach()
        if g.dtype != torch.float32 or not g.is_contiguous():
            g = g.to(torch.float32).contiguous()
        k.run("cross_entropy_bwd", logits, target, row_lse, g, loss, dlogits, rows, classes, ctx.ignore_index)
        return dlogits, None, None


class _SumFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        k = _kernels_for(x)
        xc = x.contiguous()
        partial = torch.empty(k.reduce_workspace(xc.numel()), dtype=torch.float32, device=x.device)
        out = torch.empty(1, dtype=torch.float32, device=x.device)
        k.run("sum_fwd", xc, partial, out, xc.numel())
        ctx.shape, ctx.dtype = x.shape, x.dtype
        return out[0].to(x.dtype)

    @staticmethod
    def backward(ctx, grad_out):
        return grad_out.to(ctx.dtype).expand(ctx.shape)


def cross_entropy(logits, target, ignore_index=-100):
    """Mean cross entropy over [rows, classes] logits and int64 targets (HIP kernels)."""
    return _CrossEntropyFn.apply(logits, target, ignore_index)


_tables = {}
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _table(t, who):
    """The kernel table of the tensor's own device."""
    k = _tables.get(t.get_device())
    if k is None:
        if t.device.type != "cuda":
            raise RuntimeError("%s: the HIP kernels need GPU tensors (got %s)" % (who, t.device))
        from .hip import HipKernels

        with torch.cuda.device(t.device):
            k = _tables[t.device.index] = HipKernels(t.device.index)
    return k


_modes, _mode, _proxies = torch._C._len_torch_dispatch_stack, torch._C._get_dispatch_mode, torch._C._TorchDispatchModeKey.PROXY
_tracing, _key_is_on, _before = torch._C._is_tracing, torch._C._dispatch_tls_is_dispatch_key_included, torch._C.DispatchKey.PreDispatch


def _recorded():
    """Is a graph being recorded of the calls that are made (make_fx, torch.jit.trace)?  A kernel's launch would not be in it, only the memory that it
    was about to fill."""
    return _tracing() or _modes() > 0 and _mode(_proxies) is not None or _key_is_on(_before)


def _refuse_recording(who):
    if not torch.compiler.is_compiling() and _recorded():      # (the compiler leaves such a call out of its graph)
        raise RuntimeError("%s: the call cannot be recorded in a graph (make_fx, torch.jit.trace)" % who)


def _issue(t, launch):
    """On the current stream of the tensor's device, whichever device is the current one."""
    index = t.get_device()
    if _current_device() == index:
        launch(_raw_stream(index))
    else:
        with torch.cuda.device(index):
            launch(_raw_stream(index))


def _call(t, entry, *args):
    """An entry point of the library at once, on the current stream of the tensor's device."""
    index = t.get_device()
    fn = getattr(_tables[index].lib, entry)
    if _current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc != 0:
        raise RuntimeError("%s failed: %s" % (entry, _tables[index].lib.pf_last_error().decode()))


def _need(t, entry, *args, who=None):
    """Bytes that an entry point asks for; who: refuses in its place."""
    lib = _tables[t.get_device()].lib
    need = getattr(lib, entry)(*args)
    if need < 0:
        said = lib.pf_last_error().decode()
        raise RuntimeError(said if who is None else said.replace(entry, who, 1))
    return need


def _at(t):
    return None if t is None else t.data_ptr()


# the level of forward-mode differentiation, -1 outside of it
_dual = forward_ad if hasattr(forward_ad, "_current_level") else SimpleNamespace(_current_level=0)


def _has_tangent(*tensors):
    """Is one of them a dual number of forward-mode differentiation?  (Such a tensor need not require a gradient.)  Asked at a level of it."""
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


_LOGITS = (torch.float32, torch.float16, torch.bfloat16)
_CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}      # (PF_F32, PF_F16, PF_BF16)


def _check_rows(who, logits, labels, ignore_index, temperature, shift):
    """What the three losses ask of their logits and labels.  -> (logits [B, T, V] with unit stride over the classes, labels [B, T])"""
    if not torch.is_tensor(logits) or not torch.is_tensor(labels):
        raise RuntimeError("%s: logits and labels are tensors" % who)
    _refuse_recording(who)
    _table(logits, who)
    shape = logits.shape
    if logits.dtype not in _LOGITS:
        raise RuntimeError("%s: logits are fp32, fp16 or bf16 (got %s)" % (who, logits.dtype))
    if len(shape) < 2 or shape[-1] == 0:
        raise RuntimeError("%s: logits are [..., tokens, classes] (got %s)" % (who, tuple(shape)))
    if labels.dtype != torch.int64 or labels.get_device() != logits.get_device() or labels.shape != shape[:-1]:
        raise RuntimeError("%s: labels are int64 %s on %s (got %s %s on %s)"
                           % (who, tuple(shape[:-1]), logits.device, labels.dtype, tuple(labels.shape), labels.device))
    if not isinstance(ignore_index, int) or not isinstance(shift, (bool, int)) or shift not in (0, 1):
        raise RuntimeError("%s: ignore_index is a whole number and shift a truth value" % who)
    if not 1e-6 <= temperature <= 1e6:
        raise RuntimeError("%s: temperature must lie in [1e-6, 1e6] (got %s)" % (who, temperature))
    if _dual._current_level >= 0 and _has_tangent(logits):
        raise RuntimeError("%s: there is no forward-mode derivative" % who)
    if len(shape) != 3:
        logits = logits.reshape((math.prod(shape[:-2]),) + shape[-2:])
        labels = labels.reshape(logits.shape[:-1])
    if logits.stride(-1) != 1 and shape[-1] > 1:
        logits = logits.contiguous()
    return logits, labels.contiguous()


def _constant(who, name, t, shapes, like):
    """An operand that no gradient flows to, fp32 on the logits' device, of one of these shapes."""
    if not torch.is_tensor(t) or not t.is_floating_point() or t.get_device() != like.get_device() or t.shape not in shapes:
        raise RuntimeError("%s: %s is a floating tensor of shape %s on %s (got %s)"
                           % (who, name, " or ".join(map(str, shapes)), like.device,
                              "%s %s on %s" % (t.dtype, tuple(t.shape), t.device) if torch.is_tensor(t) else type(t).__name__))
    if t.requires_grad or _dual._current_level >= 0 and _has_tangent(t):
        raise RuntimeError("%s: no gradient flows to %s: detach it" % (who, name))
    return t if t.dtype == torch.float32 else t.to(torch.float32)


def _rows(logits, labels, cfg):
    """The kernels' description of the rows; cfg = (shift, ignore_index, temperature)."""
    return _table(logits, "").token_rows(logits, *logits.shape, *logits.stride()[:2], labels, *cfg)


def _new(like, *shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device=like.device)


def _logits_gradient(ctx, logits, labels, stats, coef, g_strides, keep, scale=None, into=None, unless_one=0):
    """stats, coef: addresses within `keep`; scale: a tensor of one element.  Autograd calls this on a thread of its own, which finds little in its
    core's caches: it does no more than it must, and takes the forward pass's description of the rows where they still lie there."""
    rows, strides, k, scaled = ctx.rows
    if logits.data_ptr() != rows[0] or labels.data_ptr() != rows[7] or logits.stride() != strides:      # (hooks may move what is saved)
        rows = _rows(logits, labels, rows[8:])
    d = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device) if into is None else into
    index = logits.get_device()
    at = None if scale is None else scale.data_ptr()
    if _current_device() == index:
        k.token_gradient(rows, stats, coef, g_strides, d, at, unless_one, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            k.token_gradient(rows, stats, coef, g_strides, d, at, unless_one, _raw_stream(index))
    if scaled:
        d._pf_times = d._version, functools.partial(_gradient_times, k, rows, stats, coef, g_strides, scale, (logits, labels, keep))
    return d


def _gradient_times(k, rows, stats, coef, g_strides, scale, keep, factor, out):
    """The gradient times a loss scale, rounded once, where multiplying the fp16 gradient would find its small entries gone; -> is it written."""
    like = keep[0]
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device or out.stride(-1) != 1:
        return False
    by = factor if scale is None else scale * factor
    k.token_gradient(rows, stats, coef, g_strides, out, by.data_ptr(), 0, _raw_stream(out.get_device()))
    return True


def mark_loss_scaled(output):
    """Notes that the gradient of this output of a runner will be multiplied by a loss scale: a token loss of it, if it is in fp16, then leaves
    with its gradient how to form the product itself (`scaled_gradient`)."""
    output._pf_loss_scaled = True


def scaled_gradient(grad, factor, out):
    """`out` = grad times `factor` (fp32 on the device, of one element) from what a token loss left with it, on the current stream; -> is it written.
    Not where the gradient is a sum of several or was changed."""
    version, write = getattr(grad, "_pf_times", (None, None))
    return write is not None and grad._version == version and write(factor, out)


def _wants_scale(logits):
    return logits.dtype == torch.float16 and getattr(logits, "_pf_loss_scaled", False)


def _as_scale(g):
    return g if g.dtype == torch.float32 else g.to(torch.float32)


class _NoContext:
    """Stands for autograd's where no gradient is asked for: its bookkeeping takes longer than a small call."""

    @staticmethod
    def mark_non_differentiable(*_):
        pass

    @staticmethod
    def set_materialize_grads(_):
        pass


def _apply(fn, logits, *args):
    if torch.is_grad_enabled() and logits.requires_grad:
        return fn.apply(logits, args)
    return fn.forward(_NoContext, logits, args, False)


def _once(backward):
    """torch.autograd.function.once_differentiable where it matters: a backward pass that keeps no graph does not pay for it."""
    wrapped = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        if _dual._current_level >= 0 and _has_tangent(*grads):
            raise RuntimeError("a backward pass of the token losses has no forward-mode derivative")
        return (wrapped if torch.is_grad_enabled() else backward)(ctx, *grads)

    return staticmethod(run)


class _TokenLogprobFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, args, want=True):
        labels, cfg = args
        B, T, _ = logits.shape
        out = _new(logits, B, max(0, T - cfg[0]))
        stats = _new(logits, *out.shape, 2) if want else None
        k, rows = _table(logits, ""), _rows(logits, labels, cfg)
        _issue(logits, k.token_logprob_fwd(rows, out, stats))
        if want:
            ctx.save_for_backward(logits, labels, stats)
            ctx.rows = rows, logits.stride(), k, _wants_scale(logits)
        return out

    @_once
    def backward(ctx, grad):
        logits, labels, stats = ctx.saved_tensors
        grad = _as_scale(grad)      # (any strides: a sum's gradient is one number)
        return _logits_gradient(ctx, logits, labels, stats.data_ptr(), grad.data_ptr(), grad.stride(), (stats, grad)), None


class _PreferenceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, args, want=True):
        labels, ref, cfg, beta, smoothing, average = args
        B, T, _ = logits.shape
        k = _table(logits, "")
        rows = _rows(logits, labels, cfg)
        n, scored = k.preference_workspace(B, T, cfg[0]), B * max(0, T - cfg[0])
        # the kernels' scratch, and behind it what the backward pass takes: {reference, 1 / sum} of every row, a factor of every sequence
        work = _new(logits, n + scored + (B + 1) // 2, dtype=torch.float64)
        at = work.data_ptr()
        stats, coef = at + 8 * n, at + 8 * (n + scored)
        loss, rewards = _new(logits), _new(logits, B)
        _issue(logits, k.preference_loss(rows, ref, beta, smoothing, average, loss, rewards, stats if want else None, coef, work))
        if want:
            ctx.save_for_backward(logits, labels, work)
            ctx.rows, ctx.at = (rows, logits.stride(), k, _wants_scale(logits)), (8 * n, 8 * (n + scored))
        ctx.mark_non_differentiable(rewards)
        ctx.set_materialize_grads(False)
        return loss, rewards

    @_once
    def backward(ctx, grad, _):
        logits, labels, work = ctx.saved_tensors      # (not always where it was: hooks may have moved it)
        if grad is None:
            return None, None
        at, (stats, coef), grad = work.data_ptr(), ctx.at, _as_scale(grad)
        return _logits_gradient(ctx, logits, labels, at + stats, at + coef, (1, 0), work, grad), None


_saving_hooks = getattr(torch._C._autograd, "_top_saved_tensors_default_hooks", lambda ignore_is_tracing: None)


class _PolicyFn(torch.autograd.Function):
    """The gradient of a loss that is itself the end (`loss.backward()`) is written by the forward pass, which has the row at
    hand: a token's part of it depends on its own row alone.  The backward pass looks at what it is asked to multiply it
    by, on the device: by one it has nothing to do, by anything else it computes the gradient from the logits.  It does so too where
    hooks take what is saved (off the device, or to forget it): they are there to save memory, and the gradient is as large as the logits."""

    @staticmethod
    def forward(ctx, logits, args, want=True):
        labels, old, adv, a_strides, ref, cfg, clip, kl_coef, by_sequence, scale = args
        B, T, _ = logits.shape
        k, rows = _table(logits, ""), _rows(logits, labels, cfg)
        R = max(0, T - cfg[0])
        n = k.policy_workspace(B, T, cfg[0])
        loss, kl, logprobs = _new(logits), _new(logits), _new(logits, B, R)
        stats = coef = d = None
        strides = (0, 0)
        if want:      # behind the kernels' scratch what the backward pass takes: {reference, 1 / sum} and a factor of every row
            work = _new(logits, n + B * R + (B * R + 1) // 2, dtype=torch.float64)
            stats = work.data_ptr() + 8 * n
            coef = stats + 8 * B * R
            if _saving_hooks(False) is None:
                d = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
                strides = d.stride()[:2]
        else:
            work = _new(logits, n, dtype=torch.float64)
        _issue(logits, k.policy_loss(rows, old, adv, a_strides, ref, *clip, kl_coef, by_sequence, scale, loss, kl, logprobs, stats, coef, d, strides, work))
        if want:
            ctx.save_for_backward(logits, labels, work)
            ctx.rows, ctx.at = (rows, logits.stride(), k, _wants_scale(logits)), (8 * n, 8 * (n + B * R), (R, 1))
            ctx.d, ctx.captured = d, torch.cuda.is_current_stream_capturing()
        ctx.mark_non_differentiable(logprobs, kl)
        ctx.set_materialize_grads(False)
        return loss, logprobs, kl

    @_once
    def backward(ctx, grad, *_):
        logits, labels, work = ctx.saved_tensors
        if grad is None:
            return None, None
        # handed out once (what has it may change it), and not from an eager forward pass to a graph, whose replays would find it
        # changed
        d, ctx.d = ctx.d, None
        if d is not None and ctx.captured != torch.cuda.is_current_stream_capturing():
            d = None
        at, (stats, coef, strides), grad = work.data_ptr(), ctx.at, _as_scale(grad)
        return _logits_gradient(ctx, logits, labels, at + stats, at + coef, strides, work, grad, d, 0 if d is None else 1), None


def token_logprobs(logits, labels, *, ignore_index=-100, temperature=1.0, shift=False):
    """Log-probabilities of the labels: log softmax(logits / temperature)[label], fp32, with the gradient to the logits.

    logits [..., T, V] (fp32, fp16 or bf16), labels int64 [..., T].  shift: row t is scored against label t + 1 (labels as
    the model's own input), the result has T - 1 tokens.  Tokens whose label is `ignore_index` give 0 and take no part, whatever
    their logits hold; labels outside the vocabulary give NaN.  There are no second and no forward-mode derivatives.  A
    backward pass is captured into a graph, as any of torch's, only while no autograd graph made outside the capture holds the same
    leaves."""
    x, y = _check_rows("token_logprobs", logits, labels, ignore_index, temperature, shift)
    cfg = (int(shift), ignore_index, float(temperature))
    out = _apply(_TokenLogprobFn, x, y, cfg)
    return out if logits.dim() == 3 else out.reshape(logits.shape[:-2] + out.shape[1:])


def preference_loss(logits, labels, ref_logprobs, *, beta=0.1, label_smoothing=0.0, length_average=False, ignore_index=-100, shift=False):
    """Preference loss over pairs of answers; -> (loss, rewards).

    logits [2P, T, V], labels int64 [2P, T]: sequences 2i (preferred) and 2i + 1 (rejected) are a pair, so that a batch split into
    micro-batches of whole pairs keeps them together.  ref_logprobs [2P]: the sum (length_average: the mean) of the answer's
    token log-probabilities under the reference model (of no token: 0).  With s the same of this model, rewards = beta (s - ref) and D the preferred
    minus the rejected reward, loss = mean of -(1 - label_smoothing) log sigmoid(D) - label_smoothing log sigmoid(-D).  The
    gradient flows to the logits; `rewards` [2P] are for the log.  `shift` and `ignore_index` as for `token_logprobs`."""
    who = "preference_loss"
    x, y = _check_rows(who, logits, labels, ignore_index, 1.0, shift)
    B = logits.shape[0]
    if logits.dim() != 3 or B == 0 or B % 2:
        raise RuntimeError("%s: logits are [2 * pairs, tokens, classes] (got %s)" % (who, tuple(logits.shape)))
    if not math.isfinite(beta) or not 0.0 <= label_smoothing <= 1.0:
        raise RuntimeError("%s: beta must be finite and label_smoothing lie in [0, 1]" % who)
    ref = _constant(who, "ref_logprobs", ref_logprobs, [(B,)], logits).contiguous()
    return _apply(_PreferenceFn, x, y, ref, (int(shift), ignore_index, 1.0), float(beta), float(label_smoothing), bool(length_average))


def policy_loss(logits, labels, old_logprobs, advantages, ref_logprobs=None, *, clip=0.2, clip_high=None, kl_coef=0.0, temperature=1.0,
                reduction="tokens", scale=1.0, ignore_index=-100, shift=False):
    """Clipped policy loss of sampled tokens with a KL term; -> (loss, logprobs, kl).

    logits [B, T, V], labels int64 [B, T] (the tokens that were sampled), old_logprobs [B, T'] under the policy that sampled them,
    advantages [B], [B, 1] or [B, T'], ref_logprobs [B, T'] under a reference model (T' = T - 1 with `shift`, else T).  With r =
    exp(logprob - old) a token's loss is -min(r A, clamp(r, 1 - clip, 1 + clip_high) A) + kl_coef (exp(ref - logprob) - (ref -
    logprob) - 1); clip_high defaults to clip.  reduction "tokens": the mean over all tokens that count; "sequences": the mean over
    the sequences that have such tokens of their means; with none at all the loss is 0.  `scale` multiplies the loss (not `kl`): a factor given here is free, one that the loss is
    multiplied by afterwards has the backward pass compute the gradient anew.  The gradient flows to the logits alone;
    `logprobs` [B, T'] and `kl` (the KL term's mean) are for the log.  `ignore_index`, `shift` and `temperature` as for
    `token_logprobs`; what the other operands hold at ignored tokens does not matter.  A backward pass captured into a graph of its own is
    replayed once for every replay of the forward pass's graph."""
    who = "policy_loss"
    x, y = _check_rows(who, logits, labels, ignore_index, temperature, shift)
    if logits.dim() != 3:
        raise RuntimeError("%s: logits are [sequences, tokens, classes] (got %s)" % (who, tuple(logits.shape)))
    clip_high = clip if clip_high is None else clip_high
    if not (0.0 <= clip < math.inf and 0.0 <= clip_high < math.inf) or not math.isfinite(kl_coef) or not math.isfinite(scale):
        raise RuntimeError("%s: clip and clip_high must not be negative, and all coefficients finite" % who)
    if reduction not in ("tokens", "sequences"):
        raise RuntimeError("%s: reduction is 'tokens' or 'sequences' (got %r)" % (who, reduction))
    if ref_logprobs is None and kl_coef != 0.0:
        raise RuntimeError("%s: a KL term needs ref_logprobs" % who)
    B, T = y.shape
    R = max(0, T - int(shift))
    old = _constant(who, "old_logprobs", old_logprobs, [(B, R)], logits).contiguous()
    adv = _constant(who, "advantages", advantages, [(B,), (B, 1), (B, R)], logits)
    ref = None if ref_logprobs is None else _constant(who, "ref_logprobs", ref_logprobs, [(B, R)], logits).contiguous()
    a_strides = (adv.stride(0), adv.stride(1) if adv.dim() == 2 and adv.shape[1] > 1 else 0)
    return _apply(_PolicyFn, x, y, old, adv, a_strides, ref, (int(shift), ignore_index, float(temperature)), (float(clip), float(clip_high)),
                  float(kl_coef), reduction == "sequences", float(scale))


class _LinearCrossEntropyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, args, want=True):
        labels, shift, ignore_index, z_loss, reduction = args
        B, T, D = hidden.shape
        V, dtype, dev = weight.shape[0], _CODE[hidden.dtype], hidden.device
        head = (hidden.data_ptr(), dtype, B, T, D, *hidden.stride()[:2], weight.data_ptr(), V)
        kept = torch.empty((_need(hidden, "pf_linear_ce_kept", B * T),), dtype=torch.uint8, device=dev)
        work = torch.empty((_need(hidden, "pf_linear_ce_workspace", head[7], dtype, B * T, D, V, 0),), dtype=torch.uint8, device=dev)
        loss = torch.empty((B, max(0, T - shift)) if reduction == 0 else (), dtype=torch.float32, device=dev)
        _call(hidden, "pf_linear_ce_fwd", *head, labels.data_ptr(), shift, ignore_index, z_loss, reduction, loss.data_ptr(), kept.data_ptr(), work.data_ptr())
        if want:
            ctx.save_for_backward(hidden, weight, kept)
            ctx.cfg = z_loss, reduction, _wants_scale(hidden)
        return loss

    @_once
    def backward(ctx, grad):
        hidden, weight, kept = ctx.saved_tensors
        z_loss, reduction, scaled = ctx.cfg
        B, T, D = hidden.shape
        if grad.numel() == 0:      # ("none" of no token: a gradient without an address)
            return *(torch.zeros(t.shape, dtype=t.dtype, device=t.device) if n else None for t, n in zip((hidden, weight), ctx.needs_input_grad)), None
        V, dtype, dev = weight.shape[0], _CODE[hidden.dtype], hidden.device
        head = (hidden.data_ptr(), dtype, B, T, D, *hidden.stride()[:2], weight.data_ptr(), V)
        work = torch.empty((_need(hidden, "pf_linear_ce_workspace", head[7], dtype, B * T, D, V, 1),), dtype=torch.uint8, device=dev)
        dh = torch.empty((B, T, D), dtype=hidden.dtype, device=dev) if ctx.needs_input_grad[0] else None
        dw = torch.empty((V, D), dtype=weight.dtype, device=dev) if ctx.needs_input_grad[1] else None
        grad = _as_scale(grad)      # (any strides: a sum's gradient is one number)
        strides = grad.stride() if reduction == 0 else (0, 0)
        _call(hidden, "pf_linear_ce_bwd", *head, z_loss, int(reduction == 1), kept.data_ptr(), grad.data_ptr(), *strides, _at(dh), _at(dw), work.data_ptr())
        if scaled and dh is not None:
            # (not dh itself: a cycle would keep the workspace until Python looks for one; of the weight only where it lies)
            dh._pf_times = dh._version, functools.partial(_hidden_times, (head[7], dtype, B * T, D, V), (dh.shape, dh.dtype, dh.device), kept, work)
        return dh, dw, None


def _hidden_times(sizes, like, kept, work, factor, out):
    """The hidden state's gradient times a loss scale, rounded once, from the fp32 sums that the backward pass left; -> is it written."""
    if (out.shape, out.dtype, out.device) != like or not out.is_contiguous():
        return False
    _call(out, "pf_linear_ce_hidden_grad", *sizes, kept.data_ptr(), factor.data_ptr(), out.data_ptr(), work.data_ptr())
    return True


_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def linear_cross_entropy(hidden, weight, labels, *, ignore_index=-100, z_loss=0.0, reduction="mean", shift=False):
    """Cross entropy of the classes' logits hidden @ weight.T, which are never in memory: they are formed in pieces of the vocabulary, in
    fp32, and formed again by the backward pass.

    hidden [..., T, D] and weight [V, D] (fp32, fp16 or bf16, the same type), labels int64 [..., T].  A token's loss is lse - logit[label] +
    z_loss * lse^2, lse = log sum exp of its logits.  reduction "mean": over the tokens that count (with none of them 0), "sum", or "none": fp32
    [..., T], 0 where a token does not count.  shift: token t is scored against label t + 1 (labels as the model's own input), the last
    dimension of "none" is then T - 1.  Tokens whose label is `ignore_index` take no part, whatever their hidden state holds, and cost no
    arithmetic; a label outside the vocabulary gives NaN.  The gradient flows to hidden and weight, in their types.  For a weight of
    another type hand in `weight.to(hidden.dtype)`.  There are no second and no forward-mode derivatives.  A backward pass is captured
    into a graph, as any of torch's, only while no autograd graph made outside the capture holds the same leaves."""
    who = "linear_cross_entropy"
    if not torch.is_tensor(hidden) or not torch.is_tensor(weight) or not torch.is_tensor(labels):
        raise RuntimeError("%s: hidden, weight and labels are tensors" % who)
    _refuse_recording(who)
    _table(hidden, who)
    shape = hidden.shape
    if hidden.dtype not in _LOGITS or weight.dtype != hidden.dtype:
        raise RuntimeError("%s: hidden and weight are both fp32, fp16 or bf16 (got %s and %s)" % (who, hidden.dtype, weight.dtype))
    if len(shape) < 2 or shape[-1] == 0:
        raise RuntimeError("%s: hidden is [..., tokens, width] (got %s)" % (who, tuple(shape)))
    if weight.dim() != 2 or weight.shape[1] != shape[-1] or weight.shape[0] == 0 or weight.get_device() != hidden.get_device():
        raise RuntimeError("%s: weight is [classes, %d] on %s (got %s on %s)" % (who, shape[-1], hidden.device, tuple(weight.shape), weight.device))
    if labels.dtype != torch.int64 or labels.get_device() != hidden.get_device() or labels.shape != shape[:-1]:
        raise RuntimeError("%s: labels are int64 %s on %s (got %s %s on %s)"
                           % (who, tuple(shape[:-1]), hidden.device, labels.dtype, tuple(labels.shape), labels.device))
    if not isinstance(ignore_index, int) or not isinstance(shift, (bool, int)) or shift not in (0, 1):
        raise RuntimeError("%s: ignore_index is a whole number and shift a truth value" % who)
    if reduction not in _REDUCTIONS:
        raise RuntimeError("%s: reduction is 'mean', 'sum' or 'none' (got %r)" % (who, reduction))
    if not math.isfinite(z_loss):
        raise RuntimeError("%s: z_loss must be finite" % who)
    if _dual._current_level >= 0 and _has_tangent(hidden, weight):
        raise RuntimeError("%s: there is no forward-mode derivative" % who)
    x = hidden
    if len(shape) != 3:
        x = x.reshape((math.prod(shape[:-2]),) + shape[-2:])
    if x.stride(-1) != 1 and shape[-1] > 1:
        x = x.contiguous()
    args = (labels.reshape(x.shape[:-1]).contiguous(), int(shift), ignore_index, float(z_loss), _REDUCTIONS[reduction])
    weight = weight.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        tokens = x.shape[0] * x.shape[1]
        if (tokens + 64) * (shape[-1] + 64) >= 1 << 28:      # (fewer are never too many for a gradient)
            _need(x, "pf_linear_ce_workspace", weight.data_ptr(), _CODE[x.dtype], tokens, shape[-1], weight.shape[0], 1, who=who)
        out = _LinearCrossEntropyFn.apply(x, weight, args)
    else:
        out = _LinearCrossEntropyFn.forward(_NoContext, x, weight, args, False)
    return out.reshape(shape[:-2] + out.shape[1:]) if reduction == "none" and len(shape) != 3 else out


class LossWrapper(nn.Module):
    def forward(self, input, target, model=None):
        return _SumFn.apply(input)


class SumLoss(LossWrapper):
    def forward(self, input, target, model=None):
        if isinstance(input, (tuple, list)):
            input = input[0]
        return _SumFn.apply(input)


class MaskedLMOutputLoss(LossWrapper):
    def forward(self, input, target, model=None):
        if input.loss is not None:
            return input.loss
        return _SumFn.apply(input.logits)


class RescaleLoss(LossWrapper):
    def __init__(self, loss_fn, scale=1.0):
        super().__init__()
        self.loss_fn = loss_fn
        self.scale = scale

    def forward(self, input, target, model=None):
        return self.loss_fn(input, target, model) * self.scale


class NormalizeLoss(LossWrapper):
    """Rescales the loss by powers of two until 1/2 <= |loss| <= 1 (host-synchronising)."""

    def __init__(self, loss_fn):
        super().__init__()
        self.loss_fn = loss_fn

    def forward(self, input, target, model=None):
        loss = self.loss_fn(input, target, model)
        if loss.item() == 0:
            return loss
        while abs(loss.item()) < 1:
            loss = loss * 2
        while abs(loss.item()) > 1:
            loss = loss / 2
        return loss


class CrossEntropyLoss(LossWrapper):
    def __init__(self, num_labels=10):
        super().__init__()
        self.num_labels = num_labels

    def forward(self, input, target, model=None):
        return cross_entropy(input.view(-1, self.num_labels), target)


class HFCrossEntropyLoss(LossWrapper):
    def __init__(self, num_labels=10):
        super().__init__()
        self.num_labels = num_labels

    def forward(self, input, target, model=None):
        return cross_entropy(input.logits.view(-1, self.num_labels), target)


class PreferenceLoss(LossWrapper):
    """`preference_loss` of the logits (or of an output that has `.logits`); target: (labels, ref_logprobs)."""

    def __init__(self, **kwargs):
        super().__init__()
        self.kwargs = kwargs

    def forward(self, input, target, model=None):
        labels, ref_logprobs = target
        return preference_loss(getattr(input, "logits", input), labels, ref_logprobs, **self.kwargs)[0]


class PolicyLoss(LossWrapper):
    """`policy_loss` of the logits (or of an output that has `.logits`); target: (labels, old_logprobs, advantages[, ref_logprobs])."""

    def __init__(self, **kwargs):
        super().__init__()
        self.kwargs = kwargs

    def forward(self, input, target, model=None):
        return policy_loss(getattr(input, "logits", input), *target, **self.kwargs)[0]
