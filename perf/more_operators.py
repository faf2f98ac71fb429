"""Operators of a decoder's training step around its attention: the token table's lookup with the gradient by sorted tokens, a
gated projection (both products, the activation and their product) whose backward pass may start from pre-activations held in 8
bits, and the cross entropy of a large vocabulary from the last hidden state, whose logits are never in memory at once.

A case is one call of one operator, with its backward pass where it trains.  `run` makes it through `pfeife_amd` where `own` is
true, and in elementary torch operations where it is false.
"""
import math

import numpy as np
import torch

own = False

IGNORE = -100
BLOCK = 16            # neighbouring columns of a row whose 8-bit codes share an exponent
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _head(name, dtype, batch, seq, dim, vocab, **more):
    case = dict(name=name, op="head", dtype=dtype, batch=batch, seq=seq, dim=dim, vocab=vocab, shift=False, prompt=0, ragged=0,
                z_loss=0.0, reduction="mean", up=1.0, train=True)
    case.update(more)
    return case


def _table(name, dtype, tokens, vocab, dim, **more):
    case = dict(name=name, op="table", dtype=dtype, tokens=tokens, vocab=vocab, dim=dim, scale=1.0, skew=3.0, hot=0.0, padding=False,
                train=True)
    case.update(more)
    return case


def _gated(name, dtype, rows, dim, ffn, **more):
    case = dict(name=name, op="gated", dtype=dtype, rows=rows, dim=dim, ffn=ffn, act="silu", kept="16bit", train=True)
    case.update(more)
    return case


def listed():
    return [
        # the last token of each of sixteen answers, scored: the weight is read once, and nothing else takes long
        _head("head_scores_bf16", "bf16", 16, 1, 2048, 32000, train=False, reduction="none"),
        # full precision, an odd vocabulary, a prompt and padding that take no part, a gradient of every token's own
        _head("head_tokens_fp32", "fp32", 4, 255, 384, 10007, shift=True, prompt=31, ragged=60, reduction="none"),
        # half precision under a loss scale, rows and classes that fill no tile, the log normalizer held near zero
        _head("head_ragged_fp16", "fp16", 6, 777, 1000, 49999, shift=True, prompt=100, ragged=300, z_loss=1e-4, up=65536.0),
        # a micro-batch of the 1B decoder at its own sequence length
        _head("head_decoder_bf16", "bf16", 4, 2048, 2048, 32000, shift=True),
        # a large vocabulary on a wide model
        _head("head_vocabulary_bf16", "bf16", 2, 1024, 4096, 131072, shift=True, prompt=128, ragged=200),
        # one token of each of sixteen sequences: latency alone
        _table("table_tokens_bf16", "bf16", 16, 32000, 2048, train=False, scale=2048 ** 0.5),
        # a batch of the 1B decoder, tokens as frequent as text has them
        _table("table_decoder_bf16", "bf16", 16384, 32000, 2048, scale=2048 ** 0.5),
        # odd sizes in full precision, a third of the tokens the same, a padding token that learns nothing
        _table("table_hot_fp32", "fp32", 50021, 10007, 769, hot=0.33, padding=True),
        # one token through the feed-forward block of the 1B decoder: the weight's way to the chip
        _gated("gated_token_bf16", "bf16", 1, 2048, 5632, train=False),
        # odd rows and widths in half precision, another activation
        _gated("gated_ragged_fp16", "fp16", 777, 1000, 2732, act="gelu"),
        # the same block on a micro-batch of four sequences
        _gated("gated_decoder_bf16", "bf16", 8192, 2048, 5632),
        # ... and on eight, what its backward pass starts from held in 8 bits
        _gated("gated_kept8_bf16", "bf16", 16384, 2048, 5632, kept="8bit"),
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("head", "table", "gated"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op == "head":
        dim = _spread(rng, 64, 4096) if rng.random() < 0.4 else 64 * _spread(rng, 1, 64)
        vocab = _spread(rng, 500, 131072)
        rows = _spread(rng, 1, max(1, min(16384, int((4e10 if dtype == "fp32" else 1e12) / (dim * vocab)))))
        batch = min(rows, rng.randint(1, 8))
        seq = max(1, rows // batch)
        shift = seq > 1 and rng.random() < 0.6
        case = _head("", dtype, batch, seq, dim, vocab, shift=shift, prompt=rng.randint(0, seq // 2),
                     ragged=rng.randint(0, seq // 3), z_loss=rng.choice((0.0, 0.0, 1e-4)), reduction=rng.choice(("mean", "sum", "none")),
                     up=65536.0 if dtype == "fp16" else 1.0, train=rng.random() < 0.8)
        if case["reduction"] != "mean" and dtype == "fp16":
            case["up"] = 64.0
    elif op == "table":
        dim = _spread(rng, 32, 4096) - rng.choice((0, 0, 1))
        vocab = _spread(rng, 300, 131072)
        case = _table("", dtype, _spread(rng, 1, min(200_000, 150_000_000 // dim)), vocab, dim, scale=rng.choice((1.0, 0.5, dim ** 0.5)),
                      skew=rng.choice((1.0, 2.0, 3.0)), hot=rng.choice((0.0, 0.0, 0.2, 0.5)), padding=rng.random() < 0.4,
                      train=rng.random() < 0.8)
    else:
        dim = _spread(rng, 64, 4096) if rng.random() < 0.4 else 64 * _spread(rng, 1, 64)
        ffn = _spread(rng, 64, 14336) if rng.random() < 0.4 else 32 * _spread(rng, 2, 448)
        rows = _spread(rng, 1, max(1, min(32768, int((1e10 if dtype == "fp32" else 1.5e11) / (dim * ffn)))))
        case = _gated("", dtype, rows, dim, ffn, act=rng.choice(("silu", "silu", "gelu", "gelu_tanh", "relu")), train=rng.random() < 0.8)
        if case["train"] and dtype != "fp32" and rng.random() < 0.5:
            case["kept"] = "8bit"
    del case["name"]
    return case


def _counted(case):
    """[first, last) label positions of every sequence that are scored: answers of different length behind a prompt."""
    spans = []
    for b in range(case["batch"]):
        last = case["seq"] - (b * case["ragged"]) // max(1, case["batch"] - 1)
        first = max(case["prompt"], 1 if case["shift"] else 0)
        spans.append((first, max(first, last)))
    return spans


def _distinct(case):
    """How many tokens of the table a batch is expected to hold."""
    edge = (np.arange(case["vocab"] + 1) / case["vocab"]) ** (1.0 / case["skew"])
    return 1.0 + float(-np.expm1(case["tokens"] * (1.0 - case["hot"]) * np.log1p(-np.minimum(np.diff(edge), 1 - 1e-12))).sum())


def work(case):
    size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    if case["op"] == "head":
        rows = sum(last - first for first, last in _counted(case))
        every, weight = case["batch"] * case["seq"], case["vocab"] * case["dim"]
        # hidden state, weight and labels read; their gradients written (a row that takes no part has one of zeros)
        moved = (rows * case["dim"] + weight) * size + every * 8
        if case["train"]:
            moved += (every * case["dim"] + weight) * size
        return {"bytes": float(moved), "flops": (6.0 if case["train"] else 2.0) * rows * weight}
    if case["op"] == "table":
        n, dim = case["tokens"], case["dim"]
        moved = n * 8 + (_distinct(case) + n) * dim * size
        if case["train"]:
            moved += (n + case["vocab"]) * dim * size
        return {"bytes": float(moved), "flops": (2.0 if case["train"] else 1.0) * n * dim}
    n, weight = case["rows"], 2 * case["ffn"] * case["dim"]
    once = (n * (case["dim"] + case["ffn"]) + weight) * size
    return {"bytes": float(2 * once if case["train"] else once), "flops": (6.0 if case["train"] else 2.0) * n * weight}


# -- inputs -----------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(2000 + seed)
    rnd = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    dtype = DTYPES[case["dtype"]]
    state = dict(case=case)
    if case["op"] == "head":
        B, T, D, V = case["batch"], case["seq"], case["dim"], case["vocab"]
        weight = torch.empty(V, D, device="cuda", dtype=dtype)
        for part in weight.split(16384):
            part.copy_(rnd(*part.shape) * D ** -0.5)
        labels = torch.randint(0, V, (B, T), device="cuda", generator=gen)
        s = 1 if case["shift"] else 0
        hidden = rnd(B, T, D)
        hidden[:, :T - s] += (2.0 + 5.0 * torch.rand(B, T - s, 1, device="cuda", generator=gen)) * weight[labels[:, s:]].float()
        for b, (first, last) in enumerate(_counted(case)):
            labels[b, :first] = IGNORE
            labels[b, last:] = IGNORE
        up = torch.full((), case["up"], device="cuda")
        if case["reduction"] == "none":      # every token its own weight
            up = up * (0.5 + torch.rand(B, T - s, device="cuda", generator=gen))
        state.update(hidden=hidden.to(dtype), weight=weight, labels=labels, up=up)
    elif case["op"] == "table":
        n, V, D = case["tokens"], case["vocab"], case["dim"]
        u = torch.rand(n, device="cuda", generator=gen, dtype=torch.float64)
        ids = (u ** case["skew"] * V).long().clamp_(max=V - 1)
        if case["hot"]:
            ids = torch.where(torch.rand(n, device="cuda", generator=gen) < case["hot"], V // 3, ids)
        state.update(ids=ids, weight=(0.02 * rnd(V, D)).to(dtype), up=(1e-2 * rnd(n, D)).to(dtype),
                     padding=V // 7 if case["padding"] else None)
    else:
        n, D, F = case["rows"], case["dim"], case["ffn"]
        state.update(x=rnd(n, D).to(dtype), weight=(D ** -0.5 * rnd(2 * F, D)).to(dtype), up=(1e-2 * rnd(n, F)).to(dtype))
    return state


# -- one pass ---------------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    return (_own if own else _plain)[case["op"]](case, state)


def _own_head(case, state):
    from pfeife_amd.loss import linear_cross_entropy

    h = state["hidden"].detach().requires_grad_(case["train"])
    w = state["weight"].detach().requires_grad_(case["train"])
    loss = linear_cross_entropy(h, w, state["labels"], shift=case["shift"], z_loss=case["z_loss"], reduction=case["reduction"])
    if not case["train"]:
        return loss
    return (loss.detach(),) + torch.autograd.grad(loss, (h, w), state["up"])


def _own_table(case, state):
    from pfeife_amd.layers import embedding

    w = state["weight"].detach().requires_grad_(case["train"])
    out = embedding(state["ids"], w, scale=case["scale"], padding_idx=state["padding"])
    if not case["train"]:
        return out
    return out.detach(), torch.autograd.grad(out, w, state["up"])[0]


def _own_gated(case, state):
    from pfeife_amd.layers import gated_linear

    x = state["x"].detach().requires_grad_(case["train"])
    w = state["weight"].detach().requires_grad_(case["train"])
    y = gated_linear(x, w, act=case["act"], kept=case["kept"])
    if not case["train"]:
        return y
    return (y.detach(),) + torch.autograd.grad(y, (x, w), state["up"])


_own = {"head": _own_head, "table": _own_table, "gated": _own_gated}


def _plain_head(case, state):
    B, T, D = state["hidden"].shape
    s = 1 if case["shift"] else 0
    x, w = state["hidden"][:, :T - s].float(), state["weight"].float()
    labels = state["labels"][:, s:]
    seen = labels != IGNORE
    at = torch.where(seen, labels, 0).unsqueeze(-1)
    z = x.reshape(-1, D) @ w.t()
    z = z.view(B, T - s, -1)
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True, dtype=torch.float64)
    lse = (top + torch.log(total)).squeeze(-1)
    terms = torch.where(seen, lse - z.gather(-1, at).squeeze(-1) + case["z_loss"] * lse * lse, 0.0)
    each = torch.ones_like(terms)
    if case["reduction"] == "mean":
        each = each / seen.sum().clamp_min(1)
    loss = (terms if case["reduction"] == "none" else (terms * each).sum()).float()
    if not case["train"]:
        return loss
    factor = torch.where(seen, state["up"] * each, 0.0)
    d = e * (factor * (1.0 + 2.0 * case["z_loss"] * lse) / total.squeeze(-1)).float().unsqueeze(-1)
    d.scatter_add_(-1, at, -factor.float().unsqueeze(-1))
    d = d.reshape(-1, d.shape[-1])
    dh = torch.zeros(B, T, D, device=x.device)
    dh[:, :T - s] = (d @ w).view(B, T - s, D)
    dw = d.t() @ x.reshape(-1, D)
    return loss, dh.to(state["hidden"].dtype), dw.to(state["weight"].dtype)


def _plain_table(case, state):
    w, ids = state["weight"], state["ids"]
    out = (w[ids].float() * case["scale"]).to(w.dtype)
    if not case["train"]:
        return out
    up = state["up"].float()
    if state["padding"] is not None:
        up = torch.where((ids == state["padding"]).unsqueeze(1), 0.0, up)
    # sums of thousands of terms: in 64 bits
    d = torch.zeros(w.shape, device=w.device, dtype=torch.float64).index_add_(0, ids, up.double())
    return out, (d * case["scale"]).float().to(w.dtype)


def _act(name, g):
    """An activation and its slope."""
    if name == "relu":
        return g.clamp_min(0), (g > 0).to(g.dtype)
    if name == "silu":
        p = 1 / (1 + torch.exp(-g))
        return g * p, p * (1 + g * (1 - p))
    if name == "gelu":
        p = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
        return g * p, p + g * torch.exp(-0.5 * g * g) * (0.5 / math.pi) ** 0.5
    k, c = (2 / math.pi) ** 0.5, 0.044715
    t = torch.tanh(k * (g + c * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * c * g * g)


def _hold(case, dtype, v):
    """What the backward pass finds of a pre-activation [rows, ffn]: rounded to the inputs' type, or e4m3 codes whose neighbours in a
    row share an exponent, the smallest power of two that brings the largest of them to 448 or below."""
    if case["kept"] == "16bit":
        return v.to(dtype).to(v.dtype)
    n, F = v.shape
    b = torch.nn.functional.pad(v, (0, -F % BLOCK)).view(n, -1, BLOCK)
    mantissa, exponent = torch.frexp(b.abs().amax(-1, keepdim=True) / 448)
    exponent = torch.where(mantissa == 0.5, exponent - 1, exponent).clamp_(-126, 126)
    codes = torch.ldexp(b, -exponent).float().to(torch.float8_e4m3fn).to(v.dtype)
    return torch.ldexp(codes, exponent).view(n, -1)[:, :F]


def _plain_gated(case, state):
    x, w, up = state["x"].float(), state["weight"].float(), state["up"].float()
    F = w.shape[0] // 2
    g, u = (x @ w.t()).split(F, dim=1)
    dtype = state["x"].dtype
    y = (_act(case["act"], g)[0] * u).to(dtype)
    if not case["train"]:
        return y
    g, u = _hold(case, dtype, g), _hold(case, dtype, u)
    value, slope = _act(case["act"], g)
    d = torch.cat((up * u * slope, up * value), 1)
    return y, (d @ w).to(dtype), (d.t() @ x).to(dtype)


_plain = {"head": _plain_head, "table": _plain_table, "gated": _plain_gated}


# -- the definitions in 64 bits ---------------------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    return {"head": _exact_head, "table": _exact_table, "gated": _exact_gated}[case["op"]](case, state)


def _exact_head(case, state):
    s = 1 if case["shift"] else 0
    B, T, D = state["hidden"].shape
    w = state["weight"].double()
    place = [(b, t) for b, row in enumerate(state["labels"].tolist()) for t in range(T - s) if row[t + s] != IGNORE]
    bs, ts = [torch.tensor(c, dtype=torch.long, device="cuda") for c in ([b for b, _ in place], [t for _, t in place])]
    terms = torch.zeros(B, T - s, dtype=torch.float64, device="cuda")
    dh = torch.zeros(B, T, D, dtype=torch.float64, device="cuda")
    dw = torch.zeros_like(w)
    up = state["up"].double().expand(B, T - s) / (max(1, len(place)) if case["reduction"] == "mean" else 1)
    for k in range(0, len(place), 1024):
        b, t = bs[k:k + 1024], ts[k:k + 1024]
        x = state["hidden"][b, t].double()
        z = x @ w.t()
        label = state["labels"][b, t + s]
        lse = torch.logsumexp(z, 1)
        terms[b, t] = lse - z.gather(1, label.unsqueeze(1)).squeeze(1) + case["z_loss"] * lse ** 2
        if case["train"]:
            d = torch.softmax(z, 1) * (1 + 2 * case["z_loss"] * lse).unsqueeze(1)
            d[torch.arange(len(b), device="cuda"), label] -= 1
            d *= up[b, t].unsqueeze(1)
            dh[b, t] = d @ w
            dw += d.t() @ x
    loss = terms if case["reduction"] == "none" else terms.sum() / (max(1, len(place)) if case["reduction"] == "mean" else 1)
    return (loss, dh, dw) if case["train"] else loss


def _exact_table(case, state):
    w, ids = state["weight"].double(), state["ids"]
    out = w[ids] * case["scale"]
    if not case["train"]:
        return out
    order = torch.argsort(ids, stable=True)
    if state["padding"] is not None:
        order = order[ids[order] != state["padding"]]
    found, count = torch.unique_consecutive(ids[order], return_counts=True)
    ends = torch.cumsum(count, 0)
    dw = torch.zeros_like(w)
    for c in range(0, w.shape[1], 512):      # (differences of running sums, some columns at a time)
        run = torch.cumsum(state["up"][order, c:c + 512].double(), 0)
        at = run[ends - 1] if len(ends) else run
        at[1:] -= run[ends[:-1] - 1] if len(ends) else 0
        dw[found, c:c + 512] = at * case["scale"]
    return out, dw


def _exact_gated(case, state):
    x, w, up = state["x"].double(), state["weight"].double(), state["up"].double()
    F = w.shape[0] // 2
    act = {"silu": torch.nn.functional.silu, "relu": torch.relu, "gelu": torch.nn.functional.gelu,
           "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[case["act"]]
    g, u = x @ w[:F].t(), x @ w[F:].t()
    y = act(g) * u
    if not case["train"]:
        return y
    g, u = (_hold(case, state["x"].dtype, v).requires_grad_() for v in (g, u))
    with torch.enable_grad():
        dg, du = torch.autograd.grad(act(g) * u, (g, u), up)
    return y, dg @ w[:F] + du @ w[F:], torch.cat((dg.t() @ x, du.t() @ x))
