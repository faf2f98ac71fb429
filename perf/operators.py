"""Operators of a language model's fine-tuning step behind its stages: the log-probabilities of given tokens, a preference
loss and a clipped policy loss over them (each from the logits, with the gradient that the last stage's backward starts
from), and an AdamW step whose moments are held in 8 bits.

A case is one call of one operator.  `run` makes it through `pfeife_amd` where `own` is true, and in elementary torch
operations where it is false.
"""
import math

import torch
import torch.nn.functional as F

own = False

IGNORE = -100
BLOCK = 256           # elements of an 8-bit moment that share a scale
SMALL = 4096          # parameters of fewer elements keep 32-bit moments
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _logits(name, op, dtype, batch, seq, vocab, **more):
    case = dict(name=name, op=op, dtype=dtype, batch=batch, seq=seq, vocab=vocab, shift=False, prompt=0, ragged=0, empty=False,
                padded_vocab=0, temperature=1.0, train=True, sequences=False, reference=False)
    case.update(more)
    return case


def _adam(name, sizes, step=1000):
    return dict(name=name, op="adamw8", sizes=sizes, step=step)


def listed():
    return [
        # one sampled token of each of sixteen requests, scored by the model that sampled it: nothing but latency
        _logits("logprobs_one_token_bf16", "logprobs", "bf16", 16, 1, 32000, train=False, temperature=0.8),
        # a frozen reference model's log-probabilities of eight answers of odd length, forward alone
        _logits("logprobs_reference_bf16", "logprobs", "bf16", 8, 1021, 32000, train=False, shift=True, prompt=200, ragged=300),
        # the log-probabilities with their gradient, in full precision: what a loss of the user's own is written on
        _logits("logprobs_train_fp32", "logprobs", "fp32", 6, 255, 10007, shift=True, prompt=31, ragged=100, empty=True),
        # the looped decoder of the benchmark's small configuration on two preference pairs
        _logits("preference_small_bf16", "preference", "bf16", 4, 128, 512, shift=True, prompt=40, ragged=30),
        # pairs of odd length under an odd vocabulary in half precision, each row starting where no vector does
        _logits("preference_ragged_fp16", "preference", "fp16", 6, 777, 49999, shift=True, prompt=100, ragged=400),
        # two pairs at the 1B decoder's own sequence length and vocabulary
        _logits("preference_decoder_bf16", "preference", "bf16", 4, 2048, 32000, shift=True, prompt=512, ragged=700),
        # a policy step on eight rollouts, advantage per sequence, KL to a reference model
        _logits("policy_rollouts_bf16", "policy", "bf16", 8, 1021, 32000, shift=True, prompt=200, ragged=300, reference=True),
        # every sequence weighs the same, a temperature, a sequence that has no token left, in full precision
        _logits("policy_sequences_fp32", "policy", "fp32", 6, 255, 10007, prompt=31, ragged=100, empty=True, sequences=True,
                temperature=0.7, reference=True),
        # a large vocabulary with a padded tail that the model masks
        _logits("policy_vocabulary_bf16", "policy", "bf16", 2, 1024, 131072, shift=True, prompt=100, ragged=200, padded_vocab=800),
        # one encoder block of ViT-S/16: four matrices in 8 bits, eight vectors in 32
        _adam("adamw8_block", "442368,147456,589824,589824,1152,384,1536,384,384,384,384,384"),
        # odd sizes: blocks that end early, a matrix that starts a step count
        _adam("adamw8_odd", "2551785,4097,23907,1,255,1048577,333", step=0),
        # a layer of the 1B decoder with its embedding
        _adam("adamw8_decoder", "65536000,4194304,4194304,4194304,4194304,11534336,11534336,11534336,2048,2048"),
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("logprobs", "preference", "policy", "adamw8"))
    if op == "adamw8":
        sizes, left = [], _spread(rng, 20_000, 100_000_000)
        for _ in range(rng.randint(1, 8)):
            sizes.append(max(1, min(left, _spread(rng, 100, left))))
            left = max(1, left - sizes[-1])
        case = _adam("", ",".join(str(n) for n in sizes), step=rng.choice((0, 3, 200, 20000)))
    else:
        vocab = _spread(rng, 500, 131072) - rng.choice((0, 0, 1, 3))
        rows = _spread(rng, 1, max(1, min(16384, 200_000_000 // vocab)))
        batch = min(rows, 2 * rng.randint(1, 8))
        batch += batch % 2
        seq = max(2, rows // batch)
        case = _logits("", op, rng.choice(("bf16", "bf16", "fp16", "fp32")), batch, seq, vocab, shift=rng.random() < 0.6,
                       prompt=rng.randint(0, seq // 2), ragged=rng.randint(0, seq // 3), empty=batch > 2 and rng.random() < 0.3,
                       padded_vocab=rng.choice((0, 0, 64)), temperature=rng.choice((1.0, 1.0, 0.7)) if op != "preference" else 1.0,
                       train=op != "logprobs" or rng.random() < 0.5, sequences=op == "policy" and rng.random() < 0.5,
                       reference=op == "policy" and rng.random() < 0.5)
    del case["name"]
    return case


def _counted(case):
    """[first, last) label positions of every sequence that are scored: answers of different length behind a prompt."""
    spans = []
    for b in range(case["batch"]):
        last = case["seq"] - (b * case["ragged"]) // max(1, case["batch"] - 1)
        first = max(case["prompt"], 1 if case["shift"] else 0)
        spans.append((first, max(first, last)) if not (case["empty"] and b == 1) else (first, first))
    return spans


def work(case):
    if case["op"] == "adamw8":
        sizes = [int(n) for n in case["sizes"].split(",")]
        # parameter read and written, gradient read; moments of a byte with a scale of four to 256, or of four bytes, read and written
        return {"bytes": float(sum(n * 28 if n < SMALL else n * 16 + 16 * -(-n // BLOCK) for n in sizes)),
                "flops": 20.0 * sum(sizes)}
    size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    rows = sum(last - first for first, last in _counted(case))
    every = case["batch"] * case["seq"]
    read, written = rows * case["vocab"] * size, every * case["vocab"] * size if case["train"] else 0
    tokens = every * (8 + 4 + (4 if case["op"] == "policy" else 0) + (4 if case["reference"] else 0))
    return {"bytes": float(read + written + tokens), "flops": (8.0 if case["train"] else 4.0) * rows * case["vocab"]}


# -- inputs -----------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000 + seed)
    rnd = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    if case["op"] == "adamw8":
        return _prepare_adam(case, gen, rnd)
    B, T, V = case["batch"], case["seq"], case["vocab"]
    logits = torch.empty(B, T, V, device="cuda", dtype=DTYPES[case["dtype"]])
    for b in range(B):
        logits[b] = rnd(T, V) * 1.5
    usable = V - case["padded_vocab"]
    labels = torch.randint(0, usable, (B, T), device="cuda", generator=gen)
    s = 1 if case["shift"] else 0
    at = labels[:, s:].unsqueeze(-1)       # the model is fairly sure of the answer
    logits[:, :T - s].scatter_(2, at, (logits[:, :T - s].gather(2, at).float() + 6.0 + 2.0 * rnd(B, T - s, 1)).to(logits.dtype))
    if case["padded_vocab"]:
        logits[:, :, usable:] = -math.inf
    for b, (first, last) in enumerate(_counted(case)):
        labels[b, :first] = IGNORE
        labels[b, last:] = IGNORE
    state = dict(case=case, logits=logits, labels=labels)
    if case["op"] != "logprobs":
        now = torch.zeros(B, T - s, device="cuda")
        for b in range(B):
            lp = torch.log_softmax(logits[b, :T - s].float() / case["temperature"], -1)
            now[b] = lp.gather(1, labels[b, s:].clamp_min(0).unsqueeze(-1)).squeeze(-1)
        seen = labels[:, s:] != IGNORE
    if case["op"] == "preference":     # the reference model's log-probability of every answer
        state["ref"] = torch.where(seen, now, 0.0).double().sum(1).float() + 3.0 * rnd(B)
    if case["op"] == "policy":         # places that take no part hold what the sampler left there
        state["old"] = torch.where(seen, now + 0.15 * rnd(B, T - s), math.nan)
        state["advantages"] = rnd(B)
        state["ref"] = torch.where(seen, now + 0.2 * rnd(B, T - s), math.nan) if case["reference"] else None
    return state


def _prepare_adam(case, gen, rnd):
    state = dict(case=case, params=[], grads=[], moments=[])
    for k, n in enumerate(int(s) for s in case["sizes"].split(",")):
        state["params"].append(0.02 * rnd(n))
        state["grads"].append(10.0 ** (-2 - k % 3) * rnd(n))
        if n < SMALL:
            m = {"exp_avg": 1e-4 * rnd(n), "exp_avg_sq": 1e-6 * rnd(n).square()}
        else:
            blocks = -(-n // BLOCK)
            size = 10.0 ** (-6 - k % 3)
            m = {"exp_avg": (100.0 * rnd(n)).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn),
                 "exp_avg_scale": size * (0.5 + torch.rand(blocks, device="cuda", generator=gen)),
                 "root": (100.0 * rnd(n).abs() + 0.01).clamp_(0.0, 448.0).to(torch.float8_e4m3fn),
                 "root_scale": 3.0 * size * (0.5 + torch.rand(blocks, device="cuda", generator=gen))}
        if not case["step"]:
            m = {key: torch.zeros_like(t) for key, t in m.items()}
        state["moments"].append(m)
    state["step"] = case["step"]
    return state


ADAM = dict(lr=1e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
PREFERENCE = dict(beta=0.1, label_smoothing=0.05)
POLICY = dict(clip=0.2, clip_high=0.28)
KL = 0.04


# -- one pass ---------------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    return (_own if own else _plain)[case["op"]](case, state)


def _own_logprobs(case, state):
    from pfeife_amd.loss import token_logprobs

    x = state["logits"].detach().requires_grad_(case["train"])
    lp = token_logprobs(x, state["labels"], temperature=case["temperature"], shift=case["shift"])
    if not case["train"]:
        return lp
    return lp.detach(), torch.autograd.grad(lp, x, lp.detach())[0]     # (any upstream gradient; this one needs no pass)


def _own_preference(case, state):
    from pfeife_amd.loss import preference_loss

    x = state["logits"].detach().requires_grad_()
    loss, rewards = preference_loss(x, state["labels"], state["ref"], shift=case["shift"], **PREFERENCE)
    return loss.detach(), rewards, torch.autograd.grad(loss, x)[0]


def _own_policy(case, state):
    from pfeife_amd.loss import policy_loss

    x = state["logits"].detach().requires_grad_()
    loss, logprobs, kl = policy_loss(x, state["labels"], state["old"], state["advantages"], state["ref"],
                                     kl_coef=KL if case["reference"] else 0.0, temperature=case["temperature"],
                                     reduction="sequences" if case["sequences"] else "tokens", shift=case["shift"], **POLICY)
    return loss.detach(), logprobs, kl, torch.autograd.grad(loss, x)[0]


def _own_adam(case, state):
    from pfeife_amd.optim import AdamW8bit

    opt = state.get("optimizer")
    if opt is None:        # a program makes its optimizer once
        params = [torch.nn.Parameter(p) for p in state["params"]]
        opt = state["optimizer"] = AdamW8bit(params, min_8bit_size=SMALL, **ADAM)
        for p, g, m in zip(params, state["grads"], state["moments"]):
            p.grad = g
            opt.state[p] = {"step": torch.tensor(float(state["step"])),
                            **{{"root": "exp_avg_sq_root", "root_scale": "exp_avg_sq_root_scale"}.get(k, k): t for k, t in m.items()}}
    opt.step()
    return _adam_outputs(state)


_own = {"logprobs": _own_logprobs, "preference": _own_preference, "policy": _own_policy, "adamw8": _own_adam}


def _adam_outputs(state):
    return {"params": state["params"], "moments": state["moments"]}


def _scored(case, state):
    """(logits whose place has a label, labels, which of them count)"""
    x, labels = state["logits"], state["labels"]
    if case["shift"]:
        x, labels = x[:, :-1], labels[:, 1:]
    return x, labels, labels != IGNORE


def _softmax(case, x, labels, seen):
    """Probabilities in 32 bits and the labels' log-probabilities; the sum over the vocabulary and what is taken from it in 64,
    because an answer's log-probability is compared with others that lie close."""
    x = x.float()
    top = x.amax(-1, keepdim=True)
    e = torch.exp((x - top) / case["temperature"])
    total = e.sum(-1, keepdim=True, dtype=torch.float64)
    at = torch.where(seen, labels, 0).unsqueeze(-1)
    lp = ((x.gather(-1, at) - top).double() / case["temperature"] - torch.log(total)).squeeze(-1)
    return e / total.float(), torch.where(seen, lp, 0.0), at


def _gradient(case, state, p, at, g):
    """dlogits of g[b, t] = d loss / d logprob[b, t]: g (onehot - p) / temperature, in the logits' type."""
    g = (g / case["temperature"]).float().unsqueeze(-1)
    d = p * -g
    d.scatter_add_(-1, at, g)
    d = torch.where(g == 0, 0.0, d).to(state["logits"].dtype)
    return F.pad(d, (0, 0, 0, 1)) if case["shift"] else d


def _plain_logprobs(case, state):
    x, labels, seen = _scored(case, state)
    p, lp, at = _softmax(case, x, labels, seen)
    if not case["train"]:
        return lp.float()
    return lp.float(), _gradient(case, state, p, at, lp.float().double())


def _plain_preference(case, state):
    x, labels, seen = _scored(case, state)
    p, lp, at = _softmax(case, x, labels, seen)
    beta, eps = PREFERENCE["beta"], PREFERENCE["label_smoothing"]
    rewards = beta * (lp.sum(1) - state["ref"].double())
    delta = rewards[0::2] - rewards[1::2]
    loss = ((1 - eps) * torch.log1p(torch.exp(-delta)) + eps * torch.log1p(torch.exp(delta))).mean()
    d = (beta / delta.numel()) * (1 / (1 + torch.exp(-delta)) - (1 - eps))
    g = torch.stack((d, -d), 1).reshape(-1, 1) * seen
    return loss.float(), rewards.float(), _gradient(case, state, p, at, g)


def _plain_policy(case, state):
    x, labels, seen = _scored(case, state)
    p, lp, at = _softmax(case, x, labels, seen)
    counts = seen.sum(1, keepdim=True)
    if case["sequences"]:
        weight = seen / (counts.clamp_min(1) * (counts > 0).sum().clamp_min(1)).double()
    else:
        weight = seen / counts.sum().clamp_min(1).double()
    adv = state["advantages"].double().unsqueeze(1)
    ratio = torch.where(seen, torch.exp(lp - state["old"].double()), 0.0)
    low, high = 1 - POLICY["clip"], 1 + POLICY["clip_high"]
    gain = torch.minimum(ratio * adv, ratio.clamp(low, high) * adv)
    free = torch.where(adv >= 0, ratio <= high, ratio >= low)
    g = torch.where(free, -adv * ratio, 0.0)
    term = -gain
    kl = torch.zeros_like(lp)
    if case["reference"]:
        back = torch.where(seen, state["ref"].double() - lp, 0.0)
        kl = torch.exp(back) - back - 1
        g = g + KL * (1 - torch.exp(back))
        term = term + KL * kl
    loss, mean_kl = (weight * term).sum(), (weight * kl).sum()
    return loss.float(), lp.float(), mean_kl.float(), _gradient(case, state, p, at, torch.where(seen, weight * g, 0.0))


# the 8-bit moments: a block of 256 shares a scale, its largest magnitude over 448; codes are e4m3.  The second moment is held as its
# square root.  Codes are rounded up with the probability that keeps the mean, by bits that block, element, tensor and step give.

def _mix(x):
    x = (x ^ (x >> 16)) * 0x93D765DD & 0xFFFFFFFF
    x = (x ^ (x >> 15)) * 0x9E3779B1 & 0xFFFFFFFF
    return x ^ (x >> 16)


def _dither(block, tensor, step):
    """32 bits for each element of each block"""
    key = _mix(_mix(block + tensor * 0x9E3779B1 & 0xFFFFFFFF) + step * 0x93D765DD & 0xFFFFFFFF)
    return _mix(key.unsqueeze(1) + torch.arange(BLOCK, device=block.device) * 0x9E3779B1 & 0xFFFFFFFF)


def _encode(x, bits, root):
    top = x.abs().amax(1, keepdim=True)
    kept = top >= 2.0 ** -100
    most = torch.full_like(top, 448.0)
    inv = torch.where(kept, most / top, 0.0)
    a = x.abs() * inv
    fine = a < 2.0 ** -6                     # below it the codes are 2^-9 apart
    t = torch.where(fine, a + 2.0 ** -6, a).view(torch.int32) + (bits << 4).to(torch.int32) & ~0xFFFFF
    q = t.view(torch.float32)
    q = torch.where(fine, q - 2.0 ** -6, q).clamp(max=448.0)
    if root:                                 # a root that is there stays there: updates are divided by it
        q = torch.where((x > 0) & kept, q.clamp(min=2.0 ** -9), q)
    return torch.copysign(q, x).to(torch.float8_e4m3fn), torch.where(kept, top / most, 0.0).squeeze(1)


def _plain_adam(case, state):
    state["step"] += 1
    t, (b1, b2) = state["step"], ADAM["betas"]
    rate, bias = ADAM["lr"] / (1 - b1 ** t), math.sqrt(1 - b2 ** t)

    def update(p, g, m, v):
        m = m + (1 - b1) * (g - m)
        v = b2 * v + (1 - b2) * (g * g)
        root = torch.sqrt(v)
        bias32 = torch.full((), bias, device=p.device)
        return p * (1 - ADAM["lr"] * ADAM["weight_decay"]) - rate * (m / (root / bias32 + ADAM["eps"])), m, v, root

    params, grads, moments = state["params"], state["grads"], state["moments"]
    small = [k for k, p in enumerate(params) if p.numel() < SMALL]
    large = [k for k, p in enumerate(params) if p.numel() >= SMALL]
    if small:
        sizes = [params[k].numel() for k in small]
        olds = [torch.cat(ts) for ts in ([params[k] for k in small], [grads[k] for k in small],
                                         [moments[k]["exp_avg"] for k in small], [moments[k]["exp_avg_sq"] for k in small])]
        news = [x.split(sizes) for x in update(*olds)[:3]]
        torch._foreach_copy_([params[k] for k in small] + [moments[k]["exp_avg"] for k in small] + [moments[k]["exp_avg_sq"] for k in small],
                             [t for x in news for t in x])
    if large:
        pad = lambda ts: torch.cat([F.pad(t, (0, -t.numel() % BLOCK)) for t in ts]).view(-1, BLOCK)  # noqa: E731
        codes = lambda key: pad([moments[k][key].view(torch.uint8) for k in large]).view(torch.float8_e4m3fn).float()  # noqa: E731
        scales = lambda key: torch.cat([moments[k][key] for k in large]).unsqueeze(1)  # noqa: E731
        m, r = codes("exp_avg") * scales("exp_avg_scale"), codes("root") * scales("root_scale")
        p, m, _, r = update(pad([params[k] for k in large]), pad([grads[k] for k in large]), m, r * r)
        blocks = [-(-params[k].numel() // BLOCK) for k in large]
        dither = torch.cat([_dither(torch.arange(n, device="cuda"), k, t) for k, n in zip(large, blocks)])
        new = [(p, "params")]
        for x, key, bits, root in ((m, "exp_avg", dither >> 16, False), (r, "root", dither & 0xFFFF, True)):
            q, s = _encode(x, bits, root)
            torch._foreach_copy_([moments[k][key + "_scale"] for k in large], list(s.split(blocks)))
            new.append((q.view(torch.uint8), key))
        for x, key in new:
            parts = [part.reshape(-1)[:params[k].numel()] for k, part in zip(large, x.split(blocks))]
            torch._foreach_copy_([params[k] if key == "params" else moments[k][key].view(torch.uint8) for k in large], parts)
    return _adam_outputs(state)


_plain = {"logprobs": _plain_logprobs, "preference": _plain_preference, "policy": _plain_policy, "adamw8": _plain_adam}


# -- the definitions in 64 bits ---------------------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "adamw8":
        return _exact_adam(state)
    s = 1 if case["shift"] else 0
    B, T = state["labels"].shape
    spans = [[t for t in range(T - s) if row[t + s] != IGNORE] for row in state["labels"].tolist()]
    filled = sum(1 for span in spans if span)
    tokens = sum(len(span) for span in spans)
    lps, grads = [], []

    def sequence(b, of=None):
        """The log-probabilities of sequence b's tokens, and the gradient of `of` of them."""
        z = state["logits"][b, spans[b]].double().requires_grad_(of is not None)
        with torch.set_grad_enabled(of is not None):
            y = z / case["temperature"]
            lp = y.gather(1, state["labels"][b, [t + s for t in spans[b]]].unsqueeze(1)).squeeze(1) - torch.logsumexp(y, 1)
            value = of(lp) if of is not None and spans[b] else None
        full = torch.zeros(T - s, dtype=torch.float64, device="cuda")
        full[spans[b]] = lp.detach()
        if of is not None:
            d = torch.zeros(T, case["vocab"], dtype=torch.float64 if case["dtype"] == "fp32" else torch.float32, device="cuda")
            if value is not None:
                d[spans[b]] = torch.autograd.grad(value[0] if isinstance(value, tuple) else value, z)[0].to(d.dtype)
            grads.append(d)
        lps.append(full)
        return value

    if case["op"] == "logprobs":
        for b in range(B):
            sequence(b, (lambda lp: 0.5 * lp.square().sum()) if case["train"] else None)
        return (torch.stack(lps), torch.stack(grads)) if case["train"] else torch.stack(lps)
    if case["op"] == "preference":
        beta, eps = PREFERENCE["beta"], PREFERENCE["label_smoothing"]
        for b in range(B):
            sequence(b)
        rewards = (beta * (torch.stack(lps).sum(1) - state["ref"].double())).requires_grad_()
        with torch.enable_grad():
            margin = rewards[0::2] - rewards[1::2]
            loss = -((1 - eps) * F.logsigmoid(margin) + eps * F.logsigmoid(-margin)).mean()
        up = torch.autograd.grad(loss, rewards)[0]
        for b in range(B):
            sequence(b, lambda lp: beta * up[b] * lp.sum())
        return loss.detach(), rewards.detach(), torch.stack(grads)
    loss = kls = 0.0
    low, high = 1 - POLICY["clip"], 1 + POLICY["clip_high"]
    for b in range(B):
        weight = 1.0 / (len(spans[b]) * filled if case["sequences"] else tokens) if spans[b] else 0.0

        def objective(lp):
            ratio = torch.exp(lp - state["old"][b, spans[b]].double())
            a = state["advantages"][b].double()
            total, kl = -torch.minimum(ratio * a, torch.clamp(ratio, low, high) * a), torch.zeros_like(ratio)
            if case["reference"]:
                diff = state["ref"][b, spans[b]].double() - lp
                kl = torch.expm1(diff) - diff
                total = total + KL * kl
            return weight * total.sum(), weight * kl.sum()

        value = sequence(b, objective)
        if value is not None:
            loss, kls = loss + value[0].detach(), kls + value[1].detach()
    return loss, torch.stack(lps), kls, torch.stack(grads)


def _exact_adam(state):
    params, moments = [], []
    t, (b1, b2) = state["step"] + 1, ADAM["betas"]
    for p, g, old in zip(state["params"], state["grads"], state["moments"]):
        p, g = p.double(), g.double()
        if "root" in old:
            spread = lambda s: s.double().repeat_interleave(BLOCK)[:p.numel()]  # noqa: E731
            m = old["exp_avg"].float().double() * spread(old["exp_avg_scale"])
            v = (old["root"].float().double() * spread(old["root_scale"])).square()
        else:
            m, v = old["exp_avg"].double(), old["exp_avg_sq"].double()
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        step = (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + ADAM["eps"])
        params.append(p - ADAM["lr"] * ADAM["weight_decay"] * p - ADAM["lr"] * step)
        if "root" in old:
            top = lambda x: F.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK).abs().amax(1) / 448.0  # noqa: E731
            # (which code a value is rounded to is the dither's choice, and has no 64-bit value)
            moments.append({"exp_avg": None, "exp_avg_scale": top(m), "root": None, "root_scale": top(v.sqrt())})
        else:
            moments.append({"exp_avg": m, "exp_avg_sq": v})
    return {"params": params, "moments": moments}
