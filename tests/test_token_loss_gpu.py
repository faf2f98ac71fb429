"""Log-probabilities of given tokens, the preference loss and the policy loss against the same in 64 bits."""
import itertools
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}    # (half a step where steps end, or what flushes to zero)
IGNORE = -100


def make(dtype, B, T, V, shift, seed=0, masked=0.3, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, T, V, generator=g) * spread).to(dtype).cuda()
    y = torch.randint(0, V, (B, T), generator=g).cuda()
    y[(torch.rand(B, T, generator=g) < masked).cuda()] = IGNORE
    if B > 2:
        y[1] = IGNORE        # a sequence with nothing to score
    return x, y


def logprobs64(x, y, shift, temperature=1.0):
    """-> (differentiable logits of the scored rows in 64 bits, their log-probabilities, which count, bound of the fp32 sums' relative error)"""
    s = int(shift)
    z = x[:, :x.shape[1] - s].detach().double().requires_grad_()
    seen = y[:, s:] != IGNORE
    lp = torch.log_softmax(z / temperature, -1).gather(-1, y[:, s:].clamp(0, x.shape[-1] - 1).unsqueeze(-1)).squeeze(-1)
    with torch.no_grad():
        p = torch.softmax(z / temperature, -1)
        far = (z.amax(-1, keepdim=True) - z) / temperature
        # a term is off by the rounding of its exponent (twice: the factor's and the product's) and of the exponential; 64 lanes at least
        # share a row, and their sums and the results of 16 wavefronts are added up in turn
        rel = (x.shape[-1] / 64 + 32 + 3 * torch.where(p > 0, p * far, 0).sum(-1)) * 2.0 ** -24
    return z, torch.where(seen, lp, 0.0), seen, rel


def check_gradient(d, want, g, p, far, rel, dtype, dg):
    """d against g (onehot - p): off by p's error, by dg, the error of g, and a rounding to the result's type."""
    g = g.abs().unsqueeze(-1)
    tol = g * (p * (rel.unsqueeze(-1) + (3 * far + 8) * 2.0 ** -24) + (want != 0) * 4 * 2.0 ** -24) + (1 + p) * dg.unsqueeze(-1)
    tol = tol * (1 + U[dtype]) + U[dtype] * want.abs() + LEAST[dtype]
    off = (d.double() - want).abs() - tol
    assert (off <= 0).all(), float(off.max())


def parts(z, temperature):
    with torch.no_grad():
        return torch.softmax(z / temperature, -1), (z.amax(-1, keepdim=True) - z) / temperature


SHAPES = [(torch.float32, 1, 1, 1, 0), (torch.bfloat16, 2, 3, 2, 1), (torch.float16, 3, 5, 7, 0), (torch.float32, 2, 9, 63, 1), (torch.bfloat16, 4, 33, 512, 1),
          (torch.float16, 3, 17, 1003, 0), (torch.bfloat16, 1, 7, 8195, 0), (torch.float32, 3, 4, 16387, 1), (torch.float16, 2, 5, 50021, 1),
          (torch.bfloat16, 2, 3, 131075, 0), (torch.float32, 2, 2, 70001, 0), (torch.bfloat16, 2, 2, 300007, 1), (torch.bfloat16, 1, 1, 32000, 0),
          (torch.bfloat16, 2, 300, 4096, 1)]


@pytest.mark.parametrize("temperature", [1.0, 0.7])
@pytest.mark.parametrize("dtype,B,T,V,shift", SHAPES)
def test_token_logprobs(dtype, B, T, V, shift, temperature):
    from pfeife_amd.loss import token_logprobs

    x, y = make(dtype, B, T, V, shift, masked=0.3 if B * T > 1 else 0.0)
    z, want, seen, rel = logprobs64(x, y, shift, temperature)
    leaf = x.clone().requires_grad_()
    lp = token_logprobs(leaf, y, temperature=temperature, shift=bool(shift))
    assert lp.dtype == torch.float32 and lp.shape == want.shape
    tol = rel + 2.0 ** -24 * (want.abs() + 4)
    assert ((lp.double() - want).abs() <= tol).all()
    assert (lp[~seen] == 0).all()
    g = torch.linspace(-2, 2, want.numel(), device="cuda").view(want.shape)
    (d,) = torch.autograd.grad(lp, leaf, g)
    (dz,) = torch.autograd.grad(want, z, g.double())
    assert d.dtype == dtype and d.shape == x.shape
    check_gradient(d[:, :T - shift], dz, torch.where(seen, g.double(), 0) / temperature, *parts(z, temperature), rel, dtype, torch.zeros_like(rel))
    assert (d[:, T - shift:] == 0).all() and (d[:, :T - shift][~seen] == 0).all()
    with torch.no_grad():      # the same without a gradient
        assert torch.equal(token_logprobs(leaf, y, temperature=temperature, shift=bool(shift)), lp)


@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("dtype,B,T,V,shift", [s for s in SHAPES if s[1] % 2 == 0])
def test_preference_loss(dtype, B, T, V, shift, average):
    from pfeife_amd.loss import preference_loss

    x, y = make(dtype, B, T, V, shift, seed=1)
    z, lp, seen, rel = logprobs64(x, y, shift)
    n = seen.sum(1).clamp_min(1).double() if average else torch.ones(B, device="cuda", dtype=torch.float64)
    s = lp.sum(1) / n
    ref = (s.detach() + torch.linspace(-4, 5, B, device="cuda")).float()
    beta, eps = 0.3, 0.1
    rewards = beta * (s - ref.double())
    D = rewards[0::2] - rewards[1::2]
    want = -((1 - eps) * F.logsigmoid(D) + eps * F.logsigmoid(-D)).mean()
    leaf = x.clone().requires_grad_()
    loss, got = preference_loss(leaf, y, ref, beta=beta, label_smoothing=eps, length_average=average, shift=bool(shift))
    assert not got.requires_grad and loss.shape == ()
    # a token's log-probability is off by its sum's error and a rounding to 32 bits, a sequence's by all its tokens'
    off = beta * ((rel + 2.0 ** -24 * (lp.detach().abs() + 4)) * seen).sum(1) / n
    assert ((got.double() - rewards).abs() <= off + 2.0 ** -24 * rewards.abs()).all()
    offD = off.view(-1, 2).sum(1)
    assert abs(float(loss.detach()) - float(want.detach())) <= float(offD.mean()) + 2.0 ** -23 * float(want.detach())       # |d loss / dD| <= 1
    (dz,) = torch.autograd.grad(want, z)
    (d,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    g = torch.sigmoid(D.detach()) - (1 - eps)
    g = torch.stack((g, -g), 1).view(-1, 1) * beta / (B // 2) / n.unsqueeze(1) * seen
    dg = (offD / 4).repeat_interleave(2).unsqueeze(1) * beta / (B // 2) / n.unsqueeze(1) + 2.0 ** -22 * g.abs()     # sigma' <= 1/4
    check_gradient(d[:, :T - shift], dz, g, *parts(z, 1.0), rel, dtype, dg * seen)
    assert (d[:, T - shift:] == 0).all() and (d[:, :T - shift][~seen] == 0).all()
    (again,) = torch.autograd.grad(2 * loss, leaf)       # a power of two: the same digits
    fine = d.abs() >= LEAST[dtype] * 2 ** 12
    assert torch.equal(again[fine], (2 * d)[fine])


LOG_RATIOS = (-0.7, -0.15, 0.0, 0.1, 0.15, 0.9)      # none within 0.03 of the borders ln 0.8 and ln 1.28


def policy_operands(lp, seed):
    """Old and reference log-probabilities with ratios away from the clip's borders, advantages of both signs and zero."""
    g = torch.Generator().manual_seed(seed)
    B, R = lp.shape
    old = (lp - torch.tensor(LOG_RATIOS, dtype=torch.float64)[torch.randint(0, len(LOG_RATIOS), (B, R), generator=g)].cuda()).float()
    ref = (lp + 0.3 * torch.randn(B, R, generator=g).cuda()).float()
    adv = torch.randn(B, R, generator=g).cuda()
    adv[:, ::5] = 0.0
    return old, ref, adv


def policy64(lp, seen, old, ref, adv, kl_coef, sequences):
    n = seen.sum(1, keepdim=True).double()
    w = seen / (n.clamp_min(1) * (n > 0).sum().clamp_min(1)) if sequences else seen / n.sum().clamp_min(1)
    ratio = torch.exp(torch.where(seen, lp - old.double(), 0.0))
    a = adv.double() if adv.dim() == 2 else adv.double().unsqueeze(1)
    token = -torch.minimum(ratio * a, ratio.clamp(0.8, 1.28) * a)
    k = torch.zeros_like(lp)
    if ref is not None:
        q = torch.where(seen, ref.double() - lp, 0.0)
        k = torch.exp(q) - q - 1
    return (w * (token + kl_coef * k)).sum(), (w * k).sum(), w, ratio.detach(), a, (torch.exp(q.detach()) if ref is not None else None)


@pytest.mark.parametrize("kl_coef,by_token,sequences", [(0.0, False, False), (0.05, True, False), (0.05, False, True)])
@pytest.mark.parametrize("dtype,B,T,V,shift", SHAPES)
def test_policy_loss(dtype, B, T, V, shift, kl_coef, by_token, sequences):
    from pfeife_amd.loss import policy_loss

    x, y = make(dtype, B, T, V, shift, seed=2, masked=0.3 if B * T > 1 else 0.0)
    temperature = 0.8 if sequences else 1.0
    z, lp, seen, rel = logprobs64(x, y, shift, temperature)
    old, ref, adv = policy_operands(lp.detach(), 3)
    adv = adv if by_token else adv[:, -1].clone()
    ref = ref if kl_coef else None
    want, kl, w, ratio, a, back = policy64(lp, seen, old, ref, adv, kl_coef, sequences)
    for t in (old, ref):
        if t is not None:
            t[~seen] = math.nan
    leaf = x.clone().requires_grad_()
    loss, got, got_kl = policy_loss(leaf, y, old, adv, ref, clip=0.2, clip_high=0.28, kl_coef=kl_coef, temperature=temperature,
                                    reduction="sequences" if sequences else "tokens", shift=bool(shift))
    dlp = rel + 2.0 ** -24                             # (the kernel's own log-probability is in 64 bits, its sum is not)
    assert ((got.double() - lp).abs() <= dlp + 2.0 ** -24 * (lp.abs() + 4)).all()
    slope = ratio * a.abs() + (0 if back is None else kl_coef * (back + 1))
    assert abs(float(loss.detach()) - float(want.detach())) <= float((w * slope * dlp).sum().detach()) * 2 + 2.0 ** -24 * abs(float(want.detach())) + 1e-14
    assert abs(float(got_kl) - float(kl)) <= (0 if back is None else float((w * (back + 1) * dlp).sum()) * 2) + 2.0 ** -24 * abs(float(kl)) + 1e-14
    (dz,) = torch.autograd.grad(want, z) if want.requires_grad else (torch.zeros_like(z),)
    (d,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    first = d.clone()
    free = torch.where(a >= 0, ratio <= 1.28, ratio >= 0.8)
    g = w * (-a * ratio * free + (0 if back is None else kl_coef * (1 - back)))
    dg = 2 * w * (a.abs() * ratio + (0 if back is None else kl_coef * back)) * dlp + 2.0 ** -23 * g.abs()
    check_gradient(d[:, :T - shift], dz, g / temperature, *parts(z, temperature), rel, dtype, dg / temperature)
    assert (d[:, T - shift:] == 0).all() and (d[:, :T - shift][~seen] == 0).all()
    # a second backward pass through the same loss, after the first gradient was changed; and a factor
    d.fill_(3.0)
    (again,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    assert (again.double() - first.double()).abs().max() <= 4 * 2.0 ** -24 * first.abs().max() + 2 * U[dtype] * first.abs().max()
    check_gradient(again[:, :T - shift], dz, g / temperature, *parts(z, temperature), rel, dtype, dg / temperature)
    (scaled,) = torch.autograd.grad(-3.0 * loss, leaf)
    check_gradient(scaled[:, :T - shift], -3.0 * dz, 3.0 * g / temperature, *parts(z, temperature), rel, dtype, 3.0 * dg / temperature + 2.0 ** -23 * g.abs())
    # the factor as an argument: the same, and the KL term's mean is not touched by it
    quarter, _, same_kl = policy_loss(leaf, y, old, adv, ref, clip=0.2, clip_high=0.28, kl_coef=kl_coef, temperature=temperature, scale=0.25,
                                      reduction="sequences" if sequences else "tokens", shift=bool(shift))
    assert torch.equal(quarter, 0.25 * loss) and torch.equal(same_kl, got_kl)
    (less,) = torch.autograd.grad(quarter, leaf)
    plain = first.abs() >= LEAST[dtype] * 2 ** 13      # (fp16: 2^-12, so that a quarter is 2^-14 or more, where subnormals end)
    assert torch.equal(less[plain], (0.25 * first)[plain])
    with torch.no_grad():
        quiet, _, _ = policy_loss(leaf, y, old, adv, ref, clip=0.2, clip_high=0.28, kl_coef=kl_coef, temperature=temperature,
                                  reduction="sequences" if sequences else "tokens", shift=bool(shift))
    assert torch.equal(quiet, loss)


def test_gradients_against_differences():
    """d loss / d logit by central differences of the 64-bit formula's own inputs: fp32 logits, a handful of classes."""
    from pfeife_amd.loss import policy_loss, preference_loss

    x, y = make(torch.float32, 2, 4, 5, 0, seed=4, masked=0.2, spread=1.0)
    _, lp, seen, _ = logprobs64(x, y, 0)
    old, ref, adv = policy_operands(lp.detach(), 5)
    total = lp.detach().sum(1).float()
    h = 2.0 ** -6
    for fn in (lambda t: preference_loss(t, y, total - 1.0, beta=0.5)[0], lambda t: policy_loss(t, y, old, adv, ref, clip=0.2, clip_high=0.28, kl_coef=0.1)[0]):
        leaf = x.clone().requires_grad_()
        (d,) = torch.autograd.grad(fn(leaf), leaf)
        for i in range(x.numel()):
            step = torch.zeros(x.numel(), device="cuda")
            step[i] = h
            step = step.view_as(x)
            with torch.no_grad():
                diff = (float(fn(x + step)) - float(fn(x - step))) / (2 * h)
            # third derivative times h^2 / 6 (some 1e-4, ratios up to e^0.9 and coefficients below 1) and the losses' rounding over 2 h
            assert abs(diff - float(d.view(-1)[i])) <= 2e-3 * h + 8 * 2.0 ** -24 / h, i


def test_masked_infinite_and_foreign_values():
    from pfeife_amd.loss import policy_loss, preference_loss, token_logprobs

    for dtype, V in itertools.product((torch.float32, torch.float16, torch.bfloat16), (9, 3001, 140001)):
        x, y = make(dtype, 2, 6, V, 0, seed=6, masked=0.0)
        y[0, 2] = IGNORE
        x[0, 2] = math.nan                     # a row that takes no part
        x[0, 3, V // 2:] = -math.inf           # classes that the model masks
        y[0, 3] = 1
        x[1, 0, 4:] = torch.finfo(dtype).min   # the type's lowest value
        y[1, 0] = 2
        y[1, 1] = 5
        x[1, 1, 5] = -math.inf                 # a label that has no probability
        z, want, seen, rel = logprobs64(torch.nan_to_num(x, nan=0.0, neginf=-math.inf), y, 0)
        leaf = x.clone().requires_grad_()
        lp = token_logprobs(leaf, y)
        fine = torch.isfinite(want)
        assert lp[1, 1] == -math.inf and not fine[1, 1] and fine.sum() == 11
        assert ((lp.double() - want)[fine].abs() <= (rel + 2.0 ** -24 * (want.abs() + 4))[fine]).all()
        (d,) = torch.autograd.grad(lp.sum(), leaf)         # (an expanded gradient)
        assert torch.isfinite(d).all() and (d[0, 2] == 0).all() and (d[0, 3, max(2, V // 2):] == 0).all()
        # labels outside the vocabulary read nothing and show
        bad = y.clone()
        bad[0, 0], bad[1, 4] = V, -7
        lp = token_logprobs(leaf, bad)
        assert lp[0, 0].isnan() and lp[1, 4].isnan() and lp.isnan().sum() == 2
        (d,) = torch.autograd.grad(lp.sum(), leaf)
        assert d[0, 0].isnan().all() and d[1, 4].isnan().all() and torch.isfinite(d[0, 1]).all()
        # a row of nothing but -inf, and one with +inf: NaN, as a softmax of them is
        odd = x.clone()
        odd[0, 0], odd[1, 5, 3] = -math.inf, math.inf
        lp = token_logprobs(odd, y)
        assert lp[0, 0].isnan() and lp[1, 5].isnan() and lp.isnan().sum() == 2
        # nothing to score at all
        none = torch.full_like(y, IGNORE)
        leaf = torch.full_like(x, math.nan).requires_grad_()
        zero = torch.zeros(2, device="cuda")
        loss, logprobs, kl = policy_loss(leaf, none, torch.full((2, 6), math.nan, device="cuda"), zero)
        assert float(loss) == 0 and float(kl) == 0 and (logprobs == 0).all()
        assert (torch.autograd.grad(loss, leaf)[0] == 0).all()
        loss, rewards = preference_loss(leaf, none, zero, length_average=True)
        assert abs(float(loss) - math.log(2)) <= 2.0 ** -24 and (rewards == 0).all()
        assert (torch.autograd.grad(loss, leaf)[0] == 0).all()


def test_sequences_of_no_scored_token():
    from pfeife_amd.loss import policy_loss, preference_loss, token_logprobs

    x = torch.randn(2, 1, 11, device="cuda", requires_grad=True)
    y = torch.zeros(2, 1, dtype=torch.int64, device="cuda")
    empty = torch.zeros(2, 0, device="cuda")
    lp = token_logprobs(x, y, shift=True)
    assert lp.shape == (2, 0) and (torch.autograd.grad(lp.sum(), x)[0] == 0).all()
    loss, _, kl = policy_loss(x, y, empty, torch.ones(2, device="cuda"), shift=True)
    assert float(loss) == 0 and float(kl) == 0 and (torch.autograd.grad(loss, x)[0] == 0).all()
    loss, _ = preference_loss(x, y, torch.zeros(2, device="cuda"), shift=True)
    assert abs(float(loss) - math.log(2)) <= 2.0 ** -24 and (torch.autograd.grad(loss, x)[0] == 0).all()
    assert token_logprobs(x[:0], y[:0]).shape == (0, 1) and token_logprobs(x[:, :0], y[:, :0]).shape == (2, 0)
    none = x[:0].detach().requires_grad_()
    assert torch.autograd.grad(token_logprobs(none, y[:0]).sum(), none)[0].shape == none.shape


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_layouts(dtype):
    """Views, leading dimensions, a broadcast, classes that are not the innermost dimension: the contiguous tensor's results, up to the order of sums.

    Where in its 16 bytes a row begins decides which lane sums which class, so two layouts' sums are two orders of the same: each within
    (V / 64 + 32 + 3 E) 2^-24 of the exact one, E < 16 the mean distance from the maximum at these logits, so 2 * 96 * 2^-24 = 1.2e-5 of
    each other.  A token's log-probability and the logarithm of its ratio differ by that; a reward by a tenth of six of them, the preference loss and its
    slope (at most 1 and 1/4 per reward) by less than 2e-5; a gradient by both its factors, 3e-5, before it is rounded to its type (a step at most)."""
    from pfeife_amd.loss import policy_loss, preference_loss, token_logprobs

    g = torch.Generator().manual_seed(8)
    whole = torch.randn(5, 12, 1031, generator=g).to(dtype).cuda()
    y = torch.randint(0, 999, (4, 6), generator=g).cuda()
    for view in (whole[1:, 1:7, 5:1004], whole.transpose(0, 1)[2:6, :5, 3:1002].transpose(0, 1)[:4], whole[:1, :6, 1:1000].expand(4, 6, 999),
                 whole[:4, :6, :999].transpose(1, 2).contiguous().transpose(1, 2)):
        labels = y[:, :view.shape[1]]      # (rows of a wider tensor)
        B, T, _ = view.shape
        old, adv = torch.randn(B, T, generator=g).cuda() - 7.0, torch.randn(B, generator=g).cuda()
        plain = view.contiguous()
        for fn in (lambda t: token_logprobs(t, labels), lambda t: preference_loss(t, labels, old[:, 0] * T)[0],
                   lambda t: policy_loss(t, labels, old, adv)[0]):
            a, b = view.detach().requires_grad_(), plain.clone().requires_grad_()
            ra, rb = fn(a), fn(b)
            assert ((ra - rb).abs() <= 2e-5 * (1 + rb.abs())).all()
            (da,), (db,) = torch.autograd.grad(ra.sum(), a), torch.autograd.grad(rb.sum(), b)
            step = 0.0 if dtype == torch.float32 else 2 * U[dtype]
            assert da.shape == view.shape and ((da - db).double().abs() <= (3e-5 + step) * db.double().abs() + 2 * LEAST[dtype]).all()
    x = whole[:4, :6, :999].contiguous()
    lp = token_logprobs(x, y)
    assert torch.equal(token_logprobs(x.view(2, 2, 6, 999), y.view(2, 2, 6)), lp.view(2, 2, 6)) and torch.equal(token_logprobs(x[0], y[0]), lp[0])


def test_advantages_broadcast():
    from pfeife_amd.loss import policy_loss

    x, y = make(torch.float32, 3, 5, 77, 0, seed=9)
    lp = logprobs64(x, y, 0)[1].detach()
    old, _, adv = policy_operands(lp, 10)
    per = adv[:, 1].contiguous()
    want = policy_loss(x, y, old, per.unsqueeze(1).expand(3, 5).contiguous())
    for a in (per, per.unsqueeze(1), per.unsqueeze(1).expand(3, 5), adv[:, 1], per.double(), torch.stack((per, per), 1)[:, 0]):
        got = policy_loss(x, y, old, a)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    one = x[:, :1], y[:, :1], old[:, :1]
    assert torch.equal(policy_loss(*one, per)[0], policy_loss(*one, per.unsqueeze(1))[0])


def test_rows_behind_and_between_stay_as_they_are(hip):
    """The C entries write the rows they are given and nothing else, at any alignment."""
    g = torch.Generator().manual_seed(11)
    for dtype, V in itertools.product((torch.float32, torch.float16, torch.bfloat16), (1, 13, 1021, 20011)):
        B, T = 2, 3
        sb, st = T * (V + 3) + 5, V + 3
        src = torch.randn(B * sb + 9, generator=g).to(dtype).cuda()
        y = torch.randint(0, V, (B, T), generator=g).cuda()
        y[1, 2] = IGNORE
        for at in (0, 1, 3):
            x = src[at:].as_strided((B, T, V), (sb, st, 1), at)
            out = torch.full((B * sb + 16,), 7.0, dtype=dtype, device="cuda")
            d = out.as_strided((B, T, V), (sb, st, 1), 2 + at)
            rows = (x, B, T, V, sb, st, y, 1, IGNORE, 1.0)
            lp, stats = torch.full((7,), 7.0, device="cuda"), torch.full((12,), 7.0, device="cuda")
            hip.run("token_logprob_fwd", rows, lp, stats)
            coef = torch.ones(B, T - 1, device="cuda")
            hip.run("token_logprob_bwd", rows, stats, coef, (T - 1, 1), d, (sb, st))
            torch.cuda.synchronize()
            assert (lp[4:] == 7).all() and (stats[8:] == 7).all()
            seen = torch.zeros(out.numel(), dtype=torch.bool, device="cuda")
            seen.as_strided((B, T, V), (sb, st, 1), 2 + at).fill_(True)
            assert (out[~seen] == 7).all() and (d[:, -1] == 0).all() and (d[1, 1] == 0).all() and not (d[0, 0] == 7).any()
            want = torch.log_softmax(x[:, :-1].double(), -1)
            z = want.gather(-1, y[:, 1:].clamp_min(0).unsqueeze(-1)).squeeze(-1) * (y[:, 1:] != IGNORE)
            assert torch.allclose(lp[:4].view(2, 2).double(), z, rtol=0, atol=(V / 64 + 48) * 2.0 ** -24 + 20 * 2.0 ** -24)


def test_offsets_past_32_bits():
    """Rows whose first element lies more than 2^32 elements into their tensor (strides alone: most of it is never touched)."""
    from pfeife_amd.loss import policy_loss

    V, B, T = 1000, 2, 3
    room = torch.empty((1 << 32) + (1 << 20), dtype=torch.bfloat16, device="cuda")
    far = room.as_strided((B, T, V), (1 << 32, 300_000, 1), 0)
    x = torch.randn(B, T, V, device="cuda").to(torch.bfloat16)
    far.copy_(x)
    y = torch.randint(0, V, (B, T), device="cuda")
    old, adv = torch.full((B, T), -7.0, device="cuda"), torch.ones(B, device="cuda")
    a, b = far.detach().requires_grad_(), x.clone().requires_grad_()
    la, lb = policy_loss(a, y, old, adv)[0], policy_loss(b, y, old, adv)[0]
    assert torch.equal(la, lb) and torch.equal(torch.autograd.grad(la, a)[0], torch.autograd.grad(lb, b)[0])


def test_another_stream_and_graphs():
    from pfeife_amd.loss import policy_loss, preference_loss, token_logprobs

    x, y = make(torch.bfloat16, 4, 40, 5003, 1, seed=12)
    old, ref, adv = (t.contiguous() for t in policy_operands(logprobs64(x, y, 1)[1].detach(), 13))
    total = torch.full((4,), -100.0, device="cuda")

    def step(t):
        leaf = t.detach().requires_grad_()
        a = policy_loss(leaf, y, old, adv[:, 0], ref, kl_coef=0.1, shift=True)
        b = preference_loss(leaf, y, total, shift=True)
        c = token_logprobs(leaf, y, shift=True)
        return (*(v.detach() for v in (*a, *b, c)), torch.autograd.grad(a[0], leaf)[0], torch.autograd.grad(b[0], leaf)[0], torch.autograd.grad(c.sum(), leaf)[0])

    want = step(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    static = x.clone()
    graphs, outs = [], []
    for _ in range(2):       # two graphs, replayed in turn with eager work between
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(static))
        graphs.append(graph)
    for k in range(4):
        fresh = torch.roll(x, k, 1)
        static.copy_(fresh)
        want = step(fresh)
        graphs[k % 2].replay()
        graphs[1 - k % 2].replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(p, q) for p, q in zip(out, want)), k


def test_a_graph_of_the_backward_pass_alone():
    """The gradient that the eager forward pass wrote is not what a graph's replays hand out: somebody may have changed it."""
    from pfeife_amd.loss import policy_loss

    x, y = make(torch.float32, 2, 8, 301, 0, seed=14)
    old, _, adv = policy_operands(logprobs64(x, y, 0)[1].detach(), 15)
    leaf = x.clone().requires_grad_()
    (want,) = torch.autograd.grad(policy_loss(leaf, y, old, adv)[0], leaf)
    side = torch.cuda.Stream()       # (a backward pass runs where its forward pass ran)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = x.clone().requires_grad_()       # (a leaf of its own: of one that an eager graph holds no backward pass may be captured)
        loss = policy_loss(other, y, old, adv)[0]
        one = torch.ones_like(loss)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        (d,) = torch.autograd.grad(loss, other, one, retain_graph=True)
    for _ in range(3):
        d.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert (d - want).abs().max() <= 8 * 2.0 ** -24 * want.abs().max()
    torch.cuda.synchronize()


def test_runs_repeat_themselves_bit_for_bit():
    from pfeife_amd.loss import policy_loss

    x, y = make(torch.float16, 4, 65, 32003, 1, seed=16)
    old, ref, adv = policy_operands(logprobs64(x, y, 1)[1].detach(), 17)
    seen = []
    for _ in range(3):
        leaf = x.clone().requires_grad_()
        out = policy_loss(leaf, y, old, adv, ref, kl_coef=0.05, shift=True)
        seen.append([*(t.detach() for t in out), torch.autograd.grad(out[0], leaf)[0]])
    assert all(torch.equal(p, q) for other in seen[1:] for p, q in zip(seen[0], other))


@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("B,T", [(2, 700), (6, 300), (10, 200), (32, 520), (34, 70), (66, 9), (300, 3)])
def test_numbers_of_pairs(B, T, average):
    """From one pair, whose sequences sixteen wavefronts share, to more than one workgroup takes."""
    from pfeife_amd.loss import preference_loss

    x, y = make(torch.float32, B, T, 13, 1, seed=20 + B)
    z, lp, seen, rel = logprobs64(x, y, 1)
    n = seen.sum(1).clamp_min(1).double() if average else torch.ones(B, device="cuda", dtype=torch.float64)
    s = lp.sum(1) / n
    ref = (s.detach() + torch.linspace(-3, 3, B, device="cuda")).float()
    rewards = 0.2 * (s - ref.double())
    want = -F.logsigmoid(rewards[0::2] - rewards[1::2]).mean()
    leaf = x.clone().requires_grad_()
    loss, got = preference_loss(leaf, y, ref, beta=0.2, length_average=average, shift=True)
    off = 0.2 * ((rel + 2.0 ** -24 * (lp.detach().abs() + 4)) * seen).sum(1) / n
    assert ((got.double() - rewards.detach()).abs() <= off + 2.0 ** -24 * rewards.detach().abs()).all()
    assert abs(float(loss.detach()) - float(want.detach())) <= 2 * float(off.mean()) + 2.0 ** -23 * float(want.detach())
    (dz,), (d,) = torch.autograd.grad(want, z), torch.autograd.grad(loss, leaf)
    assert (d[:, :-1].double() - dz).abs().max() <= (2 * float(off.max()) + 64 * 2.0 ** -24) * dz.abs().max() + float(off.max()) * 0.2 / (B // 2)


@pytest.mark.parametrize("sequences", [False, True])
@pytest.mark.parametrize("B,T", [(1, 9000), (17, 40), (40, 7), (2000, 2)])
def test_numbers_of_sequences(B, T, sequences):
    from pfeife_amd.loss import policy_loss

    x, y = make(torch.float32, B, T, 11, 1, seed=30 + B)
    z, lp, seen, rel = logprobs64(x, y, 1)
    old, _, adv = policy_operands(lp.detach(), 31)
    want, _, w, ratio, a, _ = policy64(lp, seen, old, None, adv, 0.0, sequences)
    leaf = x.clone().requires_grad_()
    loss = policy_loss(leaf, y, old, adv, clip=0.2, clip_high=0.28, reduction="sequences" if sequences else "tokens", shift=True)[0]
    dlp = rel + 2.0 ** -24
    assert abs(float(loss.detach()) - float(want.detach())) <= 2 * float((w * ratio * a.abs() * dlp).sum()) + 2.0 ** -24 * abs(float(want.detach())) + 1e-14
    (dz,), (d,) = torch.autograd.grad(want, z), torch.autograd.grad(loss, leaf)
    assert (d[:, :-1].double() - dz).abs().max() <= (2 * float(dlp.max()) + 64 * 2.0 ** -24) * dz.abs().max()


@pytest.mark.parametrize("shape", [(70_000, 1, 8), (1_100_000, 9), (1 << 20, 5), (3, 70_000, 3)])
def test_many_rows(shape):
    """More sequences than a grid has rows, more rows than a launch takes."""
    from pfeife_amd.loss import token_logprobs

    g = torch.Generator().manual_seed(40)
    x = torch.randn(*shape, generator=g).cuda().requires_grad_()
    y = torch.randint(0, shape[-1], shape[:-1], generator=g).cuda()
    y.view(-1)[::7] = IGNORE
    lp = token_logprobs(x, y)
    want = torch.log_softmax(x.detach().double(), -1).gather(-1, y.clamp_min(0).unsqueeze(-1)).squeeze(-1) * (y != IGNORE)
    assert ((lp.double() - want).abs() <= 128 * 2.0 ** -24).all()
    (d,) = torch.autograd.grad(lp.sum(), x)
    dz = -torch.softmax(x.detach().double(), -1)
    dz.scatter_add_(-1, y.clamp_min(0).unsqueeze(-1), torch.ones_like(dz[..., :1]))
    assert ((d.double() - dz * (y != IGNORE).unsqueeze(-1)).abs() <= 128 * 2.0 ** -24).all()


@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 65536), (torch.float16, 49999), (torch.float32, 30000)])
def test_gradients_that_go_past_the_caches(dtype, V):
    """More than 256 MiB: rows here and there against 64 bits, the others by what every row's gradient sums up to."""
    from pfeife_amd.loss import policy_loss, preference_loss, token_logprobs

    B = 2
    T = 270_000_000 // (torch.empty((), dtype=dtype).element_size() * V * B) + 2
    g = torch.Generator(device="cuda").manual_seed(41)
    x = torch.empty(B, T, V, dtype=dtype, device="cuda")
    for b in range(B):
        x[b] = 2.0 * torch.randn(T, V, device="cuda", generator=g)
    y = torch.randint(0, V, (B, T), device="cuda", generator=g)
    y[torch.rand(B, T, device="cuda", generator=g) < 0.3] = IGNORE
    leaf = x.requires_grad_()
    rows = [(b, t) for b in range(B) for t in (0, 1, T // 3, T // 2, T - 2, T - 1)]
    seen = y != IGNORE
    ratio = torch.where(seen, 1.0, math.nan)
    for name, loss, factor in (("logprobs", token_logprobs(leaf, y).sum(), None), ("preference", preference_loss(leaf, y, torch.zeros(B, device="cuda"), beta=1e-6)[0], None),
                               ("policy", policy_loss(leaf, y, token_logprobs(x.detach(), y) * ratio, torch.ones(B, device="cuda"))[0], -1.0 / int(seen.sum()))):
        (d,) = torch.autograd.grad(loss, leaf)
        if name == "preference":      # the rewards are small: sigma(0) - 1 = -1/2
            factor = torch.tensor([-0.5e-6, 0.5e-6], device="cuda", dtype=torch.float64)
        elif name == "logprobs":
            factor = 1.0
        f = torch.as_tensor(factor, device="cuda", dtype=torch.float64).expand(B)
        for b, t in rows:
            if not seen[b, t]:
                assert (d[b, t] == 0).all()
                continue
            p = torch.softmax(x.detach()[b, t].double(), -1)
            want = -p * f[b]
            want[y[b, t]] += f[b]
            # rewards up to 1e-6 * T * 20 move sigma by a quarter of that; else the sums' errors and a rounding
            slack = 1e-6 * T * 5 if name == "preference" else 0.0
            tol = want.abs() * (slack + (V / 64 + 96) * 2.0 ** -24 + U[dtype]) + LEAST[dtype]
            assert ((d[b, t].double() - want).abs() <= tol).all(), (name, b, t)
        total = torch.stack([d[b].sum(-1, dtype=torch.float64) for b in range(B)])
        size = f.abs().unsqueeze(1)
        assert (total.abs() <= size * 2 * ((V / 64 + 96) * 2.0 ** -24 + U[dtype]) + V * LEAST[dtype]).all(), name
        assert (d[~seen] == 0).all() if name == "policy" else True
        del d


def test_a_second_derivative_is_refused():
    from pfeife_amd.loss import policy_loss, preference_loss, token_logprobs

    x = torch.randn(2, 3, 7, device="cuda", requires_grad=True)
    y = torch.ones(2, 3, dtype=torch.int64, device="cuda")
    zero = torch.zeros(2, device="cuda")
    for loss in (token_logprobs(x, y).sum(), preference_loss(x, y, zero)[0], policy_loss(x, y, torch.full((2, 3), -2.0, device="cuda"), zero + 1)[0]):
        (d,) = torch.autograd.grad(loss, x, create_graph=True)
        assert torch.isfinite(d).all()
        with pytest.raises(RuntimeError, match="once_differentiable|differentiate twice|does not require grad"):
            torch.autograd.grad(d.sum(), x)


def test_saved_tensors_that_move():
    """Hooks that keep what the backward pass needs on the host, and a forward pass that is run again for it."""
    from torch.utils.checkpoint import checkpoint

    from pfeife_amd.loss import policy_loss, preference_loss, token_logprobs

    x, y = make(torch.bfloat16, 4, 9, 1003, 1, seed=50)
    old, ref, adv = policy_operands(logprobs64(x, y, 1)[1].detach(), 51)
    zero = torch.zeros(4, device="cuda")
    for fn in (lambda t: token_logprobs(t, y, shift=True).sum(), lambda t: preference_loss(t, y, zero, shift=True)[0],
               lambda t: policy_loss(t, y, old, adv, ref, kl_coef=0.1, shift=True)[0], lambda t: 3.0 * policy_loss(t, y, old, adv, ref, kl_coef=0.1, shift=True)[0]):
        leaf = x.clone().requires_grad_()
        (want,) = torch.autograd.grad(fn(leaf), leaf)
        with torch.autograd.graph.save_on_cpu():
            loss = fn(leaf)
        junk = [torch.full((1 << k,), 1e30, device="cuda") for k in range(6, 18)]      # (where the scratch was)
        (got,) = torch.autograd.grad(loss, leaf)
        assert torch.equal(got, want)
        (got,) = torch.autograd.grad(checkpoint(fn, leaf, use_reentrant=False), leaf)
        assert torch.equal(got, want)
        del junk


@pytest.mark.parametrize("smoothing", [0.0, 1.0, 0.25])
def test_an_answer_of_no_probability(smoothing):
    """One label's logit is -inf: the difference of the rewards is infinite, the loss so only where a term with a factor other than zero is; the pair's
    gradient is the limit's."""
    from pfeife_amd.loss import preference_loss

    x, y = make(torch.bfloat16, 4, 9, 1003, 0, seed=60)
    y[:, 3] = 5
    ref = torch.zeros(4, device="cuda")
    for gone in (0, 1):
        z = x.clone()
        z[gone, 3, 5] = -torch.inf
        leaf = z.requires_grad_()
        loss, rewards = preference_loss(leaf, y, ref, label_smoothing=smoothing)
        alone, _ = preference_loss(x[2:], y[2:], ref[2:], label_smoothing=smoothing)
        (d,) = torch.autograd.grad(loss, leaf)
        assert rewards[gone] == -torch.inf and torch.isfinite(rewards[2:]).all() and torch.isfinite(d).all()
        up = (0.0 if gone == 0 else 1.0) - (1 - smoothing)           # sigmoid(D) - (1 - smoothing)
        if up == 0:
            assert abs(float(loss.detach()) - 0.5 * float(alone)) <= 2.0 ** -22 * abs(float(alone)) and not d[:2].any()
        else:
            assert loss == torch.inf and d[:2].any()


def test_a_penalty_that_is_only_looked_at():
    """kl_coef 0 with log-probabilities of a reference, some of them -inf: the loss and its gradient are those without it."""
    from pfeife_amd.loss import policy_loss

    x, y = make(torch.bfloat16, 3, 9, 1003, 1, seed=61)
    old, ref, adv = policy_operands(logprobs64(x, y, 1)[1].detach(), 62)
    ref[(y[:, 1:] != -100).nonzero(as_tuple=True)] = -torch.inf
    leaf = x.clone().requires_grad_()
    want, _, _ = policy_loss(leaf, y, old, adv, shift=True)
    loss, _, kl = policy_loss(leaf, y, old, adv, ref, shift=True)
    assert kl == torch.inf and torch.equal(loss, want) and torch.isfinite(loss)
    assert torch.equal(torch.autograd.grad(loss, leaf)[0], torch.autograd.grad(want, leaf)[0])


def test_saved_tensors_of_another_layout():
    """Hooks that hand back the saved logits without the gaps that they had."""
    from pfeife_amd.loss import policy_loss, preference_loss, token_logprobs

    wide, y = make(torch.bfloat16, 4, 9, 1100, 1, seed=52)
    y = torch.where(y < 1003, y, IGNORE)
    old, ref, adv = policy_operands(logprobs64(wide[..., :1003], y, 1)[1].detach(), 53)
    zero = torch.zeros(4, device="cuda")
    for fn in (lambda t: token_logprobs(t, y, shift=True).sum(), lambda t: preference_loss(t, y, zero, shift=True)[0],
               lambda t: 3.0 * policy_loss(t, y, old, adv, ref, kl_coef=0.1, shift=True)[0]):
        leaf = wide.clone().requires_grad_()
        (want,) = torch.autograd.grad(fn(leaf[..., :1003]), leaf)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t):
            loss = fn(leaf[..., :1003])
        (got,) = torch.autograd.grad(loss, leaf)
        assert torch.equal(got, want)
