"""The token losses at the ends of what they accept, against the same in 64 bits."""
import math

import pytest
import torch

from test_token_loss_gpu import LEAST, U, check_gradient, logprobs64, make, parts, policy_operands

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("smoothing", [0.0, 1.0, 1e-12])
def test_pairs_far_apart(smoothing):
    """The slope of a pair whose rewards differ by 30 and by 40, either way: what is left of it is small and has all its digits.  It is off by D's
    error times itself (|d ln sigma / dD| <= 1), a gradient's entry by that, p's error and a few roundings."""
    from pfeife_amd.loss import preference_loss

    x, y = make(torch.float32, 8, 5, 37, 0, seed=70)
    y[1, 2] = 3
    z, lp, seen, rel = logprobs64(x, y, 0)
    s = lp.detach().sum(1)
    far = torch.tensor([30.0, -30.0, 40.0, -40.0], device="cuda", dtype=torch.float64)
    ref = torch.stack((s[0::2] - far / 2, s[1::2] + far / 2), 1).reshape(-1).float()
    rewards = s - ref.double()
    D = rewards[0::2] - rewards[1::2]
    up = (smoothing * torch.sigmoid(D) - (1 - smoothing) * torch.sigmoid(-D)) / 4
    g = torch.stack((up, -up), 1).view(-1, 1) * seen
    off = ((rel + 2.0 ** -24 * (lp.detach().abs() + 4)) * seen).sum(1).view(-1, 2).sum(1).repeat_interleave(2).unsqueeze(1)
    leaf = x.clone().requires_grad_()
    loss, _ = preference_loss(leaf, y, ref, beta=1.0, label_smoothing=smoothing)
    (d,) = torch.autograd.grad(loss, leaf)
    (dz,) = torch.autograd.grad(lp, z, g)
    check_gradient(d, dz, g, *parts(z, 1.0), rel, torch.float32, g.abs() * (off + 2.0 ** -22))
    assert (d[seen].abs().amax(-1) > 0).all() if smoothing else (d[:2][seen[:2]].abs().amax(-1) > 1e-15).all()


@pytest.mark.parametrize("temperature", [1.0, 1e-6])
def test_huge_logits(temperature):
    """Rows whose largest logits over the temperature lie between 2^30 and 2^34, where fp32 numbers are hundreds apart: two classes share a row's
    probability to the last digit, however small the gradient that comes in."""
    from pfeife_amd.loss import policy_loss, token_logprobs

    n = 2000
    g = torch.Generator().manual_seed(71)
    top = (2.0 ** (30 + 4 * torch.rand(n, generator=g, dtype=torch.float64)) * temperature).float()
    x = torch.stack((top / 2, top, -top, top, top * 0.75), 1).unsqueeze(0).cuda()
    y = torch.full((1, n), 3, device="cuda")
    for small in (1e-6, 1e-12):
        leaf = x.clone().requires_grad_()
        lp = token_logprobs(leaf, y, temperature=temperature)
        assert ((lp + math.log(2)).abs() <= 4 * 2.0 ** -24).all()
        for out, inflow in ((lp, torch.full_like(lp, small)),
                            (policy_loss(leaf, y, lp.detach(), torch.full((1,), -small * n, device="cuda"), temperature=temperature)[0], None)):
            (d,) = torch.autograd.grad(out, leaf, inflow)
            want = 0.5 * small / temperature * torch.tensor([0.0, -1.0, 0.0, 1.0, 0.0], device="cuda", dtype=torch.float64)
            assert ((d.double() - want).abs() <= 16 * 2.0 ** -24 * want.abs()).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [1e-6, 1e6])
def test_temperatures_at_the_ends(dtype, temperature):
    """At 1e-6 a row's probability lies on its largest logits alone, at 1e6 on all alike; the labels of the first are the largest or near it."""
    from pfeife_amd.loss import policy_loss, token_logprobs

    x, y = make(dtype, 2, 40, 1003, 0, seed=72, masked=0.2)
    if temperature < 1:
        at = y.clamp_min(0).unsqueeze(-1)
        x.scatter_(2, at, x.amax(-1, keepdim=True))      # (its equal, so half of the probability)
        x[:, ::3] *= 1e-6                                # and rows whose logits over the temperature are ordinary
    z, lp, seen, rel = logprobs64(x, y, 0, temperature)
    assert torch.isfinite(lp).all()
    leaf = x.clone().requires_grad_()
    got = token_logprobs(leaf, y, temperature=temperature)
    # (x - m) / temperature of the label is formed from fp32 factors where the sum is: some 2^-23 of it
    far = ((z.amax(-1) - z.gather(-1, y.clamp_min(0).unsqueeze(-1)).squeeze(-1)) / temperature).detach()
    tol = rel + 2.0 ** -24 * (lp.detach().abs() + 4) + 2.0 ** -22 * far
    assert ((got.double() - lp).abs() <= tol)[seen].all()
    inflow = torch.linspace(-2, 2, lp.numel(), device="cuda").view(lp.shape)
    (d,), (dz,) = torch.autograd.grad(got, leaf, inflow), torch.autograd.grad(lp, z, inflow.double(), retain_graph=True)
    check_gradient(d, dz, inflow.double() * seen / temperature, *parts(z, temperature), rel, dtype, torch.zeros_like(rel))
    loss, logprobs, _ = policy_loss(leaf, y, got.detach() - 0.1, torch.ones(2, device="cuda"), temperature=temperature)
    assert ((logprobs.double() - lp).abs() <= tol)[seen].all()
    (d,) = torch.autograd.grad(loss, leaf)
    ratio = torch.exp(lp.detach() - (got.detach() - 0.1).double())
    gg = -ratio * seen / seen.sum()
    (dz,) = torch.autograd.grad(lp, z, gg)
    check_gradient(d, dz, gg / temperature, *parts(z, temperature), rel, dtype, gg.abs() / temperature * (2 * tol + 2.0 ** -22))


@pytest.mark.parametrize("clip,clip_high", [(0.0, 0.0), (1.0, 0.28), (1.5, 3.0), (0.2, 1e30)])
def test_wide_and_no_clips(clip, clip_high):
    """A lower bound of one or more never holds (a ratio is positive), nor does an upper one that no ratio reaches; with none at all every ratio
    but one is outside."""
    from pfeife_amd.loss import policy_loss

    x, y = make(torch.float32, 3, 30, 101, 0, seed=73)
    z, lp, seen, rel = logprobs64(x, y, 0)
    old, ref, adv = policy_operands(lp.detach(), 74)
    old -= 0.01 * (old == lp.float())       # (no ratio at a border)
    ratio = torch.exp(lp - old.double())
    a = adv.double()
    token = -torch.minimum(ratio * a, ratio.clamp(1 - clip, 1 + clip_high) * a)
    want = torch.where(seen, token, 0.0).sum() / seen.sum()
    leaf = x.clone().requires_grad_()
    loss = policy_loss(leaf, y, old, adv, clip=clip, clip_high=clip_high)[0]
    dlp = (rel + 2.0 ** -24) * seen
    size = (ratio.detach() * a.abs() * seen / seen.sum())
    assert abs(float(loss.detach()) - float(want.detach())) <= float((size * (dlp + 2.0 ** -23)).sum()) * 2 + 2.0 ** -24 * abs(float(want.detach())) + 1e-14
    (d,), (dz,) = torch.autograd.grad(loss, leaf), torch.autograd.grad(want, z)
    free = torch.where(a >= 0, ratio <= 1 + clip_high, ratio >= 1 - clip)
    g = torch.where(free & seen, -a * ratio.detach() / seen.sum(), 0.0)
    check_gradient(d, dz, g, *parts(z, 1.0), rel, torch.float32, 2 * size * dlp + 2.0 ** -23 * g.abs())


def test_hooks_get_all_of_the_policy_loss_memory():
    """Where hooks take what the backward pass needs off the device, or a checkpoint forgets it, the loss leaves nothing as large as the logits behind.
    The gradient may come from sums in another order (each off by (V / 64 + 96) 2^-24) and be rounded the other way."""
    from torch.utils.checkpoint import checkpoint

    from pfeife_amd.loss import policy_loss

    x, y = make(torch.bfloat16, 2, 64, 65536, 0, seed=75, masked=0.0)
    old, adv = torch.full((2, 64), -10.0, device="cuda"), torch.ones(2, device="cuda")
    leaf = x.requires_grad_()
    (want,) = torch.autograd.grad(policy_loss(leaf, y, old, adv)[0], leaf)
    size = x.numel() * 2

    def left(call):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        loss = call()
        grown = torch.cuda.memory_allocated() - before
        (d,) = torch.autograd.grad(loss, leaf)
        step = 2 * (65536 / 64 + 96) * 2.0 ** -24 + 2 * U[torch.bfloat16]
        assert ((d.double() - want.double()).abs() <= step * want.double().abs() + 2 * LEAST[torch.bfloat16]).all()
        return grown

    def on_cpu():
        with torch.autograd.graph.save_on_cpu():
            return policy_loss(leaf, y, old, adv)[0]

    assert left(lambda: policy_loss(leaf, y, old, adv)[0]) >= size      # (the gradient, which the forward pass writes)
    assert left(on_cpu) < size // 8
    assert left(lambda: checkpoint(lambda t: policy_loss(t, y, old, adv)[0], leaf, use_reentrant=False)) < size // 8
