"""fp16 logits of a runner with loss scaling: the scale is in the token losses' gradients before they are rounded to fp16."""
import pytest
import torch

from test_pipeline_gpu import _fresh_runner
from test_token_loss_gpu import IGNORE, LEAST, U, logprobs64, parts

pytestmark = pytest.mark.gpu

VOCAB, SEQ = 32000, 300


def run(fn, **option):
    """A step of two micro-batches of two sequences -> per micro-batch, (the model's logits, labels, old log-probabilities, the gradient that the last stage gets)"""
    from pfeife_amd.bench_models.llama import LlamaConfig, LlamaForCausalLM, split_stages
    from pfeife_amd.mp import partial_compiler
    from pfeife_amd.option import PipeOption

    torch.manual_seed(7)
    model = LlamaForCausalLM(LlamaConfig(vocab=VOCAB, dim=128, layers=2, heads=2, ffn=344, max_seq=SEQ)).cuda()
    with torch.no_grad():
        for p in model.parameters():
            if p.shape[0] == VOCAB:
                p.mul_(6.0)      # (logits that differ by a few)
    model = split_stages(model, [])[0]
    g = torch.Generator().manual_seed(12)
    ids = torch.randint(0, VOCAB, (4, SEQ), generator=g).cuda()
    labels = ids.clone()
    labels[:, :20] = IGNORE
    runner = _fresh_runner(PipeOption(device_cnt=2, batch_cnt=2, batch_size=2, split_points=["m.layers.1"], mixed_precision="fp16",
                                      optimizer=dict(type="sgd", lr=0.0), **option))
    cmodel = torch.compile(model, backend=partial_compiler)
    seen = []

    def step(ids, labels):
        out = cmodel(ids)
        assert out.dtype == torch.float16
        loss = fn(out, labels)
        seen.append((out.detach().clone(), labels))
        loss.backward()
        return loss.detach()

    runner.set_exec_fn(step)
    runner.step(ids, labels)
    del seen[:]
    scale = runner.worker.scaler_scale()
    runner.step(ids, labels)
    torch.cuda.synchronize()
    grads = [slot.loss_grads[0].clone() for _, slot in sorted(runner.worker.mbs.items())]
    return [(*s, g) for s, g in zip(seen, grads)], scale


def check(d, z, want, g, rel, dg, scale):
    """Every entry within its factors' errors (dg: g's) and one rounding to fp16 of the scaled gradient; z: the scored rows in 64 bits."""
    p, far = parts(z, 1.0)
    tol = g.abs().unsqueeze(-1) * (p * (rel.unsqueeze(-1) + (3 * far + 16) * 2.0 ** -24) + (want != 0) * 8 * 2.0 ** -24) + (1 + p) * dg.unsqueeze(-1)
    tol = scale * tol * (1 + U[torch.float16]) + U[torch.float16] * scale * want.abs() + LEAST[torch.float16]
    off = (d[:, :-1].double() - scale * want).abs() - tol
    assert (off <= 0).all(), float(off.max())
    assert (d[:, -1] == 0).all()


SCALES = [dict(loss_scale="dynamic", init_scale=65536.0), dict(loss_scale=4096.0)]


@pytest.mark.parametrize("option", SCALES, ids=["dynamic", "static"])
@pytest.mark.parametrize("kind", ["policy", "preference", "logprobs"])
def test_small_entries_keep_their_digits(kind, option):
    from pfeife_amd.loss import policy_loss, preference_loss, token_logprobs

    def loss(out, labels):
        with torch.no_grad():
            old = token_logprobs(out, labels, shift=True)
        if kind == "policy":
            return 0.5 * policy_loss(out, labels, old, torch.ones(2, device="cuda"), shift=True)[0]
        if kind == "preference":
            return preference_loss(out, labels, old.sum(1), beta=1e-2, shift=True)[0]
        return -token_logprobs(out, labels, shift=True).sum() / 4096

    cases, scale = run(loss, **option)
    assert scale == option.get("init_scale", option["loss_scale"]) and len(cases) == 2
    for out, labels, d in cases:
        z, lp, seen, rel = logprobs64(out, labels, 1)
        dlp = (rel + 2.0 ** -24 * (lp.detach().abs() + 4)) * seen      # (of a token's log-probability, in fp32)
        if kind == "policy":          # ratios to log-probabilities that are the same up to that
            g, dg = -0.5 * seen / seen.sum(), 0.5 * 2 * dlp / seen.sum()
        elif kind == "preference":    # rewards of 0 up to the sequence's: sigma(0) - 1, sigma' = 1 / 4
            g = torch.tensor([[-0.5e-2], [0.5e-2]], device="cuda", dtype=torch.float64) * seen
            dg = 1e-2 * seen * (1e-2 * 2 * dlp.sum() / 4)
        else:
            g, dg = -seen.double() / 4096, 0.0 * dlp
        (want,) = torch.autograd.grad(lp, z, g)
        check(d, z, want, g, rel, dg, scale)
        # what a scale is for: nothing becomes zero but what it does not lift to fp16's least number (how many these are is up to the logits)
        assert (d[:, :-1][want.abs() * scale >= 2.0 ** -24] != 0).all()


@pytest.mark.parametrize("option", SCALES, ids=["dynamic", "static"])
def test_logits_that_something_else_reads_too(option):
    """A gradient that is summed up from two is the sum, scaled, as it was: rounded to fp16 before and behind."""
    from pfeife_amd.loss import token_logprobs

    cases, scale = run(lambda out, labels: -token_logprobs(out, labels, shift=True).sum() / 64 + (out.float() ** 2).mean(), **option)
    for out, labels, d in cases:
        z, lp, seen, rel = logprobs64(out, labels, 1)
        (want,) = torch.autograd.grad(lp, z, -seen.double() / 64)
        want = torch.cat((want, torch.zeros_like(want[:, :1])), 1) + 2 * out.double() / out.numel()
        tol = scale * (2.0 ** -9 * want.abs() + 2.0 ** -23 + 2.0 ** -10 / 64 * (want.abs() > 2.0 ** -8)) + LEAST[torch.float16]
        assert ((d.double() - scale * want).abs() <= tol).all()


def test_a_hook_of_the_callers_own():
    """One that the caller's code puts on the logits sees the gradient as before, and what it returns goes where it went."""
    from pfeife_amd.loss import token_logprobs

    looked = []

    def loss(out, labels):
        out.register_hook(lambda g: looked.append(float(g.abs().max())))
        return -token_logprobs(out, labels, shift=True).sum() / 4096

    cases, scale = run(loss, loss_scale=4096.0)
    assert len(looked) >= 4 and all(0 < v <= 1 / 4096 for v in looked)
    assert all(0.5 <= float(d.abs().max()) <= 1.0 for _, _, d in cases)
