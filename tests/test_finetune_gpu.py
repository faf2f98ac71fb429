"""The fine-tuning operators together, as a training program has them: a decoder in pipeline stages, its reference model's
log-probabilities, a preference or policy loss behind the last stage, AdamW with 8-bit moments."""
import copy

import pytest
import torch
import torch.nn.functional as F

from test_pipeline_gpu import _fresh_runner

pytestmark = pytest.mark.gpu

SEQ, PROMPT = 64, 20


def decoder():
    from pfeife_amd.bench_models.llama import LlamaConfig, LlamaForCausalLM, split_stages

    torch.manual_seed(7)
    model = LlamaForCausalLM(LlamaConfig(vocab=512, dim=128, layers=4, heads=2, ffn=344, max_seq=SEQ)).cuda()
    return split_stages(model, [])[0]


def batch(sequences):
    g = torch.Generator().manual_seed(11)
    ids = torch.randint(0, 512, (sequences, SEQ), generator=g).cuda()
    labels = ids.clone()
    labels[:, :PROMPT] = -100
    for b in range(sequences):
        labels[b, SEQ - 3 * b:] = -100
    return ids, labels


def plain_logprobs(logits, labels):
    lp = torch.log_softmax(logits[:, :-1].double(), -1).gather(-1, labels[:, 1:].clamp_min(0).unsqueeze(-1)).squeeze(-1)
    return torch.where(labels[:, 1:] != -100, lp, 0.0)


def plain_preference(logits, labels, ref):
    reward = 0.2 * (plain_logprobs(logits, labels).sum(1) - ref.double())
    return -F.logsigmoid(reward[0::2] - reward[1::2]).mean()


def plain_policy(logits, labels, old, adv, ref):
    seen = labels[:, 1:] != -100
    lp = plain_logprobs(logits, labels)
    ratio, a, q = torch.exp(lp - old.double()), adv.double().unsqueeze(1), ref.double() - lp
    token = -torch.minimum(ratio * a, ratio.clamp(0.8, 1.2) * a) + 0.05 * (torch.exp(q) - q - 1)
    return (token * seen).sum() / seen.sum()


@pytest.mark.parametrize("mixed", [None, "bf16", "fp16"])
@pytest.mark.parametrize("kind", ["preference", "policy"])
def test_a_fine_tuning_step(kind, mixed):
    """Losses and gradients of two steps in two stages and four micro-batches against plain PyTorch with plain formulas, and the weights
    after the optimizer's step against AdamW's in 64 bits."""
    from pfeife_amd.loss import PolicyLoss, PreferenceLoss, token_logprobs
    from pfeife_amd.mp import partial_compiler
    from pfeife_amd.option import PipeOption

    model = decoder()
    ref = copy.deepcopy(model)
    ids, labels = batch(8)
    dtype = {"fp16": torch.float16, "bf16": torch.bfloat16}.get(mixed)
    with torch.no_grad(), torch.autocast("cuda", dtype=dtype, enabled=dtype is not None):     # the reference model: the same network, slightly off
        frozen = token_logprobs(ref(ids) * 0.95, labels, shift=True)
    total, old = frozen.sum(1), frozen + 0.05
    adv = torch.linspace(-1.5, 1.0, 8, device="cuda")
    lr = 1e-2
    option = PipeOption(device_cnt=2, batch_cnt=4, batch_size=2, split_points=["m.layers.2"], mixed_precision=mixed,
                        optimizer=dict(type="adamw8bit", lr=lr, weight_decay=0.1, min_8bit_size=1024))
    runner = _fresh_runner(option)
    cmodel = torch.compile(model, backend=partial_compiler)
    crit = PreferenceLoss(beta=0.2, shift=True) if kind == "preference" else PolicyLoss(clip=0.2, kl_coef=0.05, shift=True)

    def fn(ids, labels, total, old, adv, frozen):
        out = cmodel(ids)
        loss = crit(out, (labels, total) if kind == "preference" else (labels, old, adv, frozen))
        loss.backward()
        return loss.detach()

    runner.set_exec_fn(fn)
    for step in range(2):
        before = {n: p.detach().double().clone() for n, p in model.named_parameters()}
        ref.load_state_dict(model.state_dict())
        losses = runner.step(ids, labels, total, old, adv, frozen)
        torch.cuda.synchronize()
        for p in ref.parameters():
            p.grad = None
        for k in range(4):
            s = slice(2 * k, 2 * k + 2)
            with torch.autocast("cuda", dtype=dtype, enabled=dtype is not None):
                out = ref(ids[s])
            want = plain_preference(out, labels[s], total[s]) if kind == "preference" else plain_policy(out, labels[s], old[s], adv[s], frozen[s])
            want.backward()
            want = float(want.detach())
            assert abs(float(losses[k]) - want) <= (1e-4 if mixed is None else 3e-2) * max(1.0, abs(want)), (step, k)
        opt = runner.worker.optimizer
        assert type(opt).__name__ == "AdamW8bit"
        for (n, p), (_, q) in zip(model.named_parameters(), ref.named_parameters()):
            a, b = p.grad.double(), q.grad.double()
            if mixed is None:
                assert (a - b).abs().max() <= 1e-4 * b.abs().max() + 1e-9, (step, n)
            else:
                assert (a - b).norm() <= 3e-2 * b.norm() + 1e-9, (step, n)
            if step == 0:      # from zero moments both bias corrections cancel: a step of lr in the gradient's direction
                move = before[n] * (1 - lr * 0.1) - lr * a / (a.abs() + 1e-8)
                assert ((p.detach().double() - move).abs() <= 1e-5 * lr + 2.0 ** -22 * before[n].abs() + lr * 1e-3 * (a.abs() < 1e-6)).all(), n
            st = opt.state[p]
            assert ("exp_avg_scale" in st) == (p.numel() >= 1024)
        assert {float(st["step"]) for st in opt.state_dict()["state"].values()} == {step + 1.0}


def test_an_overflow_skips_the_step():
    """Dynamic loss scaling: a step whose gradients overflow touches neither weights nor moments nor the count, and halves the scale."""
    from pfeife_amd.loss import preference_loss
    from pfeife_amd.mp import partial_compiler
    from pfeife_amd.option import PipeOption

    model = decoder()
    ids, labels = batch(4)
    total = torch.zeros(4, device="cuda")
    runner = _fresh_runner(PipeOption(device_cnt=2, batch_cnt=2, batch_size=2, split_points=["m.layers.2"], mixed_precision="fp16",
                                      init_scale=1024.0, optimizer=dict(type="adamw8bit", lr=1e-3)))
    cmodel = torch.compile(model, backend=partial_compiler)
    factor = [1.0]

    def fn(ids, labels, total):
        loss = preference_loss(cmodel(ids), labels, total, shift=True)[0] * factor[0]
        loss.backward()
        return loss.detach()

    runner.set_exec_fn(fn)
    state = lambda: [t.clone() for p in model.parameters() for t in (p.detach(), *(v.view(torch.uint8) if v.dtype == torch.float8_e4m3fn else v  # noqa: E731
                                                                                   for k, v in runner.worker.optimizer.state[p].items() if k != "step"))]
    runner.step(ids, labels, total)
    torch.cuda.synchronize()
    before, scale = state(), runner.worker.scaler_scale()
    factor[0] = 1e30
    runner.step(ids, labels, total)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, state())) and runner.worker.scaler_scale() == scale / 2
    factor[0] = 1.0
    runner.step(ids, labels, total)
    torch.cuda.synchronize()
    assert not all(torch.equal(a, b) for a, b in zip(before, state()))
    assert {float(st["step"]) for st in runner.worker.optimizer.state_dict()["state"].values()} == {2.0}
