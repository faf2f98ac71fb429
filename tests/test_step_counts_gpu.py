"""Optimizer steps of a runner under dynamic loss scaling whose parameters are not all at one step, against torch's optimizers."""
import copy

import pytest
import torch

from test_pipeline_gpu import _fresh_runner

pytestmark = pytest.mark.gpu

LR = 1e-2


@pytest.mark.parametrize("kind", ["adam", "adamw", "adamw8bit"])
def test_counts_that_differ(kind):
    """A parameter of the caller's own that gets its first gradient after forty steps of the model's, overflows before and after it, an
    older state that is loaded: parameters as torch's optimizer has them from the same gradients (32-bit moments).  Each step's
    update is the formula's in fp32 on both sides, some eight roundings, so 2^-18 of lr (an update is at most a few lr) and a rounding of
    the parameter a step."""
    from pfeife_amd.bench_models.vit import ViTConfig, VisionTransformer
    from pfeife_amd.mp import partial_compiler
    from pfeife_amd.optim import AdamW8bit
    from pfeife_amd.option import PipeOption

    g = torch.Generator().manual_seed(42)
    x, y = torch.randn(8, 3, 32, 32, generator=g).cuda(), torch.randint(0, 10, (8,), generator=g).cuda()
    torch.manual_seed(0)
    model = VisionTransformer(ViTConfig(image_size=32, patch_size=16, dim=64, depth=2, heads=2, mlp_dim=128, num_classes=10)).cuda()
    late = torch.nn.Parameter(torch.randn(300, generator=g).cuda())
    params = [*model.parameters(), late]
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    torch_kind = torch.optim.Adam if kind == "adam" else torch.optim.AdamW
    decay = 0.0 if kind == "adam" else 0.1
    opt = AdamW8bit(params, lr=LR, weight_decay=decay, min_8bit_size=1 << 30) if kind == "adamw8bit" else torch_kind(params, lr=LR, weight_decay=decay)
    want = torch_kind(twins, lr=LR, weight_decay=decay)
    runner = _fresh_runner(PipeOption(device_cnt=2, batch_cnt=2, batch_size=4, split_points=["blocks.1"], loss_scale="dynamic", init_scale=1024.0,
                                      growth_interval=1000))
    runner.optimizer = opt
    cmodel, crit, poison = torch.compile(model, backend=partial_compiler), torch.nn.CrossEntropyLoss(), [False]

    def fn(px, labels):
        loss = crit(cmodel(px).float(), labels)
        (loss * float("inf") if poison[0] else loss).backward()
        return loss.detach()

    runner.set_exec_fn(fn)
    made = 0

    def step(overflow=False):
        nonlocal made
        poison[0] = overflow
        runner.step(x, y)
        torch.cuda.synchronize()
        if not overflow:
            for p, q in zip(params, twins):
                q.grad = None if p.grad is None else p.grad.clone()
            want.step()
            made += 1
        for p, q in zip(params, twins):
            assert ((p - q).detach().abs() <= made * (2.0 ** -18 * LR + 2.0 ** -23 * q.detach().abs())).all(), made
            with torch.no_grad():      # (the next step's gradients are of p)
                q.copy_(p)

    counts = lambda o: [float(st["step"]) for _, st in sorted(o.state_dict()["state"].items())]  # noqa: E731
    for k in range(41):
        step(overflow=k == 20)
        if k == 10:
            saved, theirs = copy.deepcopy(opt.state_dict()), copy.deepcopy(want.state_dict())
    for k in range(3):
        late.grad = torch.randn(300, generator=g).cuda()
        step(overflow=k == 1)
    assert counts(opt) == counts(want) and counts(opt)[-2:] == [42, 2]
    step()
    opt.load_state_dict(saved), want.load_state_dict(theirs)
    late.grad = None
    step()
    late.grad = torch.ones_like(late)
    step()
    assert counts(opt) == counts(want) and counts(opt)[-2:] == [13, 1]


@pytest.mark.parametrize("kind", ["adam", "adamw8bit"])
def test_a_released_worker_keeps_no_moments(kind):
    """The optimizer of the caller's own has its counts, and the one that the worker made goes away with its state."""
    import gc
    import weakref

    from pfeife_amd.bench_models.vit import ViTConfig, VisionTransformer
    from pfeife_amd.mp import partial_compiler
    from pfeife_amd.option import PipeOption

    g = torch.Generator().manual_seed(42)
    x, y = torch.randn(8, 3, 32, 32, generator=g).cuda(), torch.randint(0, 10, (8,), generator=g).cuda()
    model = VisionTransformer(ViTConfig(image_size=32, patch_size=16, dim=64, depth=2, heads=2, mlp_dim=128, num_classes=10)).cuda()
    runner = _fresh_runner(PipeOption(device_cnt=2, batch_cnt=2, batch_size=4, split_points=["blocks.1"], loss_scale="dynamic", init_scale=1024.0,
                                      optimizer=dict(type=kind, lr=1e-3)))
    cmodel, crit = torch.compile(model, backend=partial_compiler), torch.nn.CrossEntropyLoss()

    def fn(px, labels):
        loss = crit(cmodel(px).float(), labels)
        loss.backward()
        return loss.detach()

    runner.set_exec_fn(fn)
    for _ in range(3):
        runner.step(x, y)
    worker, opt = runner.worker, runner.worker.optimizer
    moments = [weakref.ref(st["exp_avg"]) for st in opt.state.values()]
    worker.release()
    assert {float(st["step"]) for st in opt.state.values()} == {3.0} and all(m() is not None for m in moments)
    opt.state.clear()
    del opt
    gc.collect()
    assert all(m() is None for m in moments)
