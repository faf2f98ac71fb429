"""Which step every parameter is at: the fused optimizer steps' bias corrections, on the CPU with a kernel table that notes the counts."""
import pytest
import torch


class Kernels:
    """What the worker asks of the kernels for an optimizer's step; `used`: per launch, the parameters in it and the step that it makes."""

    def __init__(self):
        self.used = []

    def adam_table(self, params, grads, exp_avgs, exp_avg_sqs):
        return [p.data_ptr() for p in params], len(params), 1

    def adam8_table(self, items):
        return [i[0].data_ptr() for i in items], len(items), 1

    def adam_step(self, table, n_items, n_chunks, lr, b1, b2, eps, decay, step, adamw, stream):
        self.used.append((table, float(step)))

    def adam_step_scaled(self, table, n_items, n_chunks, lr, b1, b2, eps, decay, adamw, state, stream):
        if float(state[2]) == 0.0:
            self.used.append((table, float(state[3]) + 1.0))

    def adam8_step(self, table, n_items, n_chunks, lr, b1, b2, eps, decay, step, state, stream):
        if state is None:
            self.used.append((table, float(step)))
        else:
            self.adam_step_scaled(table, n_items, n_chunks, lr, b1, b2, eps, decay, True, state, stream)


def make_worker(scaled):
    from pfeife_amd.mp.worker import StageWorker

    w = StageWorker.__new__(StageWorker)
    w.kernels, w.stream_obj, w.device, w.dyn_scale = Kernels(), None, torch.device("cpu"), scaled
    w.scaler_state = torch.tensor([1024.0] + [0.0] * 7) if scaled else None
    return w


def make_parameters(*sizes):
    return [torch.nn.Parameter(torch.randn(n)) for n in sizes]


class Steps:
    """Steps of a worker's optimizer -> {parameter: the step that it made}"""

    def __init__(self, w, opt, monkeypatch):
        from pfeife_amd import optim

        self.w = w
        w.optimizer = opt
        monkeypatch.setattr(optim, "_raw_stream", lambda index: 0)
        monkeypatch.setattr(optim.AdamW8bit, "_check", staticmethod(lambda p, g, *_: g))

    def __call__(self, *grads, overflow=False):
        """With gradients for these of the optimizer's parameters; as the worker's step does, with the scaler's update behind it."""
        from pfeife_amd.optim import AdamW8bit

        w, opt = self.w, self.w.optimizer
        for p in (p for g in opt.param_groups for p in g["params"]):
            if not any(p is q for q in grads):
                p.grad = None
            elif p.grad is None:
                p.grad = torch.ones_like(p)
        w.kernels.used = []
        if w.dyn_scale:
            w.scaler_state[2] = float(overflow)
        (w._adam8_prepare if type(opt) is AdamW8bit else w._fused_adam_prepare)(opt, w.dyn_scale)()
        if w.dyn_scale:
            w.scaler_state[3] += 1.0 - w.scaler_state[2]
            w.scaler_state[2] = 0.0
        steps = {at: t for table, t in w.kernels.used for at in table}
        assert len(steps) == sum(len(table) for table, _ in w.kernels.used)
        return [steps.get(p.data_ptr()) for p in grads]


def counts(opt):
    return [float(st["step"]) for _, st in sorted(opt.state_dict()["state"].items())]


@pytest.mark.parametrize("make", [torch.optim.Adam, torch.optim.AdamW])
def test_a_late_gradient_starts_at_step_one(make, monkeypatch):
    """Without a loss scaler: a parameter that gets its first gradient after three steps of the others, and one that goes without for a step."""
    a, b, late = make_parameters(8, 5, 6)
    opt = make([a, b, late], lr=0.1)
    step = Steps(make_worker(False), opt, monkeypatch)
    assert [step(a, b) for _ in range(3)] == [[1, 1], [2, 2], [3, 3]]
    assert step(a, late, b) == [4, 1, 4]
    assert step(a, late) == [5, 2]
    assert step(a, late, b) == [6, 3, 5]
    assert step(a, late, b) == [7, 4, 6]
    assert counts(opt) == [7, 6, 4]
