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


def optimizers():
    from pfeife_amd.optim import AdamW8bit

    return [torch.optim.Adam, torch.optim.AdamW, AdamW8bit]


@pytest.fixture(params=range(3), ids=["Adam", "AdamW", "AdamW8bit"])
def make(request):
    return optimizers()[request.param]


def test_a_late_gradient_under_a_scaler(make, monkeypatch):
    """The same where the device counts the steps, some of which an overflow skips."""
    a, b, late = make_parameters(8, 5, 6)
    opt = make([a, b, late], lr=0.1)
    step = Steps(make_worker(True), opt, monkeypatch)
    assert [step(a, b) for _ in range(3)] == [[1, 1], [2, 2], [3, 3]]
    assert step(a, b, overflow=True) == [None, None]
    assert step(a, late, b) == [4, 1, 4]
    assert step(a, late, b, overflow=True) == [None] * 3
    assert step(a, late, b) == [5, 2, 5]
    assert counts(opt) == [5, 5, 2]
    assert step(a, late) == [6, 3]
    assert step(a, late) == [7, 4]
    assert step(a, late, b) == [8, 5, 6]
    assert step(late, a, b) == [6, 9, 7]
    assert step(late) == [7]
    assert step(late, a) == [8, 10]
    assert counts(opt) == [10, 7, 8]


def test_a_group_without_gradients(make, monkeypatch):
    """All of a group's gradients gone for a while: the device's count goes on, the group's does not."""
    a, b = make_parameters(8, 5)
    opt = make([{"params": [a]}, {"params": [b], "lr": 0.2}], lr=0.1)
    step = Steps(make_worker(True), opt, monkeypatch)
    assert [step(a, b), step(a), step(a), step(a, b), step(a, b)] == [[1, 1], [2], [3], [4, 2], [5, 3]]
    assert counts(opt) == [5, 3]
    assert [step(b), step(b)] == [[4], [5]] and counts(opt) == [5, 5]


def test_an_older_state_that_is_loaded(make, monkeypatch):
    """Loaded after steps that nobody asked the counts of: the next step is the loaded state's next, not the device's."""
    import copy

    a, b = make_parameters(8, 5)
    opt = make([a, b], lr=0.1)
    step = Steps(make_worker(True), opt, monkeypatch)
    assert [step(a, b) for _ in range(2)][-1] == [2, 2]
    saved = copy.deepcopy(opt.state_dict())
    assert [step(a, b) for _ in range(3)][-1] == [5, 5]
    opt.load_state_dict(copy.deepcopy(saved))      # (torch's optimizers go on counting in the tensors that they are given)
    assert counts(opt) == [2, 2]
    assert [step(a, b), step(a, b, overflow=True), step(a, b)] == [[3, 3], [None, None], [4, 4]]
    assert counts(opt) == [4, 4]
    # a state that one parameter is not in
    del saved["state"][1]
    step(a, b)
    opt.load_state_dict(saved)
    assert [step(a, b), step(a, b)] == [[3, 1], [4, 2]] and counts(opt) == [4, 2]


def test_its_own_state_that_is_loaded(make, monkeypatch):
    """What state_dict() gives shares the optimizer's tensors, as torch's optimizers have it: it knows of the steps since."""
    a, b = make_parameters(8, 5)
    opt = make([a, b], lr=0.1)
    step = Steps(make_worker(True), opt, monkeypatch)
    step(a, b)
    live = opt.state_dict()
    step(a, b), step(a, b)
    opt.load_state_dict(live)
    assert step(a, b) == [4, 4] and counts(opt) == [4, 4]


def test_an_optimizer_that_changes_workers(make, monkeypatch):
    """One that has stepped before it is given to a worker, another in its place, and the counts that stay when the worker goes."""
    a, b, c = make_parameters(8, 5, 3)
    opt, other = make([a, b], lr=0.1), make([c], lr=0.1)
    plain = Steps(make_worker(False), opt, monkeypatch)
    assert [plain(a, b), plain(a, b)] == [[1, 1], [2, 2]]
    w = make_worker(True)
    step = Steps(w, opt, monkeypatch)
    assert [step(a, b), step(a, b)] == [[3, 3], [4, 4]]
    step = Steps(w, other, monkeypatch)
    assert [step(c), step(c)] == [[1], [2]]
    assert counts(opt) == [4, 4] and counts(other) == [2]
    step = Steps(w, opt, monkeypatch)
    assert step(a, b) == [5, 5]
    w.sync_optimizer_steps()      # (as release() does)
    assert [float(opt.state[p]["step"]) for p in (a, b)] == [5, 5] and counts(other) == [2]


def test_a_step_without_any_gradient(make, monkeypatch):
    """It is nobody's; the device's count is the others' again afterwards."""
    a, b = make_parameters(8, 5)
    opt = make([a, b], lr=0.1)
    w = make_worker(True)
    step = Steps(w, opt, monkeypatch)
    assert [step(a, b), step(a, b)] == [[1, 1], [2, 2]]
    before = float(w.scaler_state[3])
    assert step() == [] and float(w.scaler_state[3]) == before + 1 and counts(opt) == [2, 2]
    assert [step(a, b), step(a, b)] == [[3, 3], [4, 4]] and counts(opt) == [4, 4]
    # the same group in a new dict, which a table of addresses cannot tell from the old one
    group = opt.param_groups[0]
    opt.param_groups[0] = dict(group, lr=0.2)
    assert step(a, b) == [5, 5] and counts(opt) == [5, 5]


def test_a_step_that_fails_before_the_optimizers(make, monkeypatch):
    """Its tables were made; the next step finds them as they are and knows the counts all the same."""
    from pfeife_amd.optim import AdamW8bit

    a, b, late = make_parameters(8, 5, 6)
    opt = make([a, b, late], lr=0.1)
    w = make_worker(True)
    step = Steps(w, opt, monkeypatch)
    prepare = w._adam8_prepare if make is AdamW8bit else w._fused_adam_prepare
    a.grad, b.grad = torch.ones(8), torch.ones(5)
    prepare(opt, True)
    assert [step(a, b), step(a, b)] == [[1, 1], [2, 2]]
    late.grad = torch.ones(6)
    prepare(opt, True)
    assert [step(a, b, late), step(a, b, late)] == [[3, 3, 1], [4, 4, 2]] and counts(opt) == [4, 4, 2]


def test_the_first_gradients_come_late(make, monkeypatch):
    a, b = make_parameters(8, 5)
    opt = make([a, b], lr=0.1)
    step = Steps(make_worker(True), opt, monkeypatch)
    assert [step(), step()] == [[], []]
    assert [step(a, b), step(a, b)] == [[1, 1], [2, 2]] and counts(opt) == [2, 2]


@pytest.mark.parametrize("scaled", [False, True])
def test_loaded_state_lets_the_old_one_go(make, scaled, monkeypatch):
    import copy
    import weakref

    a, b = make_parameters(8, 5000)
    opt = make([a, b], lr=0.1)
    step = Steps(make_worker(scaled), opt, monkeypatch)
    step(a, b), step(a, b)
    saved = copy.deepcopy(opt.state_dict())
    old = [weakref.ref(st["exp_avg"]) for st in opt.state.values()]
    opt.load_state_dict(saved)
    assert all(t() is None for t in old)
    assert step(a, b) == [3, 3]


def test_a_launch_that_is_refused_leaves_the_count(make, monkeypatch):
    a, late = make_parameters(8, 6)
    opt = make([a, late], lr=0.1)
    w = make_worker(True)
    step = Steps(w, opt, monkeypatch)
    step(a), step(a), step(a, late)
    count, refused = float(w.scaler_state[3]), []

    def refuse(self, table, n_items, n_chunks, lr, b1, b2, eps, decay, adamw, state, stream):
        if late.data_ptr() in table:
            refused.append(float(state[3]))
            raise RuntimeError("refused")

    monkeypatch.setattr(Kernels, "adam_step_scaled", refuse)
    with pytest.raises(RuntimeError, match="refused"):
        step(a, late)
    assert refused == [1.0] and float(w.scaler_state[3]) == count
