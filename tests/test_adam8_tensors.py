"""Parameters whose memory the caller exchanges under a gradient that stays: what the kernel would read or write out of range is refused (on the
CPU, before anything looks at the device)."""
import pytest
import torch


@pytest.mark.parametrize("seen", [False, True])
@pytest.mark.parametrize("change", ["half", "larger", "smaller", "shorter gradient"])
def test_exchanged_memory(change, seen, monkeypatch):
    from pfeife_amd import optim

    p = torch.nn.Parameter(torch.zeros(6000))
    p.grad = torch.ones(6000)
    opt = optim.AdamW8bit([p])
    if seen:      # a step before, whose addresses are as they were
        monkeypatch.setattr(optim, "_raw_stream", lambda index: 0)

        class Kernels:
            def adam8_table(self, items):
                return items, 1, 1

        check = optim.AdamW8bit._check
        monkeypatch.setattr(optim.AdamW8bit, "_check", staticmethod(lambda p, g, *_: g))
        assert opt._prepare(Kernels())[1] and not opt._prepare(Kernels())[1]
        monkeypatch.setattr(optim.AdamW8bit, "_check", staticmethod(check))
    room = p.data
    if change == "half":
        p.data = room.view(torch.bfloat16)[:6000]
    elif change == "larger":
        p.data = torch.zeros(9000)
    elif change == "smaller":
        p.data = room[:5000]
    else:
        p.grad.data = p.grad.data[:100]
    if seen:
        assert not opt._as_seen(*opt._seen[0])
    st = opt._init_state(p, opt.param_groups[0])
    with pytest.raises(RuntimeError, match="parameters are fp32, gradients of their shape"):
        opt._check(p, p.grad, opt._operands(p, st), st)


def test_groups_that_are_made_anew(monkeypatch):
    """The same parameters in a new group, with another learning rate: the next step is the new group's."""
    from pfeife_amd import optim

    monkeypatch.setattr(optim, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(optim.AdamW8bit, "_check", staticmethod(lambda p, g, *_: g))

    class Kernels:
        def adam8_table(self, items):
            return items, 1, 1

    p = torch.nn.Parameter(torch.zeros(6000))
    p.grad = torch.ones(6000)
    opt = optim.AdamW8bit([p], lr=0.5)
    assert [w[0]["lr"] for w in opt._prepare(Kernels())[0]] == [0.5]
    opt.param_groups.clear()
    opt.add_param_group({"params": [p], "lr": 0.25})
    work, fresh = opt._prepare(Kernels())
    assert [w[0]["lr"] for w in work] == [0.25] and work[0][0] is opt.param_groups[0] and not fresh
    opt.param_groups[0]["lr"] = 0.125
    assert opt._prepare(Kernels())[0][0][0]["lr"] == 0.125
