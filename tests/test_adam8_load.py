"""torch.optim.AdamW's state loaded into AdamW8bit, without a GPU."""
import copy

import pytest
import torch


def saved(**kwargs):
    p = torch.nn.Parameter(torch.ones(5000))
    opt = torch.optim.AdamW([p], lr=0.5, **kwargs)
    p.grad = torch.ones(5000)
    opt.step()
    return opt.state_dict()


def test_plain_state_keeps_its_moments():
    from pfeife_amd.optim import AdamW8bit

    p = torch.nn.Parameter(torch.ones(5000))
    opt = AdamW8bit([p])
    state = saved()
    opt.load_state_dict(copy.deepcopy(state))
    assert opt.param_groups[0]["lr"] == 0.5 and float(opt.state[p]["step"]) == 1 and opt._operands(p, opt.state[p])[1] is None
    assert torch.equal(opt.state[p]["exp_avg_sq"], state["state"][0]["exp_avg_sq"])


@pytest.mark.parametrize("option", ["amsgrad", "maximize"])
def test_what_it_cannot_do_is_refused(option):
    """A step in the other direction, or with another denominator, would follow without a word."""
    from pfeife_amd.optim import AdamW8bit

    p = torch.nn.Parameter(torch.ones(5000))
    opt = AdamW8bit([p], lr=0.25)
    with pytest.raises(RuntimeError, match="amsgrad or maximize"):
        opt.load_state_dict(saved(**{option: True}))
    assert opt.param_groups[0]["lr"] == 0.25 and not opt.state.get(p)
