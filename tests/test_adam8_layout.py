"""The order of memory that 8-bit moments belong to, without a GPU."""
import copy

import pytest
import torch

CL = torch.channels_last


def parameter(layout=torch.contiguous_format, shape=(32, 16, 4, 4)):
    return torch.nn.Parameter(torch.randn(*shape).to(memory_format=layout))


def state(p):
    from pfeife_amd.optim import AdamW8bit

    opt = AdamW8bit([p])
    return opt, opt._init_state(p, opt.param_groups[0])


@pytest.mark.parametrize("mine,theirs", [(CL, torch.contiguous_format), (torch.contiguous_format, CL)])
def test_state_of_another_layout_is_refused(mine, theirs):
    """Loaded into a parameter that lies otherwise, or one that was laid out anew between two steps."""
    p, q = parameter(mine), parameter(theirs)
    opt, st = state(p)
    opt._check_layout(p, st)
    other, _ = state(q)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    with pytest.raises(RuntimeError, match="does not fit"):
        other._check_layout(q, other.state[q])
    p.data = p.data.contiguous(memory_format=theirs)
    with pytest.raises(RuntimeError, match="does not fit"):
        opt._check_layout(p, st)
    p.data = p.data.contiguous(memory_format=mine)
    opt._check_layout(p, st)


@pytest.mark.parametrize("layout", [CL, torch.contiguous_format])
def test_state_of_the_same_layout_fits(layout):
    p, q = parameter(layout), parameter(layout)
    opt, st = state(p)
    other, _ = state(q)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    other._check_layout(q, other.state[q])
    assert torch.equal(other.state[q]["layout"], st["layout"]) and other.state[q]["layout"].dtype == torch.int64
    # a state that says nothing is taken as the parameter's own, from then on
    del st["layout"]
    opt._check_layout(p, st)
    p.data = p.data.contiguous(memory_format=CL if layout is not CL else torch.contiguous_format)
    with pytest.raises(RuntimeError, match="does not fit"):
        opt._check_layout(p, st)


@pytest.mark.parametrize("shape", [(64, 80, 1, 1), (1, 80, 8, 8), (5120, 1, 2, 1)])
def test_dimensions_of_one_are_of_no_account(shape):
    """Strides that differ where they are never used, and shapes that join: the same order of memory."""
    a = torch.randn(*shape)
    p = torch.nn.Parameter(a)
    opt, st = state(p)
    p.data = a.as_strided(shape, [s if n > 1 else 7 for n, s in zip(shape, a.stride())])
    opt._check_layout(p, st)
    p.data = a.view(-1, shape[-1])
    opt._check_layout(p, st)
