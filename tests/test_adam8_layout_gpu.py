"""Steps with 8-bit moments of a parameter whose layout in memory changes, or is not the loaded state's."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

CL = torch.channels_last


def test_layouts_that_change():
    from pfeife_amd.optim import AdamW8bit

    g = torch.Generator().manual_seed(80)
    start, grads = torch.randn(32, 16, 4, 4, generator=g).cuda(), [torch.randn(32, 16, 4, 4, generator=g).cuda() for _ in range(3)]

    def make(layout):
        p = torch.nn.Parameter(start.clone(memory_format=torch.contiguous_format).to(memory_format=layout))
        return p, AdamW8bit([p], lr=1e-2)

    def step(p, opt, k):
        p.grad = grads[k].to(memory_format=CL if not p.is_contiguous() else torch.contiguous_format)
        opt.step()

    for layout, another in ((CL, torch.contiguous_format), (torch.contiguous_format, CL)):
        p, opt = make(layout)
        step(p, opt, 0)
        saved = copy.deepcopy(opt.state_dict())
        twin, resumed = make(layout)
        twin.data.copy_(p.data)
        resumed.load_state_dict(saved)
        step(p, opt, 1), step(twin, resumed, 1)
        assert torch.equal(p, twin)
        q, other = make(another)
        other.load_state_dict(saved)
        before = q.detach().clone()
        with pytest.raises(RuntimeError, match="does not fit"):
            step(q, other, 1)
        assert torch.equal(q, before)
        before, moments = p.detach().clone(), opt.state[p]["exp_avg"].view(torch.uint8).clone()
        p.data = p.data.contiguous(memory_format=another)
        with pytest.raises(RuntimeError, match="does not fit"):
            step(p, opt, 2)
        assert torch.equal(p, before) and torch.equal(opt.state[p]["exp_avg"].view(torch.uint8), moments)
        p.data = p.data.contiguous(memory_format=layout)
        step(p, opt, 2), step(twin, resumed, 2)
        assert torch.equal(p, twin) and opt.state[p]["step"] == 3
