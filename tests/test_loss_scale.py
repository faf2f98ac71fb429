"""When a gradient that reaches the runner may be formed anew with the loss scale in it, without a GPU."""
import torch

from pfeife_amd import loss


class Node(torch.autograd.Function):
    """A loss that leaves with its gradient how to write its multiples."""

    @staticmethod
    def forward(ctx, x):
        return x.sum()

    @staticmethod
    def backward(ctx, grad):
        d = torch.ones(3) * grad
        d._pf_times = d._version, lambda factor, out: out.copy_(factor.expand(3)) is out
        return d


def arrives(use):
    """What scaled_gradient says to the gradient that arrives at the leaf, and writes."""
    x, out, got = torch.zeros(3).requires_grad_(), torch.zeros(3), []
    x.register_hook(lambda g: got.append(loss.scaled_gradient(g, torch.full((1,), 8.0), out)))
    use(x).backward()
    return got, out.tolist()


def test_the_gradient_of_one_loss_alone():
    assert arrives(Node.apply) == ([True], [8.0] * 3)
    nothing = ([False], [0.0] * 3)
    assert arrives(lambda x: x.sum()) == nothing
    assert arrives(lambda x: Node.apply(x) + Node.apply(x)) == nothing
    assert arrives(lambda x: Node.apply(x) + (2 * x).sum()) == nothing
    assert arrives(lambda x: (2 * x).sum() + Node.apply(x)) == nothing
    assert arrives(lambda x: Node.apply(x * 2)) == nothing

    def changed(x):
        x.register_hook(lambda g: g.mul_(2))
        return Node.apply(x)

    assert arrives(changed) == ([True], [8.0] * 3)      # (behind the runner's own)


def test_only_fp16_outputs_of_a_runner_are_marked():
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x = torch.zeros(3, dtype=dtype)
        assert not loss._wants_scale(x)
        loss.mark_loss_scaled(x)
        assert loss._wants_scale(x) == (dtype == torch.float16) and not loss._wants_scale(x.view(3))
