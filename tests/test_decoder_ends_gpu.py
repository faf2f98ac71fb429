"""Ends of what the decoder operators accept: losses of no token, long forward passes, sizes between two rules."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,shift", [((2, 1), True), ((0, 4), False), ((3, 0), False)])
def test_a_loss_of_no_token(dtype, shape, shift):
    from pfeife_amd.loss import linear_cross_entropy

    h = torch.full((*shape, 72), float("nan"), device="cuda", dtype=dtype).requires_grad_()
    w = torch.ones(300, 72, device="cuda", dtype=dtype).requires_grad_()
    labels = torch.zeros(shape, dtype=torch.int64, device="cuda")
    for reduction in ("none", "mean", "sum"):
        out = linear_cross_entropy(h, w, labels, shift=shift, reduction=reduction)
        dh, dw = torch.autograd.grad(out.sum(), (h, w))
        assert not out.any() and not dh.any() and not dw.any()
