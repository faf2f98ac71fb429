"""Ends of what the decoder operators accept: losses of no token, compiled models, long forward passes, sizes between two rules."""
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


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
@pytest.mark.parametrize("kept,dtype", [("16bit", torch.bfloat16), ("8bit", torch.float16), ("16bit", torch.float32)])
def test_compiled_without_a_runner(backend, kept, dtype):
    """The bits of the calls that are not compiled, whichever backend runs the graph."""
    from test_decoder_compiled import Layers

    torch._dynamo.reset()
    g = torch.Generator("cuda").manual_seed(4)
    model = Layers(kept, dtype).cuda()
    with torch.no_grad():
        for p in model.parameters():
            p.copy_(torch.randn(p.shape, device="cuda", generator=g))
    ids = torch.randint(0, 11, (3, 70), device="cuda", generator=g)
    up = torch.randn(3, 70, 12, device="cuda", generator=g).to(dtype)
    want = model(ids)
    grads = torch.autograd.grad(want, list(model.parameters()), up)
    got = torch.compile(model, backend=backend, fullgraph=True)(ids)
    assert torch.equal(got, want)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, list(model.parameters()), up), grads))
