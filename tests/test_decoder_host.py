"""What the decoder operators do on the host around their launches, without a GPU: tensors of the CPU stand for the GPU's, and nothing is launched
(results hold whatever their memory held)."""
import gc
import weakref
from types import SimpleNamespace

import pytest
import torch

from pfeife_amd import loss


class NothingLaunched:
    """Entry points that succeed, and ask for 256 bytes where they are asked."""

    def __getattr__(self, name):
        return lambda *args: 256 if name.endswith(("_kept", "_workspace")) else 0


@pytest.fixture()
def on_the_cpu(monkeypatch):
    monkeypatch.setattr(loss, "_tables", {-1: SimpleNamespace(lib=NothingLaunched())})
    monkeypatch.setattr(loss, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(loss, "_current_device", lambda: -1)


def test_memory_of_a_scaled_gradient_goes_with_it(on_the_cpu, monkeypatch):
    """What a gradient that a loss scale will be multiplied into keeps (its workspace: hundreds of megabytes) is free as soon as the gradient is, without
    the collector of cycles."""
    h = torch.zeros(2, 3, 8, dtype=torch.float16).requires_grad_()
    w, y = torch.zeros(5, 8, dtype=torch.float16), torch.zeros(2, 3, dtype=torch.int64)
    made, empty = [], torch.empty

    def seen(*args, **kwargs):
        t = empty(*args, **kwargs)
        made.append(weakref.ref(t))
        return t

    loss.mark_loss_scaled(h)
    gc.collect()
    gc.disable()
    try:
        with monkeypatch.context() as patch:
            patch.setattr(torch, "empty", seen)
            out = loss.linear_cross_entropy(h, w, y)
            grad, = torch.autograd.grad(out, h)
        held = sum(t() is not None and t().dtype == torch.uint8 for t in made)
        assert held >= 2      # (what the forward pass left, and the workspace)
        del out, grad
        assert not [t() for t in made if t() is not None]
    finally:
        gc.enable()


def test_what_a_scaled_gradient_is_written_to(on_the_cpu):
    h = torch.zeros(2, 3, 8, dtype=torch.float16).requires_grad_()
    w, y = torch.zeros(5, 8, dtype=torch.float16), torch.zeros(2, 3, dtype=torch.int64)
    loss.mark_loss_scaled(h)
    grad, = torch.autograd.grad(loss.linear_cross_entropy(h, w, y), h)
    scale = torch.ones(1)
    assert loss.scaled_gradient(grad, scale, torch.empty(2, 3, 8, dtype=torch.float16))
    for out in (torch.empty(6, 8, dtype=torch.float16), torch.empty(2, 3, 8), torch.empty(2, 3, 16, dtype=torch.float16)[..., ::2]):
        assert not loss.scaled_gradient(grad, scale, out)
    grad.add_(1)      # (it is another gradient now)
    assert not loss.scaled_gradient(grad, scale, torch.empty(2, 3, 8, dtype=torch.float16))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape,shift", [((2, 1), True), ((0, 4), False), ((0, 4), True), ((3, 0), False)])
def test_a_loss_of_no_token_has_a_gradient_of_zeros(on_the_cpu, dtype, shape, shift):
    """reduction "none" of nothing: its own gradient has no memory that a kernel could be shown."""
    h, w = torch.ones(*shape, 8, dtype=dtype).requires_grad_(), torch.ones(5, 8, dtype=dtype).requires_grad_()
    out = loss.linear_cross_entropy(h, w, torch.zeros(shape, dtype=torch.int64), shift=shift, reduction="none")
    assert out.numel() == 0
    loss._tables[-1].lib = None      # (a backward pass that asks the library for anything fails)
    dh, dw = torch.autograd.grad(out.sum(), (h, w))
    assert dh.shape == h.shape and dw.shape == w.shape and dh.dtype == dw.dtype == dtype
    assert not dh.any() and not dw.any()
