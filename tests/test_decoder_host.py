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


@pytest.mark.parametrize("dtype,size", [(0, 4), (1, 2), (2, 2)])
@pytest.mark.parametrize("D", [64, 1024, 4096, 8192])
def test_how_many_tokens_a_call_takes(dtype, size, D):
    """A forward pass holds the gathered rows (16 bits: and 512 more rows in reach of a buffer's offsets), a backward pass their gradient in fp32."""
    from pfeife_amd import hip

    lib = hip.load()
    in_fp32 = ((1 << 31) - 65) // (D * 4) // 64 * 64
    for backward, most in ((0, in_fp32 if size == 4 else min(((1 << 31) // (D * 2) - 512) // 256 * 256, (1 << 24) - 1)), (1, in_fp32)):
        need = lambda n: lib.pf_linear_ce_workspace(None, dtype, n, D, 50, backward)  # noqa: E731
        assert need(most) > most * D * (4 if backward else size)
        assert need(most + 1) == -1 and b"too many for one call" in lib.pf_last_error()


def test_a_loss_without_a_possible_gradient_is_refused_before_it_runs(on_the_cpu):
    """... and scored where none is asked for."""
    from pfeife_amd import hip

    lib = hip.load()

    class Sizes(NothingLaunched):
        pf_linear_ce_workspace = staticmethod(lambda *args: 1 << 20 if lib.pf_linear_ce_workspace(*args) > 0 else -1)
        pf_last_error = staticmethod(lib.pf_last_error)

    loss._tables[-1].lib = Sizes()
    h = torch.zeros(1, dtype=torch.bfloat16).expand(1, 131072, 4096)
    w, y = torch.zeros(5, 4096, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int64).expand(1, 131072)
    assert loss.linear_cross_entropy(h, w, y, reduction="none").shape == (1, 131072)
    for a, b in ((h.detach().requires_grad_(), w), (h, w.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="linear_cross_entropy: .*too many for one call"):
            loss.linear_cross_entropy(a, b, y)
    assert loss.linear_cross_entropy(h[:, :65000], w.clone().requires_grad_(), y[:, :65000]).requires_grad


@pytest.mark.parametrize("rows,D,ffn", [(1024, 2048, 5630), (777, 1000, 2732), (300, 512, 1001), (64, 4096, 999), (2048, 64, 4097)])
def test_shares_of_a_sum_go_by_its_depth(rows, D, ffn):
    """In 16 bits the gradient of x is one sum over both halves, padded to multiples of 8: as many shares of it, and so as much memory, as at that width."""
    from pfeife_amd import hip

    lib = hip.load()
    need = lambda columns: lib.pf_gated_linear_workspace(None, None, 2, rows, D, columns, 1, 1)  # noqa: E731
    assert need(ffn) == need(-(-ffn // 8) * 8) > 0
