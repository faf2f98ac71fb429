"""Forward-mode derivatives of the token losses: there are none, and who asks for one is told so (on the CPU; nothing is launched)."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

X, Y = torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.int64)


@pytest.fixture()
def loss(monkeypatch):
    """The kernels' table and the launches stand aside: what reaches the formulas' forward pass returns its empty results."""
    from pfeife_amd import loss

    class Kernels:
        def preference_workspace(self, *_):
            return 8

        policy_workspace = preference_workspace

        def __getattr__(self, name):
            return lambda *args: None

    monkeypatch.setattr(loss, "_table", lambda t, who: Kernels())
    monkeypatch.setattr(loss, "_rows", lambda *_: ())
    monkeypatch.setattr(loss, "_issue", lambda *_: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return loss


CALLS = {
    "token_logprobs": lambda m, x, o: m.token_logprobs(x, Y),
    "preference_loss": lambda m, x, o: m.preference_loss(x, Y, o[:, 0])[0],
    "policy_loss": lambda m, x, o: m.policy_loss(x, Y, o, torch.zeros(2))[0],
}


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", CALLS)
def test_a_tangent_of_the_logits_is_refused(loss, name, grad):
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        CALLS[name](loss, X, torch.zeros(2, 3))      # (nothing to lose)
        for x in (X, X.clone().requires_grad_()):
            dual = fwd.make_dual(x, torch.ones_like(X))
            with pytest.raises(RuntimeError, match="%s: .*forward-mode" % name):
                CALLS[name](loss, dual, torch.zeros(2, 3))
            with pytest.raises(RuntimeError, match="%s: .*forward-mode" % name):
                CALLS[name](loss, dual[:, :, 0:5:1] * 2.0, torch.zeros(2, 3))


@pytest.mark.parametrize("name", ["preference_loss", "policy_loss"])
def test_a_tangent_of_an_operand_is_refused(loss, name):
    """As one that requires a gradient is: none flows to it."""
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="%s: .*detach" % name):
            CALLS[name](loss, X, fwd.make_dual(torch.zeros(2, 3), torch.ones(2, 3)))


def test_a_tangent_of_what_comes_back_is_refused(loss, monkeypatch):
    """A gradient is linear in what the backward pass is given: a tangent of that has one too, which the kernels do not form."""
    monkeypatch.setattr(loss, "_logits_gradient", lambda ctx, logits, *_: torch.zeros_like(logits))
    x = X.clone().requires_grad_()
    for name, call in CALLS.items():
        out = call(loss, x, torch.zeros(2, 3))
        (d,) = torch.autograd.grad(out, x, torch.ones_like(out), retain_graph=True)
        assert d.shape == x.shape
        with fwd.dual_level():
            (d,) = torch.autograd.grad(out, x, torch.ones_like(out), retain_graph=True)
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, x, fwd.make_dual(torch.ones_like(out), torch.ones_like(out)))
