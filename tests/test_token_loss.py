"""Arguments that the token losses and AdamW8bit refuse, without a GPU."""
import ctypes

import pytest
import torch


@pytest.fixture()
def on_any_device(monkeypatch):
    """Argument checks alone: tensors of the CPU pass for the GPU's, and nothing is launched."""
    from pfeife_amd import loss

    monkeypatch.setattr(loss, "_table", lambda t, who: None)
    return loss


def test_cpu_tensors_are_refused():
    from pfeife_amd.loss import PolicyLoss, PreferenceLoss, policy_loss, preference_loss, token_logprobs

    x, y, one = torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2)
    for call in (lambda: token_logprobs(x, y), lambda: preference_loss(x, y, one), lambda: policy_loss(x, y, torch.zeros(2, 3), one),
                 lambda: PreferenceLoss(beta=0.2)(x, (y, one)), lambda: PolicyLoss(clip=0.1)(x, (y, torch.zeros(2, 3), one))):
        with pytest.raises(RuntimeError, match="GPU tensors"):
            call()


X, Y = torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.int64)
REFUSED = [
    ("token_logprobs", (X.double(), Y), {}, "fp32, fp16 or bf16"), ("token_logprobs", (X, Y.int()), {}, "int64"), ("token_logprobs", (X, Y[:, :2]), {}, "int64"),
    ("token_logprobs", (X[0, 0], Y[0, 0]), {}, "tokens, classes"), ("token_logprobs", (X[..., :0], Y), {}, "tokens, classes"), ("token_logprobs", (X, None), {}, "tensors"),
    ("token_logprobs", (X, Y), {"temperature": 0.0}, "temperature"), ("token_logprobs", (X, Y), {"temperature": float("nan")}, "temperature"),
    ("token_logprobs", (X, Y), {"shift": 2}, "shift"), ("token_logprobs", (X, Y), {"ignore_index": 0.5}, "ignore_index"),
    ("preference_loss", (X[:1], Y[:1], torch.zeros(1)), {}, "2 \\* pairs"), ("preference_loss", (X[0], Y[0], torch.zeros(2)), {}, "2 \\* pairs"),
    ("preference_loss", (X[:0], Y[:0], torch.zeros(0)), {}, "2 \\* pairs"),
    ("preference_loss", (X, Y, torch.zeros(1)), {}, "ref_logprobs"), ("preference_loss", (X, Y, torch.zeros(2, dtype=torch.int64)), {}, "ref_logprobs"),
    ("preference_loss", (X, Y, torch.zeros(2, requires_grad=True)), {}, "no gradient"), ("preference_loss", (X, Y, torch.zeros(2)), {"beta": float("inf")}, "beta"),
    ("preference_loss", (X, Y, torch.zeros(2)), {"label_smoothing": 1.5}, "label_smoothing"),
    ("policy_loss", (X[0], Y[0], torch.zeros(3), torch.zeros(1)), {}, "sequences, tokens"), ("policy_loss", (X, Y, torch.zeros(2, 2), torch.zeros(2)), {}, "old_logprobs"),
    ("policy_loss", (X, Y, torch.zeros(2, 3), torch.zeros(2)), {"shift": True}, "old_logprobs"),
    ("policy_loss", (X, Y, torch.zeros(2, 3), torch.zeros(3)), {}, "advantages"), ("policy_loss", (X, Y, torch.zeros(2, 3), 1.0), {}, "advantages"),
    ("policy_loss", (X, Y, torch.zeros(2, 3), torch.zeros(2)), {"kl_coef": 0.1}, "ref_logprobs"),
    ("policy_loss", (X, Y, torch.zeros(2, 3), torch.zeros(2), torch.zeros(2, 4)), {}, "ref_logprobs"),
    ("policy_loss", (X, Y, torch.zeros(2, 3), torch.zeros(2)), {"clip": -0.1}, "clip"), ("policy_loss", (X, Y, torch.zeros(2, 3), torch.zeros(2)), {"clip_high": float("nan")}, "clip"),
    ("policy_loss", (X, Y, torch.zeros(2, 3), torch.zeros(2)), {"reduction": "sum"}, "reduction"),
    ("policy_loss", (X, Y, torch.zeros(2, 3), torch.zeros(2)), {"scale": float("inf")}, "finite"),
    ("policy_loss", (X, Y, torch.zeros(2, 3, requires_grad=True), torch.zeros(2)), {}, "no gradient"),
]


@pytest.mark.parametrize("name,args,kwargs,says", REFUSED)
def test_refused(on_any_device, name, args, kwargs, says):
    with pytest.raises(RuntimeError, match="%s: .*%s" % (name, says)):
        getattr(on_any_device, name)(*args, **kwargs)


def test_the_c_entries_refuse_without_a_device():
    from pfeife_amd import hip

    lib = hip.load()
    one, bad = 1 << 20, b""      # (an address that nothing reads)

    def rc(call, says):
        assert call == -1 and says in lib.pf_last_error(), lib.pf_last_error()

    fwd = lambda **k: lib.pf_token_logprob_fwd(*{**dict(x=one, dt=0, B=2, T=3, V=5, sb=15, st=5, y=one, shift=0, ig=-100, t=1.0, out=one, stats=None, s=None), **k}.values())  # noqa: E731
    rc(fwd(dt=3), b"fp32, fp16 or bf16")
    rc(fwd(V=0), b"bad sizes")
    rc(fwd(T=-1), b"bad sizes")
    rc(fwd(st=-5), b"bad sizes")
    rc(fwd(shift=2), b"shift")
    rc(fwd(t=0.0), b"temperature")
    rc(fwd(t=float("nan")), b"temperature")
    rc(fwd(x=None), b"null pointer")
    rc(fwd(y=None), b"null pointer")
    rc(fwd(out=None), b"null pointer")
    assert fwd(B=0, x=None, y=None, out=None) == 0 and fwd(T=1, shift=1) == 0
    bwd = lambda **k: lib.pf_token_logprob_bwd(*{**dict(x=one, dt=0, B=2, T=3, V=5, sb=15, st=5, y=one, shift=0, ig=-100, t=1.0, stats=one, g=one, gb=3, gt=1,  # noqa: E731
                                                        scale=None, unless=0, d=one, db=15, ds=5, s=None), **k}.values())
    rc(bwd(unless=1), b"unless_one")
    rc(bwd(d=None), b"null pointer")
    rc(bwd(stats=None), b"null pointer")
    rc(bwd(gb=-1), b"bad strides")
    assert bwd(B=0) == 0
    pref = lambda **k: lib.pf_preference_loss(*{**dict(x=one, dt=0, B=2, T=3, V=5, sb=15, st=5, y=one, shift=0, ig=-100, ref=one, beta=0.1, e=0.0, avg=0, loss=one,  # noqa: E731
                                                       r=one, stats=None, c=one, ws=one, s=None), **k}.values())
    rc(pref(B=3), b"pairs")
    rc(pref(B=0), b"pairs")
    rc(pref(e=2.0), b"label_smoothing")
    rc(pref(ws=None), b"null pointer")
    rc(pref(x=None), b"null pointer")
    rc(pref(dt=4), b"fp32, fp16 or bf16")
    assert lib.pf_preference_workspace(4, 10, 1) == 2 + 4 * 9
    pol = lambda **k: lib.pf_policy_loss(*{**dict(x=one, dt=0, B=2, T=3, V=5, sb=15, st=5, y=one, shift=0, ig=-100, t=1.0, old=one, adv=one, asb=1, ast=0, ref=None, lo=0.2, hi=0.2,  # noqa: E731
                                                  c=0.0, seq=0, scale=1.0, loss=one, kl=one, lp=one, stats=None, coef=None, d=None, db=0, ds=0, ws=one, s=None), **k}.values())
    rc(pol(lo=-1.0), b"clip")
    rc(pol(ws=None), b"workspace")
    rc(pol(old=None), b"null pointer")
    rc(pol(stats=one), b"go together")
    rc(pol(loss=None), b"null pointer")
    assert lib.pf_policy_workspace(4, 10, 1) == 4 + 2 * 4 * 9 and lib.pf_policy_workspace(4, 0, 1) == 4
    rc(lib.pf_adam8_step(None, None, 1, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None, None), b"item list")
    rc(lib.pf_adam8_step(one, one, 1, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0, None, None), b"bad arguments")
    rc(lib.pf_adam8_step(one, one, -1, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None, None), b"bad arguments")
    assert lib.pf_adam8_step(None, None, 0, 0, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None, None) == 0
