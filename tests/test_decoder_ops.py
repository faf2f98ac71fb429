"""Arguments that linear_cross_entropy, embedding and gated_linear refuse, without a GPU."""
import pytest
import torch


@pytest.fixture()
def on_any_device(monkeypatch):
    """Argument checks alone: tensors of the CPU pass for the GPU's, and nothing is launched."""
    from pfeife_amd import layers, loss

    monkeypatch.setattr(loss, "_table", lambda t, who: None)
    monkeypatch.setattr(layers, "_table", lambda t, who: None)
    return {"linear_cross_entropy": loss.linear_cross_entropy, "embedding": layers.embedding, "gated_linear": layers.gated_linear}


H, W, Y = torch.zeros(2, 3, 8), torch.zeros(5, 8), torch.zeros(2, 3, dtype=torch.int64)


def test_cpu_tensors_are_refused():
    from pfeife_amd.layers import embedding, gated_linear
    from pfeife_amd.loss import linear_cross_entropy

    for call in (lambda: linear_cross_entropy(H, W, Y), lambda: embedding(Y, W), lambda: gated_linear(H, torch.zeros(6, 8))):
        with pytest.raises(RuntimeError, match="GPU tensors"):
            call()


REFUSED = [
    ("linear_cross_entropy", (H, W, None), {}, "tensors"), ("linear_cross_entropy", (H.double(), W.double(), Y), {}, "fp32, fp16 or bf16"),
    ("linear_cross_entropy", (H.half(), W, Y), {}, "both"), ("linear_cross_entropy", (H[0, 0], W, Y[0, 0]), {}, "tokens, width"),
    ("linear_cross_entropy", (H[..., :0], W[:, :0], Y), {}, "tokens, width"), ("linear_cross_entropy", (H, W[:, :7], Y), {}, "weight is"),
    ("linear_cross_entropy", (H, W[:0], Y), {}, "weight is"), ("linear_cross_entropy", (H, W[0], Y), {}, "weight is"),
    ("linear_cross_entropy", (H, W, Y.int()), {}, "int64"), ("linear_cross_entropy", (H, W, Y[:, :2]), {}, "int64"),
    ("linear_cross_entropy", (H, W, Y), {"ignore_index": 0.5}, "ignore_index"), ("linear_cross_entropy", (H, W, Y), {"shift": 2}, "shift"),
    ("linear_cross_entropy", (H, W, Y), {"reduction": "max"}, "reduction"), ("linear_cross_entropy", (H, W, Y), {"z_loss": float("nan")}, "z_loss"),
    ("embedding", (Y, None), {}, "tensors"), ("embedding", (Y, W.double()), {}, "fp32, fp16 or bf16"), ("embedding", (Y, W[0]), {}, "rows, width"),
    ("embedding", (Y, W[:0]), {}, "rows, width"), ("embedding", (Y.int(), W), {}, "int64"), ("embedding", (Y, W), {"scale": float("inf")}, "scale"),
    ("embedding", (Y, W), {"scale": None}, "scale"), ("embedding", (Y, W), {"padding_idx": 5}, "padding_idx"), ("embedding", (Y, W), {"padding_idx": -6}, "padding_idx"),
    ("embedding", (Y, W), {"padding_idx": 1.0}, "padding_idx"),
    ("gated_linear", (H, None), {}, "tensors"), ("gated_linear", (H.double(), torch.zeros(6, 8).double()), {}, "fp32, fp16 or bf16"),
    ("gated_linear", (H, torch.zeros(6, 8).half()), {}, "both"), ("gated_linear", (H, torch.zeros(5, 8)), {}, "weight is"), ("gated_linear", (H, torch.zeros(6, 7)), {}, "weight is"),
    ("gated_linear", (H, torch.zeros(0, 8)), {}, "weight is"), ("gated_linear", (H[..., :0], torch.zeros(6, 0)), {}, "width"),
    ("gated_linear", (H, torch.zeros(6, 8)), {"act": "tanh"}, "act is"), ("gated_linear", (H, torch.zeros(6, 8)), {"kept": "4bit"}, "kept is"),
    ("gated_linear", (H, torch.zeros(6, 8)), {"kept": "8bit"}, "kept is"),
]


@pytest.mark.parametrize("name,args,kwargs,says", REFUSED)
def test_refused(on_any_device, name, args, kwargs, says):
    with pytest.raises(RuntimeError, match="%s: .*%s" % (name, says)):
        on_any_device[name](*args, **kwargs)


def test_forward_mode_is_refused(on_any_device):
    import torch.autograd.forward_ad as ad

    with ad.dual_level():
        dual = ad.make_dual(H, torch.ones_like(H))
        for call in (lambda: on_any_device["linear_cross_entropy"](dual, W, Y), lambda: on_any_device["gated_linear"](dual, torch.zeros(6, 8)),
                     lambda: on_any_device["embedding"](Y, ad.make_dual(W, torch.ones_like(W)))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_the_c_entries_refuse_without_a_device():
    from pfeife_amd import hip

    lib = hip.load()
    one = 1 << 20      # (an address that nothing reads)

    def rc(call, says):
        assert call == -1 and says in lib.pf_last_error(), (call, lib.pf_last_error())

    head = dict(h=one, dt=2, B=2, T=3, D=64, sb=192, st=64, w=one, V=100)
    fwd = lambda **k: lib.pf_linear_ce_fwd(*{**head, **dict(y=one, shift=0, ig=-100, z=0.0, red=1, loss=one, kept=one, ws=one, s=None), **k}.values())  # noqa: E731
    rc(fwd(dt=3), b"bad dtype")
    rc(fwd(V=0), b"bad sizes")
    rc(fwd(D=0), b"bad sizes")
    rc(fwd(B=-1), b"bad sizes")
    rc(fwd(shift=2), b"shift")
    rc(fwd(red=3), b"reduction")
    for name in ("h", "w", "y", "loss", "kept", "ws"):
        rc(fwd(**{name: None}), b"null pointer")
    rc(fwd(B=1 << 12, T=1 << 12), b"too many")
    rc(fwd(B=1, T=1 << 20, D=4096, sb=0, st=0), b"too many")
    bwd = lambda **k: lib.pf_linear_ce_bwd(*{**head, **dict(z=0.0, mean=1, kept=one, g=one, gb=0, gt=0, dh=one, dw=one, ws=one, s=None), **k}.values())  # noqa: E731
    for name in ("h", "w", "kept", "g", "ws"):
        rc(bwd(**{name: None}), b"null pointer")
    rc(bwd(dw=one + 2), b"16 bytes")
    assert lib.pf_linear_ce_workspace(None, 2, -1, 64, 100, 0) == -1 and lib.pf_linear_ce_workspace(None, 7, 1, 64, 100, 0) == -1
    assert lib.pf_linear_ce_workspace(None, 2, 100, 64, 1000, 1) > 0 and lib.pf_linear_ce_kept(1) == 64 + 20 * 64
    rc(lib.pf_linear_ce_hidden_grad(one, 2, 5, 64, 100, None, None, one, one, None), b"null pointer")
    assert lib.pf_linear_ce_hidden_grad(one, 2, 0, 64, 100, None, None, None, None, None) == 0

    gated = lambda **k: lib.pf_gated_linear_fwd(*{**dict(x=one, dt=2, rows=3, D=64, w=one, ffn=32, act=3, keep=1, y=one, kept=one, ws=one, s=None), **k}.values())  # noqa: E731
    rc(gated(dt=3), b"bad dtype")
    rc(gated(rows=-1), b"bad sizes")
    rc(gated(ffn=0), b"bad sizes")
    rc(gated(act=0), b"bad activation")
    rc(gated(act=5), b"bad activation")
    rc(gated(keep=3), b"8 bits")
    rc(gated(dt=0, keep=2), b"8 bits")
    for name in ("x", "w", "y", "kept"):
        rc(gated(**{name: None}), b"null pointer")
    rc(gated(D=1000, ffn=1 << 21), b"too large")
    rc(gated(rows=1 << 20, ffn=4096), b"too large")
    assert gated(rows=0, x=None, w=None, y=None, kept=None) == 0
    back = lambda **k: lib.pf_gated_linear_bwd(*{**dict(x=one, dt=2, rows=3, D=64, w=one, ffn=32, act=3, keep=1, kept=one, dy=one, dx=one, dw=one, ws=one, s=None), **k}.values())  # noqa: E731
    rc(back(keep=0), b"nothing was kept")
    for name in ("x", "w", "kept", "dy", "ws"):
        rc(back(**{name: None}), b"null pointer")
    rc(back(dx=one + 2), b"16 bytes")
    assert lib.pf_gated_linear_kept(2, 10, 20, 2) == 10 * 64 + 12 * 4 and lib.pf_gated_linear_kept(0, 10, 20, 2) == -1 and lib.pf_gated_linear_kept(2, 10, 20, 0) == 0
    assert lib.pf_gated_linear_workspace(None, None, 2, 10, 64, 0, 1, 0) == -1

    look = lambda **k: lib.pf_embedding_scaled_fwd(*{**dict(t=one, dt=2, ids=one, out=one, n=3, dim=8, V=5, scale=1.0, s=None), **k}.values())  # noqa: E731
    rc(look(dt=3), b"bad arguments")
    rc(look(n=-1), b"bad arguments")
    rc(look(dim=0), b"bad arguments")
    rc(look(n=1 << 31), b"too many")
    for name in ("t", "ids", "out"):
        rc(look(**{name: None}), b"null pointer")
    assert look(n=0, t=None, ids=None, out=None) == 0
    grad = lambda **k: lib.pf_embedding_sorted_bwd(*{**dict(d=one, dt=2, ids=one, out=one, td=2, n=300, dim=8, V=5, pad=-1, scale=1.0, acc=0, ws=one, s=None), **k}.values())  # noqa: E731
    rc(grad(td=1), b"bad arguments")
    rc(grad(V=0), b"bad arguments")
    rc(grad(pad=5), b"padding_idx")
    rc(grad(pad=-2), b"padding_idx")
    rc(grad(n=1 << 28), b"too many")
    for name in ("d", "ids", "out", "ws"):
        rc(grad(**{name: None}), b"null pointer")
    assert lib.pf_embedding_sorted_workspace(0, 8) == 0 and lib.pf_embedding_sorted_workspace(300, 8) > 0


def test_the_c_entries_refuse_memory_that_their_wide_accesses_cannot_take():
    from pfeife_amd import hip

    lib = hip.load()
    one = 1 << 20      # (an address that nothing reads)

    def rc(call, says):
        assert call == -1 and says in lib.pf_last_error(), (call, lib.pf_last_error())

    for kept, ws in ((one + 4, one), (one, one + 4)):
        rc(lib.pf_linear_ce_fwd(one, 2, 2, 3, 64, 192, 64, one, 100, one, 0, -100, 0.0, 1, one, kept, ws, None), b"boundaries")
        rc(lib.pf_linear_ce_bwd(one, 2, 2, 3, 64, 192, 64, one, 100, 0.0, 1, kept, one, 0, 0, one, one, ws, None), b"boundaries")
        rc(lib.pf_linear_ce_hidden_grad(one, 2, 6, 64, 100, kept, None, one, ws, None), b"boundaries")
        rc(lib.pf_gated_linear_fwd(one, 2, 3, 64, one, 32, 3, 1, one, kept, ws, None), b"boundaries")
        rc(lib.pf_gated_linear_bwd(one, 2, 3, 64, one, 32, 3, 1, kept, one, one, one, ws, None), b"boundaries")
    rc(lib.pf_embedding_sorted_bwd(one, 2, one, one, 2, 300, 8, 5, -1, 1.0, 0, one + 4, None), b"boundary")
    rc(lib.pf_embedding_sorted_bwd(one, 2, one, one, 2, 300, 65535 * 64 + 1, 5, -1, 1.0, 0, one, None), b"too many")


def test_an_embedding_without_a_possible_gradient_is_refused_before_it_runs(on_any_device):
    many = torch.zeros(1, dtype=torch.int64).expand((1 << 27) + 1)
    with pytest.raises(RuntimeError, match="too many ids"):
        on_any_device["embedding"](many, W.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="too many ids"):
        on_any_device["embedding"](Y, torch.zeros(1).expand(2, 65535 * 64 + 1).requires_grad_())
