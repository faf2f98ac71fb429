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


def test_recorded_graphs_run():
    """A graph recorded of the layers gives what the calls give, on other values too."""
    from torch.fx.experimental.proxy_tensor import make_fx

    from pfeife_amd.layers import embedding, gated_linear

    g = torch.Generator("cuda").manual_seed(6)
    draw = lambda: (torch.randint(0, 50, (2, 9), device="cuda", generator=g), torch.randn(50, 24, device="cuda", generator=g), torch.randn(34, 24, device="cuda", generator=g))  # noqa: E731
    both = lambda ids, table, up: gated_linear(embedding(ids, table, scale=0.5), up)  # noqa: E731
    first = draw()
    graphs = [make_fx(both)(*first), torch.jit.trace(both, first)]
    for args in (first, draw()):
        want = both(*args)
        assert all(torch.equal(graph(*args), want) for graph in graphs)


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_a_loss_in_a_compiled_function(backend):
    """The compiler leaves the loss out of its graphs; values and gradients are those of the plain call."""
    from pfeife_amd.loss import linear_cross_entropy

    torch._dynamo.reset()
    g = torch.Generator("cuda").manual_seed(8)
    h = torch.randn(2, 20, 64, device="cuda", generator=g).requires_grad_()
    w = torch.randn(90, 64, device="cuda", generator=g).requires_grad_()
    y = torch.randint(0, 90, (2, 20), device="cuda", generator=g)
    step = lambda h, w: linear_cross_entropy(h * 0.5, w, y, shift=True, z_loss=1e-3) * 2.0  # noqa: E731
    want, got = step(h, w), torch.compile(step, backend=backend)(h, w)
    assert torch.equal(got, want)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, (h, w)), torch.autograd.grad(want, (h, w))))


# rows of 1 GiB, whose gradient in fp32 no call could hold; more workgroups than one launch has
@pytest.mark.parametrize("tokens,D,V", [(131072, 4096, 300), (1 << 22, 64, 66000)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_scores_of_a_long_batch(dtype, tokens, D, V):
    """A forward pass alone, tokens scored at its ends and here and there."""
    from test_decoder_ops_gpu import IGNORE, head_reference, within

    from pfeife_amd.loss import linear_cross_entropy

    g = torch.Generator("cuda").manual_seed(9)
    w = (torch.randn(V, D, device="cuda", generator=g) * D ** -0.5).to(dtype)
    h = torch.empty(1, tokens, D, device="cuda", dtype=dtype)
    for part in h.split(1 << 16, dim=1):
        part.copy_(torch.randn(part.shape, device="cuda", generator=g))
    at = torch.cat([torch.tensor([0, 1, tokens - 2, tokens - 1], device="cuda"), torch.randint(2, tokens - 2, (600,), device="cuda", generator=g)]).unique()
    y = torch.full((1, tokens), IGNORE, device="cuda")
    y[0, at] = torch.randint(0, V, at.shape, device="cuda", generator=g)
    loss = linear_cross_entropy(h, w, y, reduction="none")
    every = linear_cross_entropy(h, w, torch.where(y == IGNORE, 7, y), reduction="none")
    assert torch.isfinite(every).all() and torch.equal(every[0, at], loss[0, at])      # (what is scored beside a token changes nothing of it)
    rest = loss.clone()
    rest[0, at] = 0
    assert not rest.any()
    term, bound = head_reference(h[:, at], w, y[:, at], 0, "none", 0.0, torch.ones((), device="cuda"))[:2]
    within(loss[:, at], term, bound, torch.float32)


@pytest.mark.parametrize("sequences", [8, 400])
def test_a_table_that_is_computed_in_a_runner(sequences):
    """Four micro-batches, ids sorted and not: the table's gradient reaches its parameter through what it is computed from, three ways."""
    from test_decoder_compiled import Computed
    from test_pipeline_gpu import _fresh_runner

    from pfeife_amd.mp import partial_compiler
    from pfeife_amd.option import PipeOption

    model, plain = Computed(False).cuda(), Computed(True).cuda()
    g = torch.Generator("cuda").manual_seed(3)
    ids = torch.randint(0, 11, (sequences, 5), device="cuda", generator=g)
    weight = torch.linspace(-1, 1, 16, device="cuda")
    runner = _fresh_runner(PipeOption(device_cnt=1, batch_cnt=4, batch_size=sequences // 4, optimizer=dict(type="sgd", lr=0.0)))
    compiled = torch.compile(model, backend=partial_compiler)

    def fn(ids):
        loss = (compiled(ids).float() * weight).sum()
        loss.backward()
        return loss.detach()

    runner.set_exec_fn(fn)
    for _ in range(3):
        model.table.grad = plain.table.grad = None
        losses = runner.step(ids)
        torch.cuda.synchronize()
        want = (plain(ids).float() * weight).sum()
        want.backward()
        # (sums of some thousand terms in fp32, of which the bf16 table's lookup rounds its gradient to 8 bits)
        assert abs(sum(float(v) for v in losses) - float(want.detach())) <= 1e-3 * float((plain(ids).float() * weight).abs().sum().detach())
        assert (model.table.grad - plain.table.grad).norm() <= 3 * 2.0 ** -8 * plain.table.grad.norm()
        assert not model.table.grad[3].any()


@pytest.mark.parametrize("rows,D,ffn", [(1024, 256, 5630), (2048, 64, 4097), (1024, 1030, 5630)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gated_linear_in_shares_of_an_odd_depth(dtype, rows, D, ffn):
    from test_decoder_ops_gpu import gated_check

    from pfeife_amd.layers import gated_linear

    g = torch.Generator("cuda").manual_seed(12)
    x = torch.randn(rows, D, device="cuda", generator=g).to(dtype).requires_grad_()
    w = (torch.randn(2 * ffn, D, device="cuda", generator=g) * D ** -0.5).to(dtype).requires_grad_()
    up = torch.randn(rows, ffn, device="cuda", generator=g).to(dtype)
    y = gated_linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), up)
    gated_check(x.detach(), w.detach(), "silu", "16bit", up, y.detach(), dx, dw)
