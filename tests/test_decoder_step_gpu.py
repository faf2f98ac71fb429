"""The decoder operators together, as a training program has them: the table's lookup, gated projections, the loss from the last hidden state;
in a runner's stages, eagerly, captured into a graph, on other streams."""
import pytest
import torch
import torch.nn.functional as F

from test_decoder_graph import Decoder, plain_of
from test_pipeline_gpu import _fresh_runner

pytestmark = pytest.mark.gpu

VOCAB, DIM, FFN, SEQ = 509, 64, 96, 40


def batch(sequences, seed=11):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, VOCAB, (sequences, SEQ), generator=g).cuda()
    labels = ids.clone()
    labels[:, :7] = -100
    for b in range(sequences):
        labels[b, SEQ - 3 * b:] = -100
    return ids, labels


@pytest.mark.parametrize("mixed,kept", [(None, "16bit"), ("bf16", "16bit"), ("bf16", "8bit"), ("fp16", "8bit")])
def test_a_training_step_in_a_runner(mixed, kept):
    """Two stages, four micro-batches, the head beside the stages: losses and gradients of two steps against plain PyTorch."""
    from pfeife_amd.loss import linear_cross_entropy
    from pfeife_amd.mp import partial_compiler
    from pfeife_amd.option import PipeOption

    torch.manual_seed(3)
    model = Decoder(vocab=VOCAB, dim=DIM, ffn=FFN, depth=4, kept=kept, padding=5).cuda()
    head = torch.nn.Parameter(torch.randn(VOCAB, DIM, device="cuda") * DIM ** -0.5)
    ref, ref_head = plain_of(model), head.detach().clone().requires_grad_()
    ids, labels = batch(8)
    dtype = {"fp16": torch.float16, "bf16": torch.bfloat16}.get(mixed, torch.float32)
    runner = _fresh_runner(PipeOption(device_cnt=2, batch_cnt=4, batch_size=2, split_points=["blocks.2"], mixed_precision=mixed, init_scale=1024.0,
                                      optimizer=dict(type="sgd", lr=0.05)))
    compiled = torch.compile(model, backend=partial_compiler)

    def fn(ids, labels):
        loss = linear_cross_entropy(compiled(ids).to(dtype), head.to(dtype), labels, shift=True)
        loss.backward()
        return loss.detach()

    runner.set_exec_fn(fn)
    for step in range(2):
        for p in (head, ref_head, *ref.parameters()):
            p.grad = None
        ref.load_state_dict(model.state_dict())
        losses = runner.step(ids, labels)
        torch.cuda.synchronize()
        for k in range(4):
            s = slice(2 * k, 2 * k + 2)
            with torch.autocast("cuda", dtype=dtype, enabled=mixed is not None):
                logits = F.linear(ref(ids[s]), ref_head)
            want = F.cross_entropy(logits[:, :-1].reshape(-1, VOCAB).float(), labels[s][:, 1:].reshape(-1), ignore_index=-100)
            want.backward()
            assert abs(float(losses[k]) - float(want.detach())) <= (2e-5 if mixed is None else 2e-2) * float(want.detach()), (step, k)
        pairs = [("head", head, ref_head)] + [(n, p, q) for (n, p), (_, q) in zip(model.named_parameters(), ref.named_parameters())]
        for n, p, q in pairs:
            a, b = p.grad.double(), q.grad.double()
            # (fp32: sums in another order through four blocks; 16 bits: every product rounded once, the loss's logits not at all; 8 bits hold four
            # binary digits of the pre-activations)
            assert (a - b).norm() <= (1e-4 if mixed is None else 3e-2 if kept == "16bit" else 6e-2) * b.norm() + 1e-9, (step, n, float((a - b).norm() / b.norm()))
        assert not model.table.grad[5].any()


def weights(dtype, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    return [(rnd(VOCAB, DIM) * 0.5).to(dtype), (rnd(2 * FFN, DIM) * DIM ** -0.5).to(dtype), (rnd(DIM, FFN) * FFN ** -0.5).to(dtype), (rnd(VOCAB, DIM) * DIM ** -0.5).to(dtype)]


def decoder_loss(ws, ids, labels, kept):
    from pfeife_amd.layers import embedding, gated_linear
    from pfeife_amd.loss import linear_cross_entropy

    table, up, down, head = ws
    x = embedding(ids, table, scale=2.0, padding_idx=-1)
    x = x + F.linear(gated_linear(x, up, kept=kept), down)
    return linear_cross_entropy(x, head, labels, shift=True, z_loss=1e-3)


def eager(ws, ids, labels, kept):
    leaves = [w.detach().requires_grad_() for w in ws]
    loss = decoder_loss(leaves, ids, labels, kept)
    return [loss.detach()] + list(torch.autograd.grad(loss, leaves))


@pytest.mark.parametrize("dtype,kept", [(torch.float32, "16bit"), (torch.bfloat16, "16bit"), (torch.bfloat16, "8bit"), (torch.float16, "8bit")])
def test_captured_and_replayed(dtype, kept):
    """A whole forward and backward pass in a graph, replayed on other inputs with eager work between: the eager bits each time.  (The number
    of tokens that take part changes from replay to replay, none among them.)"""
    ws = weights(dtype)
    ids, labels = batch(6)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        eager(ws, ids, labels, kept)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph, still, seen = torch.cuda.CUDAGraph(), ids.clone(), labels.clone()
    held = [w.clone() for w in ws]
    with torch.cuda.graph(graph):
        out = eager(held, still, seen, kept)
    for k in range(4):
        new_ids, new_labels = batch(6, seed=20 + k)
        if k == 2:
            new_labels[:] = -100
        new = weights(dtype, seed=k)
        still.copy_(new_ids)
        seen.copy_(new_labels)
        for a, b in zip(held, new):
            a.copy_(b)
        graph.replay()
        want = eager(new, new_ids, new_labels, kept)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), k


def test_two_graphs_and_an_eager_call_keep_apart():
    """Two captured passes and an eager one between them: each has workspaces of its own."""
    sets = [(weights(torch.bfloat16, seed=s), *batch(4 + 2 * s, seed=s)) for s in range(2)]
    wants = [eager(ws, ids, labels, "8bit") for ws, ids, labels in sets]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for ws, ids, labels in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(eager(ws, ids, labels, "8bit"))
        graphs.append(graph)
    for order in ((0, 1), (1, 0), (1, 1)):
        for k in order:
            graphs[k].replay()
            again = eager(*sets[1 - k], "8bit")
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs[k], wants[k])) and all(torch.equal(a, b) for a, b in zip(again, wants[1 - k]))


def test_on_another_stream():
    ws = weights(torch.bfloat16)
    ids, labels = batch(6)
    want = eager(ws, ids, labels, "8bit")
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(eager(ws, ids, labels, "8bit"))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_two_losses_before_their_backward_passes():
    """What a forward pass leaves is its own: two losses of one hidden state, the later one's gradient first."""
    from pfeife_amd.loss import linear_cross_entropy

    ws = weights(torch.bfloat16)
    g = torch.Generator("cuda").manual_seed(1)
    h = torch.randn(3, SEQ, DIM, device="cuda", generator=g).bfloat16().requires_grad_()
    _, a = batch(3, seed=1)
    _, b = batch(3, seed=2)
    head = ws[3].clone().requires_grad_()
    one = [torch.autograd.grad(linear_cross_entropy(h, head, y, shift=True), (h, head)) for y in (a, b)]
    first, second = linear_cross_entropy(h, head, a, shift=True), linear_cross_entropy(h, head, b, shift=True)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(second, (h, head)), one[1]))
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(first, (h, head)), one[0]))


def test_saved_tensors_moved_by_hooks():
    """Saved tensors that hooks take to the host and bring back elsewhere give the same gradients."""
    ws = weights(torch.bfloat16)
    ids, labels = batch(4)
    want = eager(ws, ids, labels, "8bit")
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (t.cpu(), t.device), lambda p: p[0].to(p[1])):
        got = eager(ws, ids, labels, "8bit")
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_the_hidden_states_gradient_times_a_loss_scale():
    """Where a runner will scale it, an fp16 gradient is formed with the scale before it is rounded: entries that fp16 does not hold without it."""
    from pfeife_amd.loss import linear_cross_entropy, mark_loss_scaled, scaled_gradient

    g = torch.Generator("cuda").manual_seed(2)
    h = (torch.randn(2, 30, DIM, device="cuda", generator=g) * 1.0).half().requires_grad_()
    w = (torch.randn(VOCAB, DIM, device="cuda", generator=g) * DIM ** -0.5).half()
    y = torch.randint(0, VOCAB, (2, 30), device="cuda", generator=g)
    mark_loss_scaled(h)
    loss = linear_cross_entropy(h, w, y) * 2.0 ** -12
    seen = []
    h.register_hook(lambda grad: seen.append(grad))
    loss.backward()
    scale, out = torch.tensor([2.0 ** 16], device="cuda"), torch.empty_like(h)
    assert scaled_gradient(seen[0], scale, out)
    h64 = h.detach().double().requires_grad_()
    want, = torch.autograd.grad(F.cross_entropy((h64 @ w.double().t()).view(-1, VOCAB), y.view(-1)) * 2.0 ** 4, h64)
    # dz off by a rounding of fp16 (its largest is 2^13 of their own scale), the sum's rounding, and the result's
    assert (out.double() - want).norm() <= 2 * 2.0 ** -11 * want.norm()
    assert (seen[0].double() * 2.0 ** 16 - want).norm() > 8 * 2.0 ** -11 * want.norm()      # (what multiplying the rounded one would have given)


def test_in_a_model_that_is_compiled_without_a_runner():
    """The graph's nodes run by themselves too, with their gradients."""
    torch._dynamo.reset()
    torch.manual_seed(0)
    model = Decoder(vocab=VOCAB, dim=DIM, ffn=FFN, depth=2).cuda()
    ids, _ = batch(2)
    want = model(ids)
    grads = torch.autograd.grad(want.square().sum() + want.sum(), list(model.parameters()))
    compiled = torch.compile(model, backend="eager", fullgraph=True)
    got = compiled(ids)
    again = torch.autograd.grad(got.square().sum() + got.sum(), list(model.parameters()))
    assert torch.equal(got, want)
    assert all(torch.allclose(a, b, rtol=1e-4, atol=1e-5 * float(b.abs().max())) for a, b in zip(again, grads))      # (sums over micro-tiles may start from another place)
