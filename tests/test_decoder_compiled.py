"""`layers.embedding` and `layers.gated_linear` in graphs that something else than a runner compiles or records, without a GPU: tensors of the CPU
stand for the GPU's, and nothing is launched (results hold whatever their memory held)."""
import pytest
import torch
import torch.nn as nn

from pfeife_amd import layers
from test_decoder_host import on_the_cpu  # noqa: F401  (a fixture)


class Layers(nn.Module):
    def __init__(self, kept="16bit", dtype=torch.bfloat16):
        super().__init__()
        self.table = nn.Parameter(torch.zeros(11, 16, dtype=dtype))
        self.up = nn.Parameter(torch.zeros(24, 16, dtype=dtype))
        self.kept = kept

    def forward(self, ids):
        return layers.gated_linear(layers.embedding(ids, self.table, scale=2.0, padding_idx=-2), self.up, act="gelu", kept=self.kept)


IDS = torch.zeros(2, 3, dtype=torch.int64)


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
@pytest.mark.parametrize("kept,dtype", [("16bit", torch.bfloat16), ("8bit", torch.bfloat16), ("16bit", torch.float32)])
def test_a_model_that_trains(on_the_cpu, backend, kept, dtype):  # noqa: F811
    """Forward and backward pass as the compiler's backends take them, those that trace the backward pass among them."""
    torch._dynamo.reset()
    model = Layers(kept, dtype)
    out = torch.compile(model, backend=backend, fullgraph=True)(IDS)
    assert out.shape == (2, 3, 12) and out.dtype == dtype
    grads = torch.autograd.grad(out, list(model.parameters()), torch.zeros_like(out))
    assert [(g.shape, g.dtype) for g in grads] == [(p.shape, dtype) for p in model.parameters()]


@pytest.mark.parametrize("frozen", ["table", "up"])
def test_a_model_with_a_frozen_part(on_the_cpu, frozen):  # noqa: F811
    torch._dynamo.reset()
    model = Layers()
    getattr(model, frozen).requires_grad_(False)
    out = torch.compile(model, backend="aot_eager", fullgraph=True)(IDS)
    out.sum().backward()
    assert all((p.grad is None) == (n == frozen) for n, p in model.named_parameters())


def test_the_backward_pass_is_a_node_of_the_traced_graph(on_the_cpu):  # noqa: F811
    from torch._dynamo.backends.common import aot_autograd

    torch._dynamo.reset()
    seen = []

    def keep(graph, inputs):
        seen.append({str(n.target) for n in graph.graph.nodes if n.op == "call_function"})
        return graph.forward

    out = torch.compile(Layers(), backend=aot_autograd(fw_compiler=keep, bw_compiler=keep), fullgraph=True)(IDS)
    out.sum().backward()
    assert {"pfeife_amd.embedding.default", "pfeife_amd.gated_linear.default"} <= seen[0]
    assert {"pfeife_amd.embedding_backward.default", "pfeife_amd.gated_linear_backward.default"} <= seen[1]


def test_second_derivatives_are_refused_there_too(on_the_cpu):  # noqa: F811
    torch._dynamo.reset()
    model = Layers()
    out = torch.compile(model, backend="eager", fullgraph=True)(IDS)
    for p in (model.up, model.table):
        g, = torch.autograd.grad(out, p, torch.zeros_like(out).requires_grad_(), create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum() + model.up.square().sum(), model.up)


def recorded_by_make_fx(fn, *args):
    from torch.fx.experimental.proxy_tensor import make_fx

    return {str(n.target) for n in make_fx(fn)(*args).graph.nodes}


def recorded_before_dispatch(fn, *args):
    from torch.fx.experimental.proxy_tensor import make_fx

    return {str(n.target) for n in make_fx(fn, pre_dispatch=True)(*args).graph.nodes}


def recorded_by_jit(fn, *args):
    return {n.kind().replace("::", ".") + ".default" for n in torch.jit.trace(fn, args, check_trace=False).graph.nodes()}


RECORDERS = pytest.mark.parametrize("record", [recorded_by_make_fx, recorded_before_dispatch, recorded_by_jit])


@RECORDERS
def test_calls_that_are_recorded_are_nodes(on_the_cpu, record):  # noqa: F811
    """A graph recorded from real calls holds the operators, not the memory that they were about to fill."""
    table, up = torch.zeros(11, 16), torch.zeros(24, 16)
    assert "pfeife_amd.embedding.default" in record(lambda ids, w: layers.embedding(ids, w, scale=3.0), IDS, table)
    assert "pfeife_amd.gated_linear.default" in record(lambda x, w: layers.gated_linear(x, w, act="relu"), torch.zeros(2, 16), up)


def test_a_recorded_backward_pass_is_a_node(on_the_cpu):  # noqa: F811
    up = torch.zeros(24, 16)

    def step(x, w):
        w = w.detach().requires_grad_()
        return torch.autograd.grad(layers.gated_linear(x, w), w, torch.ones(2, 12))[0]

    assert "pfeife_amd.gated_linear_backward.default" in recorded_by_make_fx(step, torch.zeros(2, 16), up)


@RECORDERS
def test_losses_that_are_recorded_are_refused(on_the_cpu, record):  # noqa: F811
    from pfeife_amd import loss

    h, w, y = torch.zeros(2, 3, 8), torch.zeros(5, 8), torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="linear_cross_entropy: .*recorded"):
        record(lambda h, w: loss.linear_cross_entropy(h, w, y), h, w)
    with pytest.raises(RuntimeError, match="token_logprobs: .*recorded"):
        record(lambda h: loss.token_logprobs(h, y), h)


@pytest.mark.parametrize("run", ["eager", "aot_eager", recorded_by_make_fx, recorded_by_jit])
def test_8_bits_of_fp32_operands_are_refused_before_anything_runs(on_the_cpu, run):  # noqa: F811
    """... as they are where nothing is compiled."""
    torch._dynamo.reset()
    model = Layers("8bit", torch.float32)
    with pytest.raises(RuntimeError, match="kept is '16bit', or for 16-bit operands '8bit'"):
        if callable(run):
            run(model, IDS)
        else:
            torch.compile(model, backend=run, fullgraph=True)(IDS)


def runner_step(model, mixed=None, ids=IDS):
    from oracle.kernels_oracle import OracleKernels
    from pfeife_amd.mp import PartialRunner, initialize_pfeife, net_states, partial_compiler
    from pfeife_amd.option import PipeOption

    torch._dynamo.reset()
    net_states._reset_state_for_tests()
    initialize_pfeife(device="cpu")
    runner = PartialRunner(PipeOption(device_cnt=1, batch_cnt=1, batch_size=2, mixed_precision=mixed, loss_scale=1.0, optimizer=dict(type="sgd", lr=0.0)),
                           kernels=OracleKernels("cpu"))
    compiled = torch.compile(model, backend=partial_compiler)

    def fn(ids):
        loss = compiled(ids).float().sum()
        loss.backward()
        return loss.detach()

    runner.set_exec_fn(fn)
    return runner.step(ids)


def test_8_bits_in_a_runner_go_by_what_it_computes_in():
    """fp32 parameters under mixed precision are operands of 16 bits."""
    from pfeife_amd.executor.lowering import Unsupported

    assert len(runner_step(Wide("8bit"), "bf16")) == 1
    with pytest.raises(Unsupported, match="kept is '16bit', or for 16-bit operands '8bit'"):
        runner_step(Wide("8bit"))


class Wide(Layers):
    """(A runner's widths are multiples of 8.)"""

    def __init__(self, kept):
        super().__init__(kept, torch.float32)
        self.up = nn.Parameter(torch.ones(32, 16))


class Computed(nn.Module):
    """A table that the model computes, once from all of a parameter and once from some of its columns"""

    def __init__(self, plain):
        super().__init__()
        self.table = nn.Parameter(torch.linspace(-1, 1, 11 * 16).view(11, 16))
        self.plain = plain

    def forward(self, ids):
        look = (lambda t, s: nn.functional.embedding(ids, t, padding_idx=3) * s) if self.plain else lambda t, s: layers.embedding(ids, t, scale=s, padding_idx=3)
        return look(self.table * 2.0, 0.5) + look(self.table.float(), 3.0) + look(self.table.to(torch.bfloat16), 2.0).float()


def test_a_table_that_is_computed_in_a_runner():
    """Its gradient reaches the parameter."""
    ids = torch.tensor([[1, 5, 3], [5, 5, 10]])
    model, plain = Computed(False), Computed(True)
    got = runner_step(model, ids=ids)
    want = plain(ids).float().sum()
    want.backward()
    assert abs(float(got[0]) - float(want.detach())) <= 1e-5 * abs(float(want.detach()))
    assert torch.allclose(model.table.grad, plain.table.grad, rtol=1e-5, atol=1e-6) and plain.table.grad[5].any() and not model.table.grad[3].any()


def test_a_table_that_learns_nothing_in_a_runner():
    model = Computed(False)
    model.table.requires_grad_(False)
    model.bias = nn.Parameter(torch.zeros(16))
    model.forward = lambda ids: layers.embedding(ids, model.table * 2.0) + model.bias
    runner_step(model)
    assert model.bias.grad is not None and model.table.grad is None
