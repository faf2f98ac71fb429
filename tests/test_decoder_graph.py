"""`layers.embedding` and `layers.gated_linear` inside a model that a runner compiles: a node of the graph each, in stages and micro-batches,
against plain PyTorch (kernel table double on the CPU)."""
import copy

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from oracle.kernels_oracle import OracleKernels
from pfeife_amd import layers
from pfeife_amd.mp import net_states
from pfeife_amd.option import PipeOption

SCALE = 5.0


class Block(nn.Module):
    def __init__(self, dim, ffn, act, kept, plain):
        super().__init__()
        self.norm = nn.RMSNorm(dim, eps=1e-5)
        self.up = nn.Parameter(torch.randn(2 * ffn, dim) * dim ** -0.5)
        self.down = nn.Linear(ffn, dim, bias=False)
        self.act, self.kept, self.plain = act, kept, plain

    def forward(self, x):
        h = self.norm(x)
        if self.plain:
            g, u = F.linear(h, self.up).chunk(2, -1)
            y = (F.silu(g) if self.act == "silu" else F.gelu(g)) * u
        else:
            y = layers.gated_linear(h, self.up, act=self.act, kept=self.kept)
        return x + self.down(y)


class Decoder(nn.Module):
    """No attention: what is tested stands around it.  The last hidden state is the result, its head is the loss's."""

    def __init__(self, vocab=61, dim=32, ffn=48, depth=3, act="silu", kept="16bit", plain=False, padding=None):
        super().__init__()
        self.table = nn.Parameter(torch.randn(vocab, dim) * 0.2)
        self.blocks = nn.ModuleList([Block(dim, ffn, act, kept, plain) for _ in range(depth)])
        self.norm = nn.RMSNorm(dim, eps=1e-5)
        self.plain, self.padding = plain, padding

    def forward(self, ids):
        x = F.embedding(ids, self.table, padding_idx=self.padding) * SCALE if self.plain else layers.embedding(ids, self.table, scale=SCALE, padding_idx=self.padding)
        for block in self.blocks:
            x = block(x)
        return self.norm(x)


def objective(out):
    """(A square of what a norm gives would have next to no gradient.)"""
    return (out.float() * torch.linspace(-1, 1, out.shape[-1], device=out.device)).sum(-1).tanh().mean()


def plain_of(model):
    ref = copy.deepcopy(model)
    for m in ref.modules():
        if hasattr(m, "plain"):
            m.plain = True
    return ref


@pytest.mark.parametrize("mixed,act,kept", [(None, "silu", "16bit"), (None, "gelu", "16bit"), ("bf16", "silu", "16bit"), ("bf16", "gelu", "8bit")])
def test_in_a_runner(mixed, act, kept):
    from pfeife_amd.mp import PartialRunner, initialize_pfeife, partial_compiler

    torch._dynamo.reset()
    net_states._reset_state_for_tests()
    initialize_pfeife(device="cpu")
    torch.manual_seed(0)
    model = Decoder(act=act, kept=kept, padding=3)
    ref = plain_of(model)
    runner = PartialRunner(PipeOption(device_cnt=2, batch_cnt=2, batch_size=2, split_points=["blocks.1"], mixed_precision=mixed, loss_scale=1.0,
                                      optimizer=dict(type="sgd", lr=0.0)), kernels=OracleKernels("cpu"))
    compiled = torch.compile(model, backend=partial_compiler)

    def fn(ids):
        loss = objective(compiled(ids))
        loss.backward()
        return loss.detach()

    runner.set_exec_fn(fn)
    ids = torch.randint(0, 61, (4, 9), generator=torch.Generator().manual_seed(1))
    ids[:, 2] = 3
    got = runner.step(ids)
    for k in range(2):
        with torch.autocast("cpu", dtype=torch.bfloat16, enabled=mixed is not None):
            want = objective(ref(ids[2 * k:2 * k + 2]))
        want.backward()
        assert abs(float(got[k]) - float(want.detach())) <= (1e-5 if mixed is None else 3e-2)
    # bf16 results round every product once, in another place of the plain model's chain; 8 bits hold 4 digits of the pre-activations
    for (n, p), (_, q) in zip(model.named_parameters(), ref.named_parameters()):
        far = (p.grad - q.grad).norm() / (q.grad.norm() + 1e-12)
        assert far <= (1e-5 if mixed is None else 3e-2 if kept == "16bit" else 8e-2), (n, float(far))
    assert not model.table.grad[3].any()


def test_widths_without_a_kernel_are_refused():
    from pfeife_amd.executor.lowering import Unsupported
    from pfeife_amd.mp import PartialRunner, initialize_pfeife, partial_compiler

    torch._dynamo.reset()
    net_states._reset_state_for_tests()
    initialize_pfeife(device="cpu")
    model = Decoder(ffn=44)
    runner = PartialRunner(PipeOption(device_cnt=1, batch_cnt=1, batch_size=2, optimizer=dict(type="sgd", lr=0.0)), kernels=OracleKernels("cpu"))
    compiled = torch.compile(model, backend=partial_compiler)

    def fn(ids):
        loss = objective(compiled(ids))
        loss.backward()
        return loss.detach()

    runner.set_exec_fn(fn)
    with pytest.raises(Unsupported, match="multiples of 8"):
        runner.step(torch.randint(0, 61, (2, 9)))
