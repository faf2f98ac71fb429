"""The decoder operators where one launch is not enough: a vocabulary in pieces, sums in shares, rows and ids of several launches."""
import pytest
import torch
import torch.nn.functional as F

from test_decoder_ops_gpu import IGNORE, TYPES, U32, head_inputs, head_reference, table_reference, within

pytestmark = pytest.mark.gpu


# 1000 tokens: pieces of 131072 classes in 16 bits, 65536 in fp32.  The last piece is of fewer rows than it would have shares, or a few of its shares'
PIECES = [(1, 1000, 64, 131072 + 300), (4, 250, 33, 131072 + 1), (1, 990, 72, 65536 * 2 + 5000)]


@pytest.mark.parametrize("B,T,D,V", PIECES)
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_cross_entropy_in_pieces_of_the_vocabulary(dtype, B, T, D, V):
    from pfeife_amd.loss import linear_cross_entropy

    h, w, y = head_inputs(dtype, B, T, D, V)
    y[0, 5], y[0, 6], y[0, 7] = V - 1, 65536, 131071      # labels at the pieces' ends
    h.requires_grad_()
    w.requires_grad_()
    loss = linear_cross_entropy(h, w, y)
    dh, dw = torch.autograd.grad(loss, (h, w))
    term, bound, rh, eh, rw, ew = head_reference(h.detach(), w.detach(), y, 0, "mean", 0.0, torch.ones((), device="cuda"))
    within(loss.detach(), term, bound, torch.float32)
    within(dh, rh, eh, dtype)
    within(dw, rw, ew, dtype)
    again = torch.autograd.grad(linear_cross_entropy(h, w, y), (h, w))
    assert torch.equal(again[0], dh) and torch.equal(again[1], dw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scored", [0, 1, 2, 3, 65, 255, 256, 257])
def test_linear_cross_entropy_counts_on_the_device(dtype, scored):
    """Grids cover 700 tokens, `scored` take part: the counted dimension ends anywhere in a tile, a stage or a vector."""
    from pfeife_amd.loss import linear_cross_entropy

    h, w, y = head_inputs(dtype, 1, 700, 132, 1003, masked=0.0)
    order = torch.randperm(700, generator=torch.Generator().manual_seed(scored)).cuda()
    y[0, order[scored:]] = IGNORE
    h[0, order[scored:]] = float("nan")
    h.requires_grad_()
    w.requires_grad_()
    loss = linear_cross_entropy(h, w, y, reduction="sum")
    dh, dw = torch.autograd.grad(loss, (h, w))
    clean = torch.where((y == IGNORE).unsqueeze(-1), torch.zeros_like(h.detach()), h.detach())
    term, bound, rh, eh, rw, ew = head_reference(clean, w.detach(), y, 0, "sum", 0.0, torch.ones((), device="cuda"))
    within(loss.detach(), term, bound, torch.float32)
    within(dh, rh, eh, dtype)
    within(dw, rw, ew, dtype)


@pytest.mark.parametrize("n,D,V", [(48, 257, 1000), (47, 1030, 65), (49, 130, 300), (1, 4, 17), (9, 2051, 1)])
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_cross_entropy_of_a_few_tokens(dtype, n, D, V):
    from pfeife_amd.loss import linear_cross_entropy

    h, w, y = head_inputs(dtype, 1, n, D, V, masked=0.2)
    h.requires_grad_()
    w.requires_grad_()
    loss = linear_cross_entropy(h, w, y, reduction="none")
    up = 0.5 + torch.rand(loss.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    dh, dw = torch.autograd.grad(loss, (h, w), up)
    term, bound, rh, eh, rw, ew = head_reference(h.detach(), w.detach(), y, 0, "none", 0.0, up)
    within(loss.detach(), term, bound, torch.float32)
    within(dh, rh, eh, dtype)
    within(dw, rw, ew, dtype)


def test_embedding_of_more_ids_than_a_launch_takes():
    from pfeife_amd.layers import embedding

    n = (1 << 25) + 77
    ids = torch.randint(0, 100, (n,), device="cuda", generator=torch.Generator("cuda").manual_seed(0))
    w = torch.randn(100, 3, device="cuda").half()
    out = embedding(ids, w)
    for at in (slice(0, 1000), slice((1 << 25) - 500, n)):
        assert torch.equal(out[at], w[ids[at]])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gated_linear_of_more_rows_than_a_launch_takes(dtype):
    """Without a backward pass rows come in launches of 65024 here; with one they are refused, in words."""
    from pfeife_amd.layers import gated_linear

    g = torch.Generator("cuda").manual_seed(0)
    rows, D, ffn = 65024 + 333, 64, 8192
    x = torch.randn(rows, D, device="cuda", generator=g).to(dtype)
    w = (torch.randn(2 * ffn, D, device="cuda", generator=g) * D ** -0.5).to(dtype)
    y = gated_linear(x, w)
    for at in (slice(0, 64), slice(65024 - 40, 65024 + 40), slice(rows - 40, rows)):
        x64, w64 = x[at].double(), w.double()
        z, off = x64 @ w64.t(), (D + 8) * U32 * (x64.abs() @ w64.abs().t())
        a, b, ea, eb = z[:, :ffn], z[:, ffn:], off[:, :ffn], off[:, ffn:]
        v = F.silu(a)
        # an activation's slope is at most 1.1, its own arithmetic off by 2e-6 or 8 units of 2^-24
        within(y[at], v * b, (1.2 * ea + 2e-6 * a.abs().clamp_max(1.0) + 8 * U32 * a.abs()) * (b.abs() + eb) + v.abs() * eb, dtype)
    with pytest.raises(RuntimeError, match="too large for one call"):
        gated_linear(x, w.requires_grad_())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scored", [0, 1, 300, 700, 1025, 1300, 2048])
def test_linear_cross_entropy_in_shares_by_the_count(dtype, scored):
    """2048 tokens by 1024 columns: 32 tiles of 256, and with fewer tokens more shares of the vocabulary, whose number the device finds."""
    from pfeife_amd.loss import linear_cross_entropy

    h, w, y = head_inputs(dtype, 2, 1024, 1024, 70001, masked=0.0)
    order = torch.randperm(2048, generator=torch.Generator().manual_seed(scored)).cuda()
    y.view(-1)[order[scored:]] = IGNORE
    h.requires_grad_()
    w.requires_grad_()
    loss = linear_cross_entropy(h, w, y, reduction="sum")
    dh, dw = torch.autograd.grad(loss, (h, w))
    term, bound, rh, eh, rw, ew = head_reference(h.detach(), w.detach(), y, 0, "sum", 0.0, torch.ones((), device="cuda"))
    within(loss.detach(), term, bound, torch.float32)
    within(dh, rh, eh, dtype)
    within(dw, rw, ew, dtype)


@pytest.mark.parametrize("n,V,D", [(256, 1, 2100), (256, 3, 600), (70, 5000, 1100), (65, 2, 513), (256, 1500, 1024), (1, 7, 4000), (200, 2, 30)])
@pytest.mark.parametrize("dtype", TYPES)
def test_embedding_gradient_of_a_few_ids_in_wide_rows(dtype, n, V, D):
    """One launch does it all: rows that several wavefronts share, tokens that most of the list is, one row to a workgroup or many."""
    from pfeife_amd.layers import embedding

    g = torch.Generator().manual_seed(n + D)
    ids = torch.randint(0, V, (n,), generator=g)
    ids[n // 4: n // 2] = V - 1
    ids = ids.cuda()
    w = torch.randn(V, D, generator=g).to(dtype).cuda().requires_grad_()
    up = torch.randn(n, D, generator=g).to(dtype).cuda()
    dw, = torch.autograd.grad(embedding(ids, w, scale=1.5), w, up)
    rw, ew = table_reference(ids, w, 1.5, None, up)
    within(dw, rw, ew, dtype)


@pytest.mark.parametrize("n,D,ffn", [(1, 1030, 333), (4, 515, 40), (3, 8, 1), (4, 2048, 2050), (5, 77, 129), (16, 513, 31), (17, 513, 31), (2, 64, 9000)])
@pytest.mark.parametrize("dtype,kept", [(torch.float16, "16bit"), (torch.bfloat16, "8bit")])
def test_gated_linear_backward_of_a_few_rows(dtype, kept, n, D, ffn):
    """Kernels of their own up to 4 rows (x) and 16 (weight): widths that end inside a lane's eight columns, a block of rows, a half."""
    from pfeife_amd.layers import gated_linear
    from test_decoder_ops_gpu import gated_check

    g = torch.Generator().manual_seed(n + D)
    x = torch.randn(n, D, generator=g).to(dtype).cuda().requires_grad_()
    w = (torch.randn(2 * ffn, D, generator=g) * D ** -0.5).to(dtype).cuda().requires_grad_()
    up = torch.randn(n, ffn, generator=g).to(dtype).cuda()
    y = gated_linear(x, w, act="gelu", kept=kept)
    dx, dw = torch.autograd.grad(y, (x, w), up)
    gated_check(x.detach(), w.detach(), "gelu", kept, up, y.detach(), dx, dw)
