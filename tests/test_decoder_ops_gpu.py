"""linear_cross_entropy, embedding and gated_linear against the same in 64 bits.

Bounds follow the arithmetic: U is half a step of a type, a sum of n terms in fp32 is off by at most n 2^-24 times the sum of their
magnitudes in any order, the hardware's exponential by two units of 2^-24 besides its argument's rounding."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}    # (half a step where steps end, or what flushes to zero)
U32 = 2.0 ** -24
IGNORE = -100
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def within(got, want, tol, dtype):
    """got against want: off by tol, and a rounding to the type."""
    tol = tol * (1 + U[dtype]) + U[dtype] * want.abs() + LEAST[dtype]
    off = (got.double() - want).abs() - tol
    assert got.dtype == dtype and torch.isfinite(got).all() and (off <= 0).all(), float(off.max())


# -- linear_cross_entropy -----------------------------------------------------------------------------------------------------

def head_inputs(dtype, B, T, D, V, seed=0, masked=0.3, sure=3.0):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, D, generator=g) * D ** -0.5).to(dtype).cuda()
    y = torch.randint(0, V, (B, T), generator=g).cuda()
    h = (torch.randn(B, T, D, generator=g).cuda() + sure * w[y].float()).to(dtype)
    y[(torch.rand(B, T, generator=g) < masked).cuda()] = IGNORE
    if B > 2:
        y[1] = IGNORE        # a sequence with nothing to score
    return h, w, y


def head_reference(h, w, y, shift, reduction, z_loss, up):
    """-> (loss, its bound, dh, bound, dw, bound) in 64 bits"""
    s, dtype = int(shift), h.dtype
    B, T, D = h.shape
    V = w.shape[0]
    x, w64, label = h[:, :T - s].double(), w.double(), y[:, s:]
    seen = label != IGNORE
    z = x @ w64.t()
    dz_ = (D + 8) * U32 * (x.abs() @ w64.abs().t())              # of every logit
    top, lse, p = z.amax(-1, keepdim=True), torch.logsumexp(z, -1), torch.softmax(z, -1)
    far = torch.where(p > 0, p * (top - z), 0).sum(-1)
    off = dz_.amax(-1)
    # sums of up to 64 terms in a lane, their merges; the exponent's rounding; what the logits are off by
    rel = (80 + 4 * far) * U32 + off
    at = torch.where(seen, label, 0).unsqueeze(-1)
    term = torch.where(seen, lse - z.gather(-1, at).squeeze(-1) + z_loss * lse ** 2, 0)
    bound = torch.where(seen, (rel + off) * (1 + 2 * z_loss * lse.abs()) + 4 * U32 * (lse.abs() + 1) * (1 + z_loss * lse.abs()), 0)
    n = seen.sum().clamp_min(1)
    c = torch.where(seen, up.double().expand(B, T - s) / (n if reduction == "mean" else 1), 0)
    if reduction != "none":
        term, bound = term.sum(), bound.sum() + (abs(term.sum()) * 2 * U32)
        if reduction == "mean":
            term, bound = term / n, bound / n
    onehot = torch.zeros_like(z).scatter_(-1, at, 1.0)
    f = c * (1 + 2 * z_loss * lse)
    d = f.unsqueeze(-1) * p - c.unsqueeze(-1) * onehot
    # the factors' own roundings, the probability's error, and dz's rounding to the type, which fp16 does at 2^13 over the largest factor
    e = (f.abs() * (2 * rel + 6 * U32) + c.abs() * 2 * z_loss * rel).unsqueeze(-1) * p + c.abs().unsqueeze(-1) * onehot * 4 * U32
    if dtype != torch.float32:
        e = e + U[dtype] * d.abs()
        if dtype == torch.float16:
            e = e + LEAST[dtype] * torch.maximum(f.abs().max(), c.abs().max()) / 8192
    dh = torch.zeros(B, T, D, dtype=torch.float64, device=h.device)
    eh = torch.zeros_like(dh)
    dh[:, :T - s] = d @ w64
    eh[:, :T - s] = (e + (V + 32) * U32 * d.abs()) @ w64.abs()
    flat = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
    dw = flat(d).t() @ flat(x)
    ew = flat(e + (B * T + 128) * U32 * d.abs()).t() @ flat(x).abs()
    return term, bound, dh, eh, dw, ew


HEADS = [(1, 1, 64, 64, 0, "mean", 0.0), (2, 5, 8, 3, 1, "none", 0.0), (1, 1, 1, 1, 0, "sum", 0.0), (3, 50, 100, 1000, 1, "sum", 1e-3), (2, 130, 128, 777, 0, "mean", 0.0),
         (4, 90, 96, 5003, 1, "none", 1e-4), (2, 600, 192, 3001, 1, "mean", 0.0), (1, 3, 37, 129, 0, "mean", 1e-3), (2, 300, 65, 515, 0, "sum", 0.0),
         (1, 64, 64, 256, 0, "none", 0.0), (5, 13, 128, 257, 0, "mean", 0.0), (3, 1700, 64, 300, 1, "none", 0.0), (1, 16, 256, 40007, 0, "mean", 0.0)]


@pytest.mark.parametrize("B,T,D,V,shift,reduction,z_loss", HEADS)
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_cross_entropy(dtype, B, T, D, V, shift, reduction, z_loss):
    from pfeife_amd.loss import linear_cross_entropy

    h, w, y = head_inputs(dtype, B, T, D, V)
    h.requires_grad_()
    w.requires_grad_()
    loss = linear_cross_entropy(h, w, y, shift=bool(shift), reduction=reduction, z_loss=z_loss)
    scale = 256.0 if dtype == torch.float16 else 1.0
    up = scale * (0.5 + torch.rand(loss.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(5)))
    dh, dw = torch.autograd.grad(loss, (h, w), up)
    term, bound, rh, eh, rw, ew = head_reference(h.detach(), w.detach(), y, shift, reduction, z_loss, up)
    within(loss.detach(), term, bound, torch.float32)
    within(dh, rh, eh, dtype)
    within(dw, rw, ew, dtype)
    with torch.no_grad():
        assert torch.equal(linear_cross_entropy(h, w, y, shift=bool(shift), reduction=reduction, z_loss=z_loss), loss)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_cross_entropy_against_differences(dtype):
    """The gradient along a direction against the loss's difference along it (fp32 alone has the digits for that; the others by their own
    bounds above): second-order terms are below 1e-3 of it at this step."""
    from pfeife_amd.loss import linear_cross_entropy

    h, w, y = head_inputs(torch.float32, 2, 40, 48, 333)
    if dtype != torch.float32:
        h, w = h.to(dtype).float(), w.to(dtype).float()
    h.requires_grad_()
    w.requires_grad_()
    dh, dw = torch.autograd.grad(linear_cross_entropy(h, w, y, reduction="sum"), (h, w))
    gen = torch.Generator("cuda").manual_seed(3)
    vh, vw = torch.randn(h.shape, device="cuda", generator=gen), 0.1 * torch.randn(w.shape, device="cuda", generator=gen)
    step = 1e-2
    with torch.no_grad():
        up, down = (float(linear_cross_entropy(h + s * vh, w + s * vw, y, reduction="sum")) for s in (step, -step))
    along = float((dh.double() * vh).sum() + (dw.double() * vw).sum())
    # losses of some 60 tokens around 6, each off by 1e-6; third derivatives of a log-sum-exp are at most the cube of the logits' change
    assert abs((up - down) / (2 * step) - along) <= 400 * 1e-6 / (2 * step) + 5e-3 * abs(along)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_cross_entropy_nothing_to_score(dtype):
    from pfeife_amd.loss import linear_cross_entropy

    h, w, y = head_inputs(dtype, 2, 70, 64, 100)
    y[:] = IGNORE
    h[:] = float("nan")      # (what ignored tokens hold does not matter)
    for reduction in ("mean", "sum", "none"):
        a, b = h.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
        loss = linear_cross_entropy(a, b, y, reduction=reduction)
        ga, gb = torch.autograd.grad(loss, (a, b), torch.ones_like(loss))
        assert not loss.any() and not ga.any() and not gb.any() and torch.isfinite(loss).all()
    empty = torch.zeros(0, 5, 64, dtype=dtype, device="cuda", requires_grad=True)
    b = w.detach().clone().requires_grad_()
    loss = linear_cross_entropy(empty, b, torch.zeros(0, 5, dtype=torch.int64, device="cuda"))
    ge, gb = torch.autograd.grad(loss, (empty, b))
    assert float(loss.detach()) == 0 and ge.shape == empty.shape and not gb.any()
    one = h[:, :1].clone().requires_grad_()
    assert linear_cross_entropy(one, w, y[:, :1], shift=True, reduction="none").shape == (2, 0)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_cross_entropy_masked_places(dtype):
    """Infinities and NaN in tokens that take no part reach nothing; a label outside the vocabulary is NaN in its own token."""
    from pfeife_amd.loss import linear_cross_entropy

    h, w, y = head_inputs(dtype, 2, 40, 72, 300)
    clean = linear_cross_entropy(h, w, y, reduction="none")
    bad = h.clone()
    bad[y == IGNORE] = float("inf")
    bad[0, (y[0] == IGNORE).nonzero()[0, 0]] = float("nan")
    bad.requires_grad_()
    loss = linear_cross_entropy(bad, w, y, reduction="none")
    assert torch.equal(loss, clean)
    g, = torch.autograd.grad(loss, bad, torch.ones_like(loss))
    assert torch.isfinite(g).all() and not g[y == IGNORE].any()
    for label in (300, -1, 1 << 40):
        wrong = y.clone()
        wrong[1, 3] = label
        a = h.clone().requires_grad_()
        loss = linear_cross_entropy(a, w, wrong, reduction="none")
        keep = torch.ones_like(y, dtype=torch.bool)
        keep[1, 3] = False
        assert torch.isnan(loss[1, 3]) and torch.equal(loss[keep], linear_cross_entropy(h, w, torch.where(keep, y, IGNORE), reduction="none")[keep])
        g, = torch.autograd.grad(loss, a, torch.ones_like(loss))
        assert torch.isnan(g[1, 3]).all() and torch.isfinite(g[keep]).all()


def test_linear_cross_entropy_sure_and_far():
    """Losses near zero keep their digits, logits of hundreds do not overflow."""
    from pfeife_amd.loss import linear_cross_entropy

    for dtype in TYPES:
        w = torch.eye(64, device="cuda").to(dtype)
        h = torch.zeros(1, 4, 64, device="cuda")
        for t, v in enumerate((8.0, 16.0, 300.0, -300.0)):
            h[0, t, 5] = v
        h = h.to(dtype)
        y = torch.full((1, 4), 5, device="cuda")
        z = h.double() @ w.double().t()
        want = torch.logsumexp(z, -1) - z[..., 5]
        got = linear_cross_entropy(h, w, y, reduction="none").double()
        # beside the label's 1 lie 63 terms e^-v: the partial sums that hold the 1 are off by 8 roundings of it, the others relatively
        assert ((got - want).abs() <= 12 * U32 * torch.maximum(want.abs() + 300 * (want > 100), torch.tensor(1.0, device="cuda").double())).all(), (dtype, got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_cross_entropy_layouts(dtype):
    """Strided, expanded, transposed and 2-D operands give the dense ones' bits."""
    from pfeife_amd.loss import linear_cross_entropy

    h, w, y = head_inputs(dtype, 3, 50, 64, 200)
    want = linear_cross_entropy(h, w, y, shift=True, reduction="none")
    wide = torch.randn(3, 50, 80, device="cuda").to(dtype)
    wide[..., 8:72] = h
    odd = torch.randn(3, 50, 67, device="cuda").to(dtype)
    odd[..., 3:67] = h
    swapped = h.transpose(0, 1).contiguous().transpose(0, 1)
    turned = h.transpose(1, 2).contiguous().transpose(1, 2)
    wt = w.t().contiguous().t()
    base = torch.zeros(w.numel() + 1, dtype=dtype, device="cuda")
    shifted = base[1:].view_as(w)
    shifted.copy_(w)
    for a in (wide[..., 8:72], odd[..., 3:67], swapped, turned):
        assert torch.equal(linear_cross_entropy(a, w, y, shift=True, reduction="none"), want)
        b = a.detach().requires_grad_()
        g, = torch.autograd.grad(linear_cross_entropy(b, w, y, shift=True), b)
        c = h.detach().requires_grad_()
        assert torch.equal(g, torch.autograd.grad(linear_cross_entropy(c, w, y, shift=True), c)[0])
    for v in (wt, shifted):
        assert torch.equal(linear_cross_entropy(h, v, y, shift=True, reduction="none"), want)
    # fewer tokens may be summed in other groups: each sum of exponentials is off by at most the test above's (80 + 4 far) 2^-24, far being
    # the distance from the largest logit in the mean, below 8 here: 2 * 112 * 2^-24
    flat = linear_cross_entropy(h[0], w, y[0], shift=True, reduction="none")
    assert flat.shape == (49,) and ((flat - want[0]).abs() <= 224 * U32).all()
    four = linear_cross_entropy(h.view(1, 3, 50, 64), w, y.view(1, 3, 50), shift=True, reduction="none")
    assert four.shape == (1, 3, 49) and torch.equal(four[0], want)


def test_linear_cross_entropy_parts_of_the_gradient():
    """A frozen weight or hidden state gets none, and the other the same bits; the upstream gradient of a sum is one number without strides."""
    from pfeife_amd.loss import linear_cross_entropy

    h, w, y = head_inputs(torch.bfloat16, 2, 90, 128, 500)
    a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
    dh, dw = torch.autograd.grad(linear_cross_entropy(a, b, y), (a, b))
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(a, w, y), a)[0], dh)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(h, b, y), b)[0], dw)
    linear_cross_entropy(a, b, y, reduction="none").sum().backward()
    total = torch.autograd.grad(linear_cross_entropy(a, b, y, reduction="sum"), (a, b))
    assert torch.equal(a.grad, total[0]) and torch.equal(b.grad, total[1])
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        g, = torch.autograd.grad(linear_cross_entropy(a, b, y), a, create_graph=True)
        g.sum().backward()


# -- embedding ----------------------------------------------------------------------------------------------------------------

def table_reference(ids, w, scale, padding, up):
    s = float(torch.tensor(scale, dtype=torch.float32))
    keep = (ids >= 0) & (ids < w.shape[0])
    if padding is not None:
        keep &= ids != padding % w.shape[0]
    at, d = ids[keep].cpu(), up.reshape(-1, w.shape[1])[keep.reshape(-1)].double().cpu()
    add = lambda v: torch.zeros((w.shape[0],) + v.shape[1:], dtype=torch.float64).index_add_(0, at, v).to(w.device)  # noqa: E731
    dw, most, count = add(d) * s, add(d.abs()) * abs(s), add(torch.ones(len(at), dtype=torch.float64))
    return dw, count.unsqueeze(1) * U32 * most + U32 * dw.abs()


TABLES = [(1, 5, 3, 0.0), (7, 1, 8, 0.0), (256, 300, 64, 0.3), (257, 300, 64, 0.3), (64, 2000, 33, 0.0), (2048, 77, 100, 0.0), (2049, 5000, 17, 0.3), (5000, 40, 520, 0.5),
          (9001, 70000, 31, 0.2), (16384, 3000, 96, 0.4), (20000, 300, 16, 0.0), (65536, 1000, 8, 0.9), (65537, 1000, 9, 0.9), (70001, 300007, 4, 0.4), (3000, 2200000, 2, 0.0)]


@pytest.mark.parametrize("n,V,D,hot", TABLES)
@pytest.mark.parametrize("dtype", TYPES)
def test_embedding(dtype, n, V, D, hot):
    """Rows and gradients, tokens that are most of the list (their runs cross chunks and blocks of chunks), ids outside the table, a padding row."""
    from pfeife_amd.layers import embedding

    g = torch.Generator().manual_seed(n + V)
    ids = torch.randint(0, V, (n,), generator=g)
    ids[torch.rand(n, generator=g) < hot] = V // 2
    if n > 5:
        ids[n // 3], ids[n // 2] = -1, V + 3
    ids = ids.cuda()
    w = torch.randn(V, D, generator=g).to(dtype).cuda().requires_grad_()
    padding = None if n % 2 else -(V // 3) - 1
    scale = 0.37
    out = embedding(ids, w, scale=scale, padding_idx=padding)
    ok = (ids >= 0) & (ids < V)
    want = w.detach()[ids.clamp(0, V - 1)].double() * scale
    within(out.detach()[ok], want[ok], 2 * U32 * want[ok].abs(), dtype)
    assert torch.isnan(out.detach()[~ok]).all()
    up = torch.randn(n, D, generator=g).to(dtype).cuda()
    dw, = torch.autograd.grad(out, w, up)
    rw, ew = table_reference(ids, w, scale, padding, up)
    within(dw, rw, ew, dtype)
    if padding is not None:
        assert not dw[padding].any()
    again, = torch.autograd.grad(embedding(ids, w, scale=scale, padding_idx=padding), w, up)
    assert torch.equal(again, dw)      # the same ids give the same bits


@pytest.mark.parametrize("n", [200, 3000, 70001])
def test_embedding_gradient_added_to_what_is_there(n):
    """The entry point's accumulate form, into fp32 from 16-bit gradients: rows that no id names are left as they were, bit for bit."""
    import pfeife_amd.loss as loss

    V, D = 500, 40
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, V // 2, (n,), generator=g).cuda()
    up = torch.randn(n, D, generator=g).bfloat16().cuda()
    old = torch.randn(V, D, generator=g).cuda()
    into, w = old.clone(), torch.zeros(V, D, device="cuda")
    loss._table(up, "test")
    ws = torch.empty(max(1, loss._need(up, "pf_embedding_sorted_workspace", n, D)), dtype=torch.uint8, device="cuda")
    loss._call(up, "pf_embedding_sorted_bwd", up.data_ptr(), 2, ids.data_ptr(), into.data_ptr(), 0, n, D, V, -1, 2.0, 1, ws.data_ptr())
    dw, ew = table_reference(ids, w, 2.0, None, up)
    assert torch.equal(into[V // 2:], old[V // 2:])
    within(into, dw + old.double(), ew + U32 * (dw.abs() + old.double().abs()), torch.float32)


def test_embedding_layouts():
    from pfeife_amd.layers import embedding

    w = torch.randn(50, 24, device="cuda")
    ids = torch.randint(0, 50, (6, 7), device="cuda")
    want = w[ids]
    assert torch.equal(embedding(ids, w), want)
    assert torch.equal(embedding(ids.t(), w), want.transpose(0, 1))
    assert torch.equal(embedding(ids, w.t().contiguous().t()), want)
    assert embedding(ids[:0], w).shape == (0, 7, 24) and embedding(ids[0, 0], w).shape == (24,)
    a = w.clone().requires_grad_()
    assert not torch.autograd.grad(embedding(ids[:0], a), a, torch.zeros(0, 7, 24, device="cuda"))[0].any()
    base = torch.zeros(50 * 24 + 1, dtype=torch.bfloat16, device="cuda")      # a table that begins between 4 bytes
    b = base[1:].view(50, 24)
    b.copy_(w)
    assert torch.equal(embedding(ids, b), b[ids])
    # a gradient that comes expanded, and one of a view
    g1, = torch.autograd.grad(embedding(ids, a).sum(), a)
    assert torch.equal(g1, torch.bincount(ids.reshape(-1), minlength=50).float().unsqueeze(1).expand(50, 24))
    g2, = torch.autograd.grad(embedding(ids, a)[:, ::2].sum(), a)
    assert torch.equal(g2, torch.bincount(ids[:, ::2].reshape(-1), minlength=50).float().unsqueeze(1).expand(50, 24))


# -- gated_linear -------------------------------------------------------------------------------------------------------------

ACTS = {"silu": F.silu, "relu": torch.relu, "gelu": F.gelu, "gelu_tanh": lambda v: F.gelu(v, approximate="tanh")}


def e4m3(v, e):
    """v over 2^e as the nearest e4m3 code, times 2^e; v in 64 bits"""
    x = torch.ldexp(v, -e).clamp(-448, 448)
    _, k = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), torch.clamp(k - 4, min=-9))
    return torch.ldexp(torch.round(x / step) * step, e)


def held(v, off, kept, dtype):
    """-> (what a pre-activation is kept as, how far the kernel's may be from that, v being off by `off`)"""
    if kept == "16bit":
        if dtype == torch.float32:
            return v, off
        to = lambda t: t.to(dtype).double()  # noqa: E731
        q = to(v)
        return q, torch.maximum((to(v + off) - q).abs(), (to(v - off) - q).abs()) * (1 + 2 * U[dtype])
    n, width = v.shape
    block = lambda t: F.pad(t, (0, -width % 16)).view(n, -1, 16)  # noqa: E731
    b, o = block(v), block(off)

    def exponent(top):
        m, e = torch.frexp(top / 448)
        e = torch.where(m == 0.5, e - 1, e).clamp(-126, 126)
        return torch.where(top == 0, 0, e)

    top, slack = b.abs().amax(-1, keepdim=True), o.amax(-1, keepdim=True)
    q = e4m3(b, exponent(top))
    far = torch.zeros_like(b)
    for t in (top, top + slack, (top - slack).clamp_min(0)):
        for u in (b - o, b + o):
            far = torch.maximum(far, (e4m3(u, exponent(t)) - q).abs())
    flat = lambda t: t.reshape(n, -1)[:, :width]  # noqa: E731
    return flat(q), flat(far)


def gated_check(x, w, act, kept, up, y, dx, dw):
    dtype, (n, D), ffn = x.dtype, x.shape, w.shape[0] // 2
    x64, w64, d = x.double(), w.double(), up.double()
    z, off = x64 @ w64.t(), (D + 8) * U32 * (x64.abs() @ w64.abs().t())
    g, u, eg, eu = z[:, :ffn], z[:, ffn:], off[:, :ffn], off[:, ffn:]
    fn = ACTS[act]
    # an activation's slope is at most 1.13, its own arithmetic off by 2e-6 or 8 units of 2^-24
    arith = lambda t: 2e-6 * t.abs().clamp_max(1.0) + 8 * U32 * t.abs()  # noqa: E731
    within(y, fn(g) * u, (1.2 * eg + arith(g)) * (u.abs() + eu) + fn(g).abs() * eu, dtype)
    if dx is None:
        return
    g, eg = held(g, eg, kept, dtype)
    u, eu = held(u, eu, kept, dtype)
    leaf = g.clone().requires_grad_()
    slope, = torch.autograd.grad(fn(leaf).sum(), leaf)
    value = fn(g)
    # slopes change by at most 1 a unit (relu's jumps where its argument may be on either side of zero)
    es = torch.minimum(eg, torch.ones_like(eg)) + 4e-6 if act != "relu" else ((g.abs() <= eg) & (eg > 0)).double()
    dg, du = d * u * slope, d * value
    edg = d.abs() * (eu * (slope.abs() + es) + u.abs() * es) + 4 * U32 * dg.abs()
    edu = d.abs() * (1.2 * eg + arith(g)) + 4 * U32 * du.abs()
    dgu, e = torch.cat((dg, du), 1), torch.cat((edg, edu), 1)
    if dtype != torch.float32:
        e = e * (1 + U[dtype]) + U[dtype] * dgu.abs() + LEAST[dtype]
    within(dx, dgu @ w64, (e + (2 * ffn + 64) * U32 * dgu.abs()) @ w64.abs(), dtype)
    within(dw, dgu.t() @ x64, (e + (n + 64) * U32 * dgu.abs()).t() @ x64.abs(), dtype)


GATED = [(1, 64, 64, "silu"), (1, 1, 1, "silu"), (2, 100, 96, "gelu"), (7, 72, 33, "relu"), (3, 8, 5, "silu"), (8, 512, 40, "gelu_tanh"), (9, 520, 48, "silu"), (130, 128, 200, "gelu_tanh"),
         (300, 192, 320, "silu"), (513, 200, 364, "gelu"), (777, 333, 71, "silu"), (2100, 64, 600, "relu"), (64, 64, 1000, "silu"), (5, 1000, 17, "gelu"), (4, 40, 3000, "silu")]


@pytest.mark.parametrize("n,D,ffn,act", GATED)
@pytest.mark.parametrize("dtype,kept", [(torch.float32, "16bit"), (torch.float16, "16bit"), (torch.bfloat16, "16bit"), (torch.float16, "8bit"), (torch.bfloat16, "8bit")])
def test_gated_linear(dtype, kept, n, D, ffn, act):
    from pfeife_amd.layers import gated_linear

    g = torch.Generator().manual_seed(n + D)
    x = torch.randn(n, D, generator=g).to(dtype).cuda().requires_grad_()
    w = (torch.randn(2 * ffn, D, generator=g) * 1.5 * D ** -0.5).to(dtype).cuda().requires_grad_()
    y = gated_linear(x, w, act=act, kept=kept)
    up = torch.randn(n, ffn, generator=g).to(dtype).cuda()
    dx, dw = torch.autograd.grad(y, (x, w), up)
    gated_check(x.detach(), w.detach(), act, kept, up, y.detach(), dx, dw)
    with torch.no_grad():
        assert torch.equal(gated_linear(x, w, act=act, kept=kept), y)
    assert torch.equal(torch.autograd.grad(gated_linear(x.detach(), w, act=act, kept=kept), w, up)[0], dw)
    assert torch.equal(torch.autograd.grad(gated_linear(x, w.detach(), act=act, kept=kept), x, up)[0], dx)


def test_gated_linear_against_differences():
    from pfeife_amd.layers import gated_linear

    gen = torch.Generator("cuda").manual_seed(0)
    x, w = torch.randn(20, 48, device="cuda", generator=gen), torch.randn(72, 48, device="cuda", generator=gen) * 0.15
    c, vx, vw = (torch.randn(s, device="cuda", generator=gen) for s in ((20, 36), (20, 48), (72, 48)))
    for act in ("silu", "gelu", "gelu_tanh"):
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        dx, dw = torch.autograd.grad(gated_linear(a, b, act=act), (a, b), c)
        along = float((dx * vx).double().sum() + (dw * 0.1 * vw).double().sum())
        step = 1e-3
        f = lambda s: float((gated_linear(x + s * vx, w + s * 0.1 * vw, act=act).double() * c).sum())  # noqa: E731
        # 720 products of some 1 off by 2e-6 each, and the third derivative's term below 1e-3
        assert abs((f(step) - f(-step)) / (2 * step) - along) <= 720 ** 0.5 * 4e-6 / step + 2e-3 * abs(along) + 1e-2, act


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gated_linear_blocks_of_8_bits(dtype):
    """Blocks of zeros, of one large value among small ones, and of a width that ends inside one."""
    from pfeife_amd.layers import gated_linear

    D, ffn, n = 64, 40, 70
    x = torch.zeros(n, D, device="cuda")
    x[torch.arange(n), torch.arange(n) % D] = 1.0
    x[5] = 0
    w = torch.randn(2 * ffn, D, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    w[3], w[17] = 300.0, 0.0
    w[ffn:ffn + 16] = 0
    w[20:36] *= 2.0 ** -9
    x, w = x.to(dtype).requires_grad_(), w.to(dtype).requires_grad_()
    y = gated_linear(x, w, kept="8bit")
    up = torch.randn(n, ffn, device="cuda", generator=torch.Generator("cuda").manual_seed(4)).to(dtype)
    dx, dw = torch.autograd.grad(y, (x, w), up)
    gated_check(x.detach(), w.detach(), "silu", "8bit", up, y.detach(), dx, dw)


def test_gated_linear_layouts():
    from pfeife_amd.layers import gated_linear

    x, w = torch.randn(4, 9, 64, device="cuda").bfloat16(), torch.randn(96, 64, device="cuda").bfloat16()
    want = gated_linear(x, w)
    assert want.shape == (4, 9, 48)
    base = torch.zeros(x.numel() + 1, dtype=torch.bfloat16, device="cuda")
    moved = base[1:].view_as(x)
    moved.copy_(x)
    wbase = torch.zeros(w.numel() + 1, dtype=torch.bfloat16, device="cuda")
    wmoved = wbase[1:].view_as(w)
    wmoved.copy_(w)
    for a in (x.transpose(0, 1).contiguous().transpose(0, 1), x.transpose(1, 2).contiguous().transpose(1, 2), moved):
        assert torch.equal(gated_linear(a, w), want)
    assert torch.equal(gated_linear(x, wmoved), want) and torch.equal(gated_linear(x, w.t().contiguous().t()), want)
    assert gated_linear(x[:0], w).shape == (0, 9, 48) and torch.equal(gated_linear(x[0, 0], w), gated_linear(x[:1, :1], w)[0, 0])
    a, b = x[:0].clone().requires_grad_(), w.clone().requires_grad_()
    ga, gb = torch.autograd.grad(gated_linear(a, b).sum(), (a, b))
    assert ga.shape == a.shape and not gb.any()
    c = x.clone().requires_grad_()      # a gradient that comes expanded
    g1, = torch.autograd.grad(gated_linear(c, w).sum(), c)
    g2, = torch.autograd.grad(gated_linear(c, w), c, torch.ones_like(want))
    assert torch.equal(g1, g2)
