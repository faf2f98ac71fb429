"""AdamW with 8-bit moments: against its formula step by step, bit by bit where the formula says so, and against 64 bits."""
import copy
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BLOCK = 256
SIZES = (1, 255, 256, 257, 1023, 1024, 1025, 4099, 70_001, 300_000)
LR, B1, B2, EPS = 1e-3, 0.9, 0.999, 1e-8


def mix(x):
    x = ((x ^ (x >> 16)) * 0x93D765DD) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x9E3779B1) & 0xFFFFFFFF
    return x ^ (x >> 16)


def dither(blocks, tensor, step):
    key = mix((torch.arange(blocks, device="cuda") + tensor * 0x9E3779B1) & 0xFFFFFFFF)
    key = mix((key + step * 0x93D765DD) & 0xFFFFFFFF)
    return mix((key.unsqueeze(1) + torch.arange(BLOCK, device="cuda") * 0x9E3779B1) & 0xFFFFFFFF)


def blocks_of(t):
    return torch.nn.functional.pad(t.reshape(-1), (0, -t.numel() % BLOCK)).view(-1, BLOCK)


def update(p, g, m, v, step, decay):
    """One rounding to an operation."""
    t = lambda x: torch.tensor(x, dtype=torch.float32, device="cuda")  # noqa: E731
    m = m + t(1 - B1) * (g - m)
    v = t(B2) * v + t(1 - B2) * (g * g)
    root = torch.sqrt(v)
    p = p * t(1 - LR * decay) - t(LR / (1 - B1 ** step)) * (m / (root / t(math.sqrt(1 - B2 ** step)) + t(EPS)))
    return p, m, v, root


def encode(x, bits, root):
    top = x.abs().amax(1, keepdim=True)
    keep = top >= 2.0 ** -100
    a = x.abs() * torch.where(keep, torch.full_like(top, 448.0) / top, torch.zeros_like(top))
    fine = a < 2.0 ** -6
    t = torch.where(fine, a + 2.0 ** -6, a)
    q = ((t.view(torch.int32).to(torch.int64) + (bits << 4)) & 0xFFF00000).to(torch.int32).view(torch.float32)
    q = torch.where(fine, q - 2.0 ** -6, q).clamp(max=448.0)
    if root:
        q = torch.where((x > 0) & keep, q.clamp(min=2.0 ** -9), q)
    return torch.copysign(q, x).to(torch.float8_e4m3fn), torch.where(keep, top / torch.full_like(top, 448.0), torch.zeros_like(top)).squeeze(1)


def expected(p, g, st, tensor, step, decay):
    """-> the parameter and the state after a step, from what they are before it"""
    if "exp_avg_scale" not in st:
        p, m, v, _ = update(p.reshape(-1), g.reshape(-1), st["exp_avg"].reshape(-1), st["exp_avg_sq"].reshape(-1), step, decay)
        return p, {"exp_avg": m, "exp_avg_sq": v}
    n = p.numel()
    m, r = (blocks_of(st[k].float()) * st[k + "_scale"].unsqueeze(1) for k in ("exp_avg", "exp_avg_sq_root"))
    new, m, _, r = update(blocks_of(p), blocks_of(g), m, r * r, step, decay)
    bits = dither(m.shape[0], tensor, step)
    valid = (torch.arange(m.numel(), device="cuda") < n).view(m.shape)
    m, r = torch.where(valid, m, 0.0), torch.where(valid, r, 0.0)
    (mq, ms), (rq, rs) = encode(m, bits >> 16, False), encode(r, bits & 0xFFFF, True)
    return new.reshape(-1)[:n], {"exp_avg": mq.view(torch.uint8).reshape(-1)[:n], "exp_avg_scale": ms, "exp_avg_sq_root": rq.view(torch.uint8).reshape(-1)[:n], "exp_avg_sq_root_scale": rs}


def raw(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


@pytest.mark.parametrize("decay,least", [(0.0, 0), (0.1, 1024), (0.1, 10 ** 9)])
def test_steps_are_the_formulas(decay, least):
    """Five steps, every bit of parameters, codes and scales; gradients over eight orders of magnitude with zeros, empty blocks and
    blocks below what a scale can hold."""
    from pfeife_amd.optim import AdamW8bit

    g = torch.Generator().manual_seed(1)
    params = [torch.nn.Parameter(torch.randn(n, generator=g).cuda()) for n in SIZES]
    opt = AdamW8bit(params, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=decay, min_8bit_size=least)
    for step in range(1, 6):
        before = []
        for k, p in enumerate(params):
            grad = (torch.randn(p.numel(), generator=g) * 10.0 ** torch.randint(-6, 3, (p.numel(),), generator=g)).cuda()
            grad[::7] = 0.0
            if p.numel() > 2000:
                grad[512:1024] = 0.0
                grad[1024:1536] *= 1e-35
            if k == 6 and step == 2:       # (no gradient: not this one's step)
                p.grad = None
            else:
                p.grad = grad
            before.append((p.detach().clone(), copy.deepcopy(opt.state.get(p, {})) if p in opt.state else {}))
        opt.step()
        torch.cuda.synchronize()
        for k, p in enumerate(params):
            old, st = before[k]
            if p.grad is None:
                assert torch.equal(p.detach(), old)
                continue
            own = opt.state[p]
            assert ("exp_avg_scale" in own) == (p.numel() >= max(1, least))
            if not st:
                st = {key: torch.zeros_like(t) for key, t in own.items() if key != "step"}
            count = step - 1 if k == 6 and step > 2 else step
            assert int(own["step"]) == count
            want_p, want = expected(old, p.grad, st, k, count, decay)
            assert torch.equal(p.detach(), want_p.view_as(p)), (step, k)
            for key, t in want.items():
                assert torch.equal(raw(own[key]).reshape(-1), t.reshape(-1)), (step, k, key)


def test_parameters_against_64_bits():
    """One step from warm moments: parameters within eight roundings of the formula's magnitudes."""
    from pfeife_amd.optim import AdamW8bit

    g = torch.Generator().manual_seed(2)
    n = 100_003
    p = torch.nn.Parameter(torch.randn(n, generator=g).cuda())
    opt = AdamW8bit([p], lr=LR, betas=(B1, B2), eps=EPS, weight_decay=0.1)
    for _ in range(3):
        p.grad = torch.randn(n, generator=g).cuda()
        opt.step()
    old = p.detach().double()
    st = opt.state[p]
    m, r = (((blocks_of(st[k].float()).double() * st[k + "_scale"].double().unsqueeze(1)).reshape(-1)[:n]) for k in ("exp_avg", "exp_avg_sq_root"))
    p.grad = torch.randn(n, generator=g).cuda()
    gd = p.grad.double()
    opt.step()
    new_m, v = B1 * m + (1 - B1) * gd, B2 * r * r + (1 - B2) * gd * gd
    move = LR / (1 - B1 ** 4) / (v.sqrt() / math.sqrt(1 - B2 ** 4) + EPS)
    want = old * (1 - LR * 0.1) - move * new_m
    tol = 8 * 2.0 ** -24 * (old.abs() + move * (m.abs() + gd.abs()))
    assert ((p.detach().double() - want).abs() <= tol).all()
    # and what is held is within a code's step of the moment: 2^-3 of the value, or the grid's least step
    for key, x in (("exp_avg", new_m), ("exp_avg_sq_root", v.sqrt())):
        held = (blocks_of(st[key].float()).double() * st[key + "_scale"].double().unsqueeze(1)).reshape(-1)[:n]
        unit = st[key + "_scale"].double().repeat_interleave(BLOCK)[:n]
        assert ((held - x).abs() <= 0.1251 * x.abs() + 2.0 ** -9 * 1.0001 * unit).all()


def test_rounding_keeps_the_mean():
    """A gradient that stays gives a second moment that comes to its square, though beta2 moves it by a sixtieth of half a code a
    step; and one that ends lets it go.  The mean over 65536 elements after 2000 steps: an element's root is off by the codes' noise, at most
    2^-4 of it (half the widest step, times two for its memory of 1 / (1 - beta2) steps), the mean of so many by 2^-8 of that; the square's mean is
    above by the noise's square, 2^-8."""
    from pfeife_amd.optim import AdamW8bit

    p = torch.nn.Parameter(torch.zeros(65536, device="cuda"))
    opt = AdamW8bit([p], lr=0.0, betas=(B1, B2), weight_decay=0.0)
    p.grad = torch.linspace(0.5, 1.0, p.numel(), device="cuda")
    root = lambda: blocks_of(opt.state[p]["exp_avg_sq_root"].float()) * opt.state[p]["exp_avg_sq_root_scale"].unsqueeze(1)  # noqa: E731
    for _ in range(2000):
        opt.step()
    share = float((root().reshape(-1) / p.grad).mean())
    assert abs(share - math.sqrt(1 - B2 ** 2000)) <= 2.0 ** -6, share
    p.grad = torch.zeros_like(p)
    for _ in range(1000):
        opt.step()
    share = float((root().reshape(-1) / torch.linspace(0.5, 1.0, p.numel(), device="cuda")).mean())
    assert abs(share - math.sqrt((1 - B2 ** 2000) * B2 ** 1000)) <= 2.0 ** -6, share


def test_not_finite_gradients_show():
    from pfeife_amd.optim import AdamW8bit

    for bad in (math.nan, math.inf, -math.inf):
        p = torch.nn.Parameter(torch.zeros(5000, device="cuda"))
        opt = AdamW8bit([p], lr=LR)
        p.grad = torch.ones_like(p)
        p.grad[300] = bad
        opt.step()
        p.grad = torch.ones_like(p)
        opt.step()
        hit = torch.zeros(5000, dtype=torch.bool, device="cuda")
        hit[256:512] = True
        assert p[hit].isnan().all() and torch.isfinite(p[~hit]).all()


def test_neighbours_stay_as_they_are():
    """Parameters that are pieces of one buffer at odd places, a gradient of another layout."""
    from pfeife_amd.optim import AdamW8bit

    g = torch.Generator().manual_seed(3)
    room = torch.full((40_000,), 7.0, device="cuda")
    spots = [(1, 4097), (5003, 33), (6002, 20_001)]
    params = [torch.nn.Parameter(room[a:a + n]) for a, n in spots]
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    chan = torch.nn.Parameter(torch.randn(16, 8, 8, 8, generator=g).cuda().to(memory_format=torch.channels_last))
    flat = torch.nn.Parameter(chan.detach().permute(0, 2, 3, 1).contiguous())
    a, b = AdamW8bit([*params, chan], lr=LR), AdamW8bit([*twins, flat], lr=LR)
    for _ in range(3):
        grads = torch.randn(40_000, generator=g).cuda()
        for p, q, (at, n) in zip(params, twins, spots):
            p.grad, q.grad = grads[at + 1:at + 1 + n], grads[at + 1:at + 1 + n].clone()
        chan.grad = torch.randn(16, 8, 8, 8, generator=g).cuda()
        flat.grad = chan.grad.permute(0, 2, 3, 1).contiguous()
        a.step(), b.step()
    assert all(torch.equal(p, q) for p, q in zip(params, twins)) and torch.equal(chan.permute(0, 2, 3, 1), flat)
    mask = torch.ones(40_000, dtype=torch.bool, device="cuda")
    for at, n in spots:
        mask[at:at + n] = False
    assert (room[mask] == 7).all()


def test_state_dict_round_trip():
    """A resumed optimizer takes the same steps, bit for bit: codes keep their type."""
    from pfeife_amd.optim import AdamW8bit

    g = torch.Generator().manual_seed(4)
    params = [torch.nn.Parameter(torch.randn(n, generator=g).cuda()) for n in (5000, 300)]
    opt = AdamW8bit(params, lr=LR)

    def steps(ps, o, grads):
        for gs in grads:
            for p, x in zip(ps, gs):
                p.grad = x.clone()
            o.step()

    grads = [[torch.randn(p.numel(), generator=g).cuda() for p in params] for _ in range(4)]
    steps(params, opt, grads[:2])
    saved = copy.deepcopy(opt.state_dict())
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = AdamW8bit(twins, lr=123.0)
    other.load_state_dict(saved)
    assert other.state[twins[0]]["exp_avg"].dtype == torch.float8_e4m3fn and other.param_groups[0]["lr"] == LR
    steps(params, opt, grads[2:])
    steps(twins, other, grads[2:])
    assert all(torch.equal(p, q) for p, q in zip(params, twins))
    assert all(torch.equal(raw(opt.state[p][k]), raw(other.state[q][k])) for p, q in zip(params, twins) for k in opt.state[p] if k != "step")
    assert all(opt.state[p]["step"] == other.state[q]["step"] == 4 for p, q in zip(params, twins))
    other.state[twins[0]]["exp_avg"] = other.state[twins[0]]["exp_avg"][:-1]
    with pytest.raises(RuntimeError, match="does not fit"):
        other.step()


def test_a_capture_is_refused():
    from pfeife_amd.optim import AdamW8bit

    p = torch.nn.Parameter(torch.zeros(5000, device="cuda"))
    p.grad = torch.ones_like(p)
    opt = AdamW8bit([p])
    opt.step()
    x = torch.zeros(4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(RuntimeError, match="cannot be captured"):
            opt.step()
    graph.replay()
    torch.cuda.synchronize()
    assert int(opt.state[p]["step"]) == 1


def test_many_tensors_in_two_groups():
    """More tensors than a wavefront has lanes, two learning rates, an empty tensor; each tensor as in an optimizer with itself at the same place."""
    from pfeife_amd.optim import AdamW8bit

    g = torch.Generator().manual_seed(5)
    sizes = [1 + 37 * k % 6000 for k in range(150)] + [0]
    params = [torch.nn.Parameter(torch.randn(n, generator=g).cuda()) for n in sizes]
    start = [p.detach().clone() for p in params]
    opt = AdamW8bit([{"params": params[:70]}, {"params": params[70:], "lr": 1e-2, "min_8bit_size": 0}], lr=LR)
    for _ in range(2):
        for p in params:
            p.grad = torch.ones_like(p) * 0.1
        opt.step()
    for k, (p, old) in enumerate(zip(params, start)):
        if not p.numel():
            continue
        lr = LR if k < 70 else 1e-2
        # both gradients are the same: every step moves by lr m^ / (root^ + eps), within a code's step of lr each
        moved = old * (1 - lr * 1e-2) ** 2 - p.detach()
        assert ((moved - 2 * lr).abs() <= 2 * lr * 0.13 + 4 * 2.0 ** -24 * old.abs()).all(), k
        assert ("exp_avg_scale" in opt.state[p]) == (k >= 70 or p.numel() >= 4096)


def test_what_changes_between_steps_is_seen():
    """Gradients that come and go or move, state that is replaced, a parameter that is given other memory, a group that is added, another
    stream: always the step that an optimizer made anew from the same state takes."""
    from pfeife_amd.optim import AdamW8bit

    g = torch.Generator().manual_seed(6)
    params = [torch.nn.Parameter(torch.randn(n, generator=g).cuda()) for n in (5000, 300, 9000)]
    opt = AdamW8bit(params, lr=LR)
    side = torch.cuda.Stream()
    late = torch.nn.Parameter(torch.randn(6000, generator=g).cuda())

    def both(stream=None):
        torch.cuda.synchronize()
        twins = [[torch.nn.Parameter(p.detach().clone()) for p in grp["params"]] for grp in opt.param_groups]
        other = AdamW8bit([{"params": t} for t in twins], lr=LR)
        other.load_state_dict(opt.state_dict())
        for grp, t in zip(opt.param_groups, twins):
            for p, q in zip(grp["params"], t):
                q.grad = None if p.grad is None else p.grad.clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            opt.step()
        torch.cuda.synchronize()
        other.step()
        for grp, t in zip(opt.param_groups, twins):
            for p, q in zip(grp["params"], t):
                assert torch.equal(p, q)
                for key, v in opt.state.get(p, {}).items():
                    w = other.state[q][key]
                    assert torch.equal(raw(v), raw(w)) if torch.is_tensor(v) and torch.is_tensor(w) else float(v) == float(w), key

    rnd = lambda p: torch.randn(p.shape, generator=g).cuda()  # noqa: E731
    for p in params:
        p.grad = rnd(p)
    both()
    both()
    params[0].grad.mul_(0.5)
    both()
    params[1].grad = None
    both()
    params[1].grad = rnd(params[1])      # one step behind the others from here on
    both()
    both()
    params[2].grad = rnd(params[2])
    both()
    opt.state[params[0]]["exp_avg"] = opt.state[params[0]]["exp_avg"].clone()
    both()
    params[2].data = rnd(params[2])
    both()
    both(side)
    both(side)
    both()
    opt.add_param_group({"params": [late]})
    both()
    late.grad = rnd(late)
    both()
    both()
    late.grad = rnd(late).view(2, 3000).t().reshape(-1)[:6000].view(3000, 2).t().reshape(-1)
    both()
    opt.load_state_dict(copy.deepcopy(opt.state_dict()))
    both()
    both()


@pytest.mark.filterwarnings("ignore:.*duplicate parameters")
def test_what_one_launch_cannot_update_is_refused():
    """Parameters that share memory (in one launch, so in no order), one that is listed twice, a sparse gradient: nothing is changed."""
    from pfeife_amd.optim import AdamW8bit

    room = torch.randn(12_000, generator=torch.Generator().manual_seed(7)).cuda()
    start = room.clone()
    one = torch.nn.Parameter(room[:5000])
    for params in ([one, one], [one, torch.nn.Parameter(room[:5000])], [torch.nn.Parameter(room[4999:9000]), one], [one, torch.nn.Parameter(room[100:101])]):
        for p in params:
            p.grad = torch.ones_like(p)
        opt = AdamW8bit(params, lr=LR)
        for _ in range(2):
            with pytest.raises(RuntimeError, match="share memory"):
                opt.step()
    sparse = torch.nn.Parameter(room[6000:].view(100, 60))
    sparse.grad = torch.ones(100, 60, device="cuda").to_sparse()
    with pytest.raises(RuntimeError, match="dense"):
        AdamW8bit([sparse], lr=LR).step()
    torch.cuda.synchronize()
    assert torch.equal(room, start)
    # neighbours are fine, and so are groups, whose launches follow one another
    opt = AdamW8bit([{"params": [one, torch.nn.Parameter(room[5000:9000])]}, {"params": [torch.nn.Parameter(room[:5000])]}], lr=LR)
    for p in (p for grp in opt.param_groups for p in grp["params"]):
        p.grad = torch.ones_like(p)
    opt.step()
    assert not torch.equal(room[:9000], start[:9000]) and torch.equal(room[9000:], start[9000:])


@pytest.mark.parametrize("layout", [torch.contiguous_format, torch.channels_last])
def test_loaded_state_is_new(layout):
    """Also where its memory is the old state's, which is given back: a loss scaler's count of steps starts from what was loaded."""
    import weakref

    from pfeife_amd.loss import _table
    from pfeife_amd.optim import AdamW8bit

    p = torch.nn.Parameter(torch.randn(16, 8, 8, 8, generator=torch.Generator().manual_seed(8)).cuda().to(memory_format=layout))
    p.grad = torch.ones_like(p)
    opt = AdamW8bit([p], lr=LR)
    opt.step()
    kernels = _table(p, "")
    assert not opt._prepare(kernels)[1]
    saved = copy.deepcopy(opt.state_dict())
    old = weakref.ref(opt.state[p]["exp_avg"])
    opt.load_state_dict(saved)
    assert old() is None and opt._prepare(kernels)[1] and not opt._prepare(kernels)[1]
    opt.step()
    assert opt.state[p]["step"] == 2
