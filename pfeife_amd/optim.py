"""AdamW with moments of 8 bits: `PipeOption(optimizer=dict(type="adamw8bit", ...))`, or an optimizer of the user's own
like any of torch.optim (which is what the reference offers, pfeife/option.py:9-29).

A parameter of `min_8bit_size` elements or more keeps its moments as e4m3 codes with an fp32 scale to every 256 elements
(2.03 bytes a parameter instead of 8), a smaller one in fp32.  One launch (`pf_adam8_step`) updates all parameters of a group.
"""
import torch

from .hip import ADAM8_BLOCK
from .loss import _raw_stream, _table


def _layout(p):
    """How a dense tensor's elements lie in memory: [(size, stride)] of its dimensions, those that follow one another taken as one."""
    runs = []
    for size, stride in zip(p.shape, p.stride()):
        if size > 1 and runs and runs[-1][1] == size * stride:
            runs[-1] = (runs[-1][0] * size, stride)
        elif size > 1:
            runs.append((size, stride))
    return runs or [(1, 1)]


class AdamW8bit(torch.optim.Optimizer):
    """torch.optim.AdamW's update on fp32 parameters and gradients, with 8-bit moments.

    state[p] of a large parameter, in the order of p's storage: `exp_avg` and `exp_avg_sq_root` (float8_e4m3fn codes [n]; the second is the
    square root of AdamW's `exp_avg_sq`), `exp_avg_scale` and `exp_avg_sq_root_scale` (fp32 [ceil(n / 256)]), `layout` (sizes and strides that
    order is of: a parameter that lies in memory otherwise is refused); of a small one `exp_avg` and `exp_avg_sq` in fp32; both `step`.  Codes are rounded so that their mean is kept, by bits that the element, the parameter's
    place in the optimizer and the step give: a run repeats itself."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, min_8bit_size=4096):
        for name, value, ok in (("lr", lr, lr >= 0.0), ("eps", eps, eps >= 0.0), ("weight_decay", weight_decay, weight_decay >= 0.0),
                                ("betas", betas, all(0.0 <= b < 1.0 for b in betas)), ("min_8bit_size", min_8bit_size, min_8bit_size >= 0)):
            if not ok:
                raise ValueError("AdamW8bit: bad %s: %s" % (name, value))
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, min_8bit_size=min_8bit_size))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dtype != torch.float32:
                self.param_groups.pop()
                raise RuntimeError("AdamW8bit: parameters are fp32 (got %s)" % p.dtype)

    def load_state_dict(self, state_dict):
        if any(g.get(name) for g in state_dict["param_groups"] for name in ("amsgrad", "maximize")):
            raise RuntimeError("AdamW8bit: state of an optimizer with amsgrad or maximize, of which there is neither here")
        super().load_state_dict(state_dict)      # gives every state tensor the parameter's type, and may share the dict's tensors
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(ids, (p for g in self.param_groups for p in g["params"])):
            for key, value in state_dict["state"].get(i, {}).items():
                if torch.is_tensor(value):
                    self.state[p][key] = value.detach().clone() if key in ("step", "layout") else value.detach().clone().to(p.device)
        # new state may lie where the old one did, and the old one's memory is wanted back
        for name in ("_seen", "_tables"):
            self.__dict__.pop(name, None)

    def _init_state(self, p, group):
        st = self.state[p]
        if len(st) == 0:
            n = p.numel()
            st["step"] = 0
            if n < max(1, group.get("min_8bit_size", self.defaults["min_8bit_size"])):
                st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
            else:
                st["layout"] = torch.tensor(_layout(p))
                for key in ("exp_avg", "exp_avg_sq_root"):
                    st[key] = torch.zeros(n, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn)
                    st[key + "_scale"] = torch.zeros(-(-n // ADAM8_BLOCK), dtype=torch.float32, device=p.device)
        return st

    @staticmethod
    def _operands(p, st):
        """(first moment, its scales, second moment, its scales)"""
        if "exp_avg_scale" in st:
            return st["exp_avg"], st["exp_avg_scale"], st["exp_avg_sq_root"], st["exp_avg_sq_root_scale"]
        return st["exp_avg"], None, st["exp_avg_sq"], None

    @staticmethod
    def _check_layout(p, st):
        """Codes are in the order of a parameter's storage: that has to be the one they were made in."""
        held, now = st.get("layout"), _layout(p)
        if held is None:      # (not noted: taken as the parameter's)
            st["layout"] = torch.tensor(now)
        elif [tuple(run) for run in held.tolist()] != now:
            raise RuntimeError("AdamW8bit: the optimizer's state does not fit its parameter of shape %s: its elements lie in memory by (size, stride) %s, "
                               "the moments' by %s" % (tuple(p.shape), now, held.tolist()))

    @staticmethod
    def _check(p, g, ops, st):
        """The gradient as the kernel addresses it; errors where it, the parameter or the state is not what the kernel takes."""
        if p.dtype != torch.float32 or g.shape != p.shape:
            raise RuntimeError("AdamW8bit: parameters are fp32, gradients of their shape (got %s %s and %s)" % (p.dtype, tuple(p.shape), tuple(g.shape)))
        if p.device.type != "cuda":
            raise RuntimeError("AdamW8bit: the HIP step needs GPU parameters (got %s)" % p.device)
        if g.dtype != torch.float32 or g.device != p.device:
            raise RuntimeError("AdamW8bit: gradients are dense fp32 on the parameter's device (got %s on %s)" % (g.dtype, g.device))
        if not p.is_contiguous() and torch.empty_like(p, device="meta").stride() != p.stride():
            raise RuntimeError("AdamW8bit: a parameter's elements have to lie in memory without gaps (strides %s)" % (p.stride(),))
        n = p.numel()
        if ops[1] is not None:
            fits = all(t.dtype == dtype and t.numel() == size and t.is_contiguous() and t.device == p.device for t, dtype, size in
                       zip(ops, (torch.float8_e4m3fn, torch.float32) * 2, (n, -(-n // ADAM8_BLOCK)) * 2))
        else:
            fits = all(t.dtype == torch.float32 and t.numel() == n and t.device == p.device and (t.stride() == p.stride() or t.dim() == 1 and t.is_contiguous())
                       for t in ops[::2])
        if not fits:
            raise RuntimeError("AdamW8bit: the optimizer's state does not fit its parameter of shape %s" % (tuple(p.shape),))
        if ops[1] is not None:
            AdamW8bit._check_layout(p, st)
        return g if g.stride() == p.stride() or g.is_contiguous() and p.is_contiguous() else torch.empty_like(p)     # (of another layout: copied for each step)

    @staticmethod
    def _check_apart(params):
        """One launch updates them all, in no order: none may be updated twice."""
        spans = sorted((p.data_ptr(), p.data_ptr() + 4 * p.numel()) for p, *_ in params)
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise RuntimeError("AdamW8bit: parameters share memory, or one is in a group twice")

    def _prepare(self, kernels):
        """[(group, states, device, table, copies)] of what has a gradient, parameters at one step count together, and whether a table
        is new.  A table holds addresses: it is made again when one of them is another, or the stream is.  Reads no gradient."""
        seen = self.__dict__.get("_seen")
        if seen is not None and self._as_seen(*seen[0]):
            return seen[1], False
        cache = self.__dict__.setdefault("_tables", {})
        work, fresh, place, records, plain = [], False, 0, [], True
        for gi, group in enumerate(self.param_groups):
            by_step = {}
            for p in group["params"]:
                place += 1
                g = p.grad
                if g is None or p.numel() == 0:
                    records.append((p, None, None, 0, 0, 0, ()))
                    continue
                if g.layout is not torch.strided:
                    raise RuntimeError("AdamW8bit: gradients are dense fp32 on the parameter's device (got %s)" % g.layout)
                st = self._init_state(p, group)
                key = (float(st["step"]), p.get_device())
                found = by_step.get(key)
                if found is None:
                    found = by_step[key] = ([], [], [])
                ops = self._operands(p, st)
                found[0].append(st)
                found[1].append((p, g, ops, place - 1))
                found[2].append((place, *[t if t is None else (t.data_ptr(), t.dtype, t.numel()) for t in (p, g, *ops)], g.stride(), p.stride()))
                keys = ("exp_avg", "exp_avg_scale", "exp_avg_sq_root", "exp_avg_sq_root_scale") if ops[1] is not None else ("exp_avg", "exp_avg_sq")
                records.append((p, st, found[0], p.data_ptr(), 4 * p.numel(), g.data_ptr(), [(k, st[k], st[k].data_ptr(), st[k].numel()) for k in keys]))
                plain = plain and p.is_contiguous() and g.is_contiguous()
            for n, key in enumerate(sorted(by_step)):
                states, params, now = by_step[key]
                now.append(_raw_stream(key[1]) if key[1] >= 0 else None)
                ent = cache.get((gi, n))
                if ent is None or ent[0] != now:
                    fresh = True
                    items = [(p.data, self._check(p, g, ops, st), *ops, index) for (p, g, ops, index), st in zip(params, states)]
                    self._check_apart(params)
                    copies = [(i[1], p) for (p, g, _, _), i in zip(params, items) if i[1] is not g]
                    ent = cache[gi, n] = (now, kernels.adam8_table(items), copies)
                work.append((group, states, params[0][0].device, *ent[1:]))
        devices = {w[2].index for w in work}
        # (one device, dense tensors: what _as_seen looks at says that all is as it was)
        self._seen = ((records, [(g, len(g["params"])) for g in self.param_groups], devices.pop(), work and _raw_stream(work[0][2].index)), work) \
            if plain and len(devices) == 1 else None
        return work, fresh

    def _as_seen(self, records, counts, device, stream):
        """Is every address where the last step's tables have it, and every count of steps still its group's?"""
        if len(counts) != len(self.param_groups) or any(g is not h or len(g["params"]) != n for g, (h, n) in zip(self.param_groups, counts)) or _raw_stream(device) != stream:
            return False
        at = iter(records)
        state = self.state
        for group in self.param_groups:
            for p in group["params"]:
                seen, st, first, where, size, g_where, held = next(at)
                g = p.grad
                if seen is not p:
                    return False
                if st is None:
                    if g is not None and p.numel():
                        return False
                    continue
                if (g is None or state.get(p) is not st or st["step"] != first[0]["step"] or p.data_ptr() != where or p.nbytes != size
                        or g.data_ptr() != g_where or g.nbytes != size or not p.is_contiguous() or not g.is_contiguous()):
                    return False
                for key, t, t_where, n in held:
                    if st.get(key) is not t or t.data_ptr() != t_where or t.numel() != n:
                        return False
        return True

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        first = next((p for g in self.param_groups for p in g["params"] if p.grad is not None), None)
        if first is None:
            return loss
        if first.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW8bit: a step cannot be captured into a graph: its count would stay the same")
        kernels = _table(first, "AdamW8bit")
        for group, states, device, table, copies in self._prepare(kernels)[0]:
            if device.index == torch.cuda.current_device():
                self._launch(kernels, group, states, table, copies, _raw_stream(device.index))
            else:
                with torch.cuda.device(device):
                    self._launch(kernels, group, states, table, copies, _raw_stream(device.index))
        return loss

    @staticmethod
    def _launch(kernels, group, states, table, copies, stream, scaler_state=None):
        """One launch, on the current stream; with a loss scaler's state the count of steps is the device's, and the states' entries are not
        touched."""
        for mine, p in copies:
            mine.copy_(p.grad)
        b1, b2 = group["betas"]
        step = int(states[0]["step"]) + 1
        kernels.adam8_step(*table, float(group["lr"]), float(b1), float(b2), float(group["eps"]), float(group["weight_decay"]), step,
                           scaler_state, stream)
        if scaler_state is None:
            for st in states:      # (a number: adding one to a hundred tensors takes longer than the launch)
                st["step"] = step
