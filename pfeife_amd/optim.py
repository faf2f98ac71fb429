"""AdamW with moments of 8 bits: `PipeOption(optimizer=dict(type="adamw8bit", ...))`, or an optimizer of the user's own
like any of torch.optim (which is what the reference offers, pfeife/option.py:9-29).

A parameter of `min_8bit_size` elements or more keeps its moments as e4m3 codes with an fp32 scale to every 256 elements
(2.03 bytes a parameter instead of 8), a smaller one in fp32.  One launch (`pf_adam8_step`) updates all parameters of a group.
"""
import torch

from .hip import ADAM8_BLOCK


class AdamW8bit(torch.optim.Optimizer):
    """torch.optim.AdamW's update on fp32 parameters and gradients, with 8-bit moments.

    state[p] of a large parameter, in the order of p's storage: `exp_avg` and `exp_avg_sq_root` (float8_e4m3fn codes [n]; the second is the
    square root of AdamW's `exp_avg_sq`), `exp_avg_scale` and `exp_avg_sq_root_scale` (fp32 [ceil(n / 256)]); of a small one `exp_avg`
    and `exp_avg_sq` in fp32; both `step`.  Codes are rounded so that their mean is kept, by bits that the element, the parameter's
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
                raise RuntimeError("AdamW8bit: parameters are fp32 (got %s)" % p.dtype)

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)      # gives every state tensor the parameter's type, and may share the dict's tensors
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(ids, (p for g in self.param_groups for p in g["params"])):
            for key, value in state_dict["state"].get(i, {}).items():
                if torch.is_tensor(value):
                    self.state[p][key] = value.detach().clone() if key == "step" else value.detach().clone().to(p.device)

    def _init_state(self, p, group):
        st = self.state[p]
        if len(st) == 0:
            n = p.numel()
            st["step"] = torch.tensor(0.0, dtype=torch.float32)
            if n < max(1, group["min_8bit_size"]):
                st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
            else:
                for key in ("exp_avg", "exp_avg_sq_root"):
                    st[key] = torch.zeros(n, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn)
                    st[key + "_scale"] = torch.zeros(-(-n // ADAM8_BLOCK), dtype=torch.float32, device=p.device)
        return st

    @staticmethod
    def _check(p, st):
        """The operands as the kernel addresses them: (gradient, first moment, its scales, second moment, its scales)"""
        g = p.grad
        if p.device.type != "cuda":
            raise RuntimeError("AdamW8bit: the HIP step needs GPU parameters (got %s)" % p.device)
        if g.is_sparse or g.dtype != torch.float32 or g.device != p.device:
            raise RuntimeError("AdamW8bit: gradients are dense fp32 on the parameter's device (got %s %s on %s)" % (g.layout, g.dtype, g.device))
        if not torch.empty_like(p, device="meta").stride() == p.stride():
            raise RuntimeError("AdamW8bit: a parameter's elements have to lie in memory without gaps (strides %s)" % (p.stride(),))
        if g.stride() != p.stride():
            g = torch.empty_like(p).copy_(g)
        if "exp_avg_scale" in st:
            ops = [(st["exp_avg"], torch.float8_e4m3fn, p.numel()), (st["exp_avg_scale"], torch.float32, -(-p.numel() // ADAM8_BLOCK)),
                   (st["exp_avg_sq_root"], torch.float8_e4m3fn, p.numel()), (st["exp_avg_sq_root_scale"], torch.float32, -(-p.numel() // ADAM8_BLOCK))]
        else:
            ops = [(st["exp_avg"], torch.float32, p.numel()), None, (st["exp_avg_sq"], torch.float32, p.numel()), None]
        for op in ops:
            if op is not None and (op[0].dtype != op[1] or op[0].numel() != op[2] or op[0].device != p.device
                                   or op[0].dim() == 1 and not op[0].is_contiguous() or op[0].dim() > 1 and op[0].stride() != p.stride()):
                raise RuntimeError("AdamW8bit: the optimizer's state does not fit its parameter of shape %s" % (tuple(p.shape),))
        return (g,) + tuple(None if op is None else op[0] for op in ops)

    def _prepare(self, kernels):
        """[(group, states, table, items, chunks)] of what has a gradient, parameters at one step count together, and whether a table is new."""
        cache = self.__dict__.setdefault("_tables", {})
        work, fresh, place = [], False, 0
        for gi, group in enumerate(self.param_groups):
            by_step = {}
            for p in group["params"]:
                place += 1
                if p.grad is None or p.numel() == 0:
                    continue
                st = self._init_state(p, group)
                by_step.setdefault((float(st["step"]), p.device), []).append((p, st, place - 1))
            for n, (_, found) in enumerate(sorted(by_step.items(), key=lambda kv: (kv[0][0], str(kv[0][1])))):
                items = []
                for p, st, index in found:
                    g, m, ms, r, rs = self._check(p, st)
                    items.append((p.data, g, m, ms, r, rs, index))
                key = [(i[6], i[0].numel()) + tuple(None if t is None else t.data_ptr() for t in i[:6]) for i in items]
                ent = cache.get((gi, n))
                if ent is None or ent[0] != key:
                    fresh = True
                    ent = cache[gi, n] = (key, kernels.adam8_table(items))
                work.append((group, [st for _, st, _ in found], items, ent[1]))
        return work, fresh

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        first = next((p for g in self.param_groups for p in g["params"] if p.grad is not None), None)
        if first is None:
            return loss
        from .loss import _table

        if first.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW8bit: a step cannot be captured into a graph: its count would stay the same")
        kernels = _table(first, "AdamW8bit")
        for group, states, items, table in self._prepare(kernels)[0]:
            device = items[0][0].device
            with torch.cuda.device(device):
                self._launch(_table(items[0][0], "AdamW8bit"), group, states, table, torch.cuda.current_stream(device).cuda_stream)
        return loss

    @staticmethod
    def _launch(kernels, group, states, table, stream, scaler_state=None):
        """One launch; with a loss scaler's state the count of steps is the device's, and the states' entries are not touched."""
        b1, b2 = group["betas"]
        step = int(states[0]["step"]) + 1
        kernels.adam8_step(*table, float(group["lr"]), float(b1), float(b2), float(group["eps"]), float(group["weight_decay"]), step,
                           scaler_state, stream)
        if scaler_state is None:
            for st in states:
                st["step"] += 1
