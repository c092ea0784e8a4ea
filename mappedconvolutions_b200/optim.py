"""Optimisers on the library's kernels.  Not in the reference, which trains with torch's."""
import torch

from .host import impl


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW (decoupled weight decay) with one kernel over all parameters of a group.

    state_bits: 32, moments in float32 (float64 for float64 parameters), or 8, moments as 8-bit codes with a float32 scale for
    256 elements each: 2 bytes per element instead of 8.  master_weights: bfloat16 parameters keep a float32 copy that the steps
    are taken on, so that a value written into such a parameter between steps lasts until the next one.  Parameters are float32, bfloat16 or float64 CUDA tensors, each dense in any order of its dimensions.

    state[p]: "step" (a number), "exp_avg" and "exp_avg_sq" - with 8 bits int8 and uint8 codes, "exp_avg_scale" and
    "exp_avg_sq_scale" -, and "master" where there is one.  moments() gives the values.  Step counts are kept on the host: a step
    cannot be captured into a CUDA graph.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, master_weights=False):
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      master_weights=bool(master_weights)))

    def add_param_group(self, param_group):
        self._check_options({**self.defaults, **param_group})
        super().add_param_group(param_group)

    @staticmethod
    def _check_options(group):
        for name in ("lr", "eps", "weight_decay"):
            if not group[name] >= 0:
                raise ValueError("%s must not be negative: %r" % (name, group[name]))
        if len(group["betas"]) != 2 or not all(0 <= b < 1 for b in group["betas"]):
            raise ValueError("betas must be two numbers in [0, 1): %r" % (group["betas"],))
        if group.get("state_bits", 32) not in (8, 32):
            raise ValueError("state_bits must be 8 or 32: %r" % (group["state_bits"],))
        for name in ("amsgrad", "maximize"):
            if group.get(name):
                raise ValueError("%s is not supported" % name)

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:  # (of a torch.optim.AdamW, say)
            group.setdefault("state_bits", 32)
            group.setdefault("master_weights", False)

    @staticmethod
    def _new_state(p, group):
        state = {"step": 0}
        if group["state_bits"] == 8 and p.dtype != torch.float64:
            scales = (p.numel() + 255) // 256
            state["exp_avg"] = torch.zeros_like(p, dtype=torch.int8)
            state["exp_avg_scale"] = torch.zeros(scales, dtype=torch.float32, device=p.device)
            state["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.uint8)
            state["exp_avg_sq_scale"] = torch.zeros(scales, dtype=torch.float32, device=p.device)
        else:
            wide = torch.float64 if p.dtype == torch.float64 else torch.float32
            state["exp_avg"] = torch.zeros_like(p, dtype=wide)
            state["exp_avg_sq"] = torch.zeros_like(p, dtype=wide)
        if group["master_weights"] and p.dtype == torch.bfloat16:
            state["master"] = p.detach().to(torch.float32, copy=True)
        return state

    def step(self, closure=None):
        """One step over all parameters that have a gradient; the others, and their step counts, stay as they are."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a step counts on the host and cannot be captured into a CUDA graph")
        for group in self.param_groups:
            by_device = {}
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                state = self.state[p]
                if not state:
                    state.update(self._new_state(p, group))
                lists = by_device.get(p.device)
                if lists is None:
                    lists = by_device[p.device] = ([], [], [], [], [], [], [], [], [])
                get = state.get
                for column, value in zip(lists, (p, g, state["exp_avg"], state["exp_avg_sq"], get("exp_avg_scale"),
                                                 get("exp_avg_sq_scale"), get("master"), int(state["step"]) + 1, state)):
                    column.append(value)
            for *lists, states in by_device.values():
                impl.adamw_step(*lists, float(group["lr"]), float(group["betas"][0]), float(group["betas"][1]), float(group["eps"]),
                                float(group["weight_decay"]))
                for s, n in zip(states, lists[-1]):
                    s["step"] = n
        return loss

    def moments(self):
        """(exp_avg, exp_avg_sq) of every parameter that has taken a step, in the groups' order: the state's own tensors, or the
        float32 values that 8-bit codes stand for."""
        states = [self.state[p] for group in self.param_groups for p in group["params"] if self.state.get(p)]
        out = [(s["exp_avg"], s["exp_avg_sq"]) for s in states]
        by_device = {}
        for i, s in enumerate(states):
            if "exp_avg_scale" in s:
                by_device.setdefault(s["exp_avg"].device, []).append(i)
        for members in by_device.values():
            values = impl.adamw_moments(*[[states[i][k] for i in members]
                                          for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")])
            for i, m, v in zip(members, *values):
                out[i] = (m, v)
        return out

    def load_state_dict(self, state_dict):
        """torch's, but every tensor of the state keeps its own type (torch would cast moments to the parameter's)."""
        for group in state_dict["param_groups"]:
            self._check_options(group)
        super().load_state_dict(state_dict)
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        for i, p in zip(ids, params):
            kept = state_dict["state"].get(i)
            if kept:
                self.state[p] = {k: v.detach().to(p.device, copy=True) if isinstance(v, torch.Tensor) else v
                                 for k, v in kept.items()}
