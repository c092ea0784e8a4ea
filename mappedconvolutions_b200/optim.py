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
            by_device, masters = {}, group["master_weights"]
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                state = self.state[p]
                if not state:
                    state.update(self._new_state(p, group))
                elif masters and p.dtype == torch.bfloat16 and "master" not in state:  # (a state of torch's)
                    state["master"] = p.detach().to(torch.float32, copy=True)
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
        """torch's, but a state is kept as its parameter needs it: moments float32 (float64 for float64 parameters) in the
        parameter's order of memory, or 8-bit codes as they are.  A state of torch.optim.AdamW leaves this optimiser's state_bits and
        master_weights in place and takes their form; one that cannot go on the same way is refused before anything changes."""
        loaded = state_dict["param_groups"]
        for group in loaded:
            self._check_options(group)
            if group["weight_decay"] and not group.get("decoupled_weight_decay", True):
                raise ValueError("a state whose weight decay goes through the moments is not supported")
        kept = ("state_bits", "master_weights")
        groups = [{**{k: mine[k] for k in kept}, **group} for mine, group in zip(self.param_groups, loaded)]
        states = {}
        if [len(g["params"]) for g in groups] == [len(g["params"]) for g in self.param_groups]:  # (else torch's own refuses it)
            for mine, group, given in zip(self.param_groups, groups, loaded):
                bits = 32 if "state_bits" in given else group["state_bits"]
                for p, i in zip(mine["params"], group["params"]):
                    if state_dict["state"].get(i):
                        states[p] = self._state_for(p, state_dict["state"][i], bits)
        super().load_state_dict({**state_dict, "param_groups": groups + list(loaded[len(groups):])})
        self.state.update(states)

    @staticmethod
    def _state_for(p, given, bits):
        """`given` as the state of p; bits 8: moments that are values become codes"""
        missing = [k for k in ("step", "exp_avg", "exp_avg_sq") if k not in given]
        if missing:
            raise ValueError("a state of AdamW has %s" % ", ".join(missing))
        state = {k: v.detach().to(p.device, copy=True) if isinstance(v, torch.Tensor) else v for k, v in given.items()}
        coded = state["exp_avg"].dtype == torch.int8
        for k in ("exp_avg", "exp_avg_sq", "master"):
            v = state.get(k)
            if v is None:
                continue
            if v.shape != p.shape:
                raise ValueError("%s has shape %s, its parameter %s" % (k, tuple(v.shape), tuple(p.shape)))
            if k == "master" and p.dtype != torch.bfloat16:
                raise ValueError("only bfloat16 parameters have master weights, not %s" % p.dtype)
            if coded and k != "master":
                if p.dtype == torch.float64 or v.dtype != (torch.int8 if k == "exp_avg" else torch.uint8) or \
                        any(n > 1 and a != b for n, a, b in zip(p.shape, p.stride(), v.stride())) or \
                        k + "_scale" not in state or tuple(state[k + "_scale"].shape) != ((p.numel() + 255) // 256,):
                    raise ValueError("moments in 8 bits belong to float32 or bfloat16 parameters that lie as they do, with a scale for 256 elements")
            else:
                wide = torch.float64 if p.dtype == torch.float64 else torch.float32
                state[k] = torch.empty_like(p, dtype=wide, requires_grad=False).copy_(v)
        if bits == 8 and not coded and p.dtype != torch.float64:
            state.update(_codes(state["exp_avg"], state["exp_avg_sq"]))
        return state


def _codes(m, v):
    """The 8-bit form of float32 moments (see mc_adamw_step), the operations of float32 one by one."""
    def blocks(t):  # as they lie in memory
        t = t.as_strided((t.numel(),), (1,))
        return torch.nn.functional.pad(t, (0, -t.numel() % 256)).view(-1, 256)

    def scale(largest, codes):
        s = largest * torch.tensor(1 / codes, dtype=torch.float32, device=largest.device)
        s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
        return s, torch.where(s == 0, torch.zeros_like(s), 1 / s)

    def put(c, like, dtype):
        out = torch.empty_like(like, dtype=dtype)
        out.as_strided((like.numel(),), (1,)).copy_(c.reshape(-1)[:like.numel()])
        return out
    a, r = blocks(m), torch.sqrt(blocks(v))
    s, inverse = scale(a.abs().amax(1, keepdim=True), 127.0 ** 2)
    c = torch.copysign(torch.sqrt(a.abs() * inverse).round().clamp(max=127), a).nan_to_num(0.0)
    q, inverse = scale(r.amax(1, keepdim=True), 255.0 ** 2)
    d = torch.sqrt(r * inverse).round().clamp(max=255)
    d = torch.where((r > 0) & (q > 0), d.clamp(min=1), d).nan_to_num(0.0)  # (a v that is not zero keeps a code that is not zero)
    return dict(exp_avg=put(c, m, torch.int8), exp_avg_scale=s[:, 0].contiguous(), exp_avg_sq=put(d, v, torch.uint8),
                exp_avg_sq_scale=q[:, 0].contiguous())
