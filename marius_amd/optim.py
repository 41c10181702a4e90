"""AdamW over all parameters of a model in one launch (marius_adamw_step), beside the dense Adagrad / Adam steps of marius_amd.hip."""
import torch

from . import hip as H


class AdamW:
    """AdamW with decoupled weight decay over device tensors, their states in 32 bits or in 8 (state_bits=8: e4m3 codes and a float32 scale for every 256 elements, the
    second moment as its root; 2 instead of 8 bytes a parameter).  step() takes the gradients from `.grad`; a parameter without one is left as it is and its count of steps,
    which its bias correction goes by, stays.  capturable=True: the counts live on the device and step() may be captured into a graph and replayed (the gradients then are the
    captured tensors)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, capturable=False):
        self.params = [p for p in params]
        if state_bits not in (32, 8):
            raise H.MariusHipError("AdamW: states are held in 32 or in 8 bits")
        if not self.params:
            raise H.MariusHipError("AdamW: no parameters")
        self.lr, self.betas, self.eps, self.weight_decay, self.state_bits, self.capturable = lr, tuple(betas), eps, weight_decay, state_bits, capturable
        kind = torch.float32 if state_bits == 32 else torch.float8_e4m3fn
        self.exp_avg, self.exp_avg_sq = ([torch.zeros(p.shape, dtype=torch.float32, device=p.device).to(kind) for p in self.params] for _ in range(2))
        blocks = lambda p: torch.zeros(-(-p.numel() // H.ADAMW_BLOCK), dtype=torch.float32, device=p.device)  # noqa: E731
        self.exp_avg_scale, self.exp_avg_sq_scale = (None if state_bits == 32 else [blocks(p) for p in self.params] for _ in range(2))
        groups = {}
        for i, p in enumerate(self.params):
            groups.setdefault((p.device, p.dtype), []).append(i)
        of = lambda ts, at: None if ts is None else [ts[i] for i in at]  # noqa: E731
        self._groups = [(at, H.AdamWTensors(of(self.params, at), of(self.exp_avg, at), of(self.exp_avg_sq, at), of(self.exp_avg_scale, at), of(self.exp_avg_sq_scale, at)))
                        for at in groups.values()]
        self._steps = [0] * len(self.params)
        self._steps_dev = [torch.zeros(len(at), dtype=torch.int64, device=tensors.device) for at, tensors in self._groups] if capturable else None

    @property
    def steps(self):
        """how many steps every parameter has taken (capturable: read back from the device)"""
        if not self.capturable:
            return list(self._steps)
        steps = [0] * len(self.params)
        for (at, _), counts in zip(self._groups, self._steps_dev):
            for i, n in zip(at, counts.tolist()):
                steps[i] = n
        return steps

    @property
    def num_steps(self):
        """the steps of the parameter that has taken the most"""
        return max(self.steps)

    def zero_grad(self):
        for p in self.params:
            p.grad = None

    @torch.no_grad()
    def step(self, grad_scale=None):
        """one step; grad_scale: float32 device tensor of one element that multiplies every gradient (a clipping factor, the inverse of a loss scale).  A step that is
        refused does not count and leaves every parameter and state as it was."""
        calls = []
        for k, (at, tensors) in enumerate(self._groups):
            grads = [self.params[i].grad for i in at]
            # a call takes gradients of one type and, on the host, one number of steps: one call a group in most programs
            which = [None if g is None else (g.dtype, 0 if self.capturable else self._steps[i]) for i, g in zip(at, grads)]
            for one in dict.fromkeys(w for w in which if w is not None):
                calls.append((tensors, [g if w == one else None for g, w in zip(grads, which)], self._steps_dev[k] if self.capturable else one[1] + 1,
                              self.lr, *self.betas, self.eps, self.weight_decay, grad_scale))
        if self.capturable or len(calls) > 1:  # (a single call checks itself before it launches)
            for call in calls:
                H.adamw_check(*call)
        if self.capturable:
            for (at, _), counts in zip(self._groups, self._steps_dev):
                stepped = [n for n, i in enumerate(at) if self.params[i].grad is not None]
                if len(stepped) == len(at):
                    counts.add_(1)
                elif stepped:
                    torch._foreach_add_([counts[n] for n in stepped], 1)
        for call in calls:
            H.adamw_step(*call)
        if not self.capturable:
            for i, p in enumerate(self.params):
                self._steps[i] += p.grad is not None

    def state_dict(self):
        steps = self.steps
        return {"num_steps": max(steps), "steps": steps, "state_bits": self.state_bits, "lr": self.lr, "betas": self.betas, "eps": self.eps, "weight_decay": self.weight_decay,
                "exp_avg": self.exp_avg, "exp_avg_sq": self.exp_avg_sq, "exp_avg_scale": self.exp_avg_scale, "exp_avg_sq_scale": self.exp_avg_sq_scale}

    def load_state_dict(self, state):
        if state["state_bits"] != self.state_bits or [t.shape for t in state["exp_avg"]] != [t.shape for t in self.exp_avg]:
            raise H.MariusHipError("AdamW: the state is of other parameters, or held in other bits")
        self.lr, self.betas, self.eps, self.weight_decay = state["lr"], tuple(state["betas"]), state["eps"], state["weight_decay"]
        self._steps = list(state.get("steps") or [state["num_steps"]] * len(self.params))  # (a state without counts of its own: one for all)
        for name in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"):
            for mine, theirs in zip(getattr(self, name) or [], state[name] or []):
                mine.copy_(theirs)
        for (at, _), counts in zip(self._groups, self._steps_dev or []):
            counts.copy_(torch.tensor([self._steps[i] for i in at], dtype=torch.int64))
