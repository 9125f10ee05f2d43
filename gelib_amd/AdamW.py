"""AdamW over all parameters of a model in one launch or a few, complex matrices of SO3linear among them, moments in 32 or 8 bits.  No
counterpart in the reference, whose users take torch's."""
import torch

from gelib_amd.gelib_common import backend

BLOCK = 256   # parameters start at multiples of this many elements in the moment arrays (8 bits: the elements of one scale)


class AdamW(torch.optim.Optimizer):
    """m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2, p = p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps) for float32,
    bfloat16 and complex64 parameters on one GPU (complex: real and imaginary parts are elements of their own, as in torch).

    state_bits=32 keeps m and v in float32.  state_bits=8 keeps each in a byte, an exponent and three bits of the mantissa, with a scale
    for every 256 elements; these and bfloat16 parameters are rounded at random, so that steps far below a unit in the last place
    add up (to the nearest, v would not follow the gradients at all).  The random bits are a function of seed, step and element:
    runs repeat.  t counts the steps of each parameter; one whose gradient is None takes none.  (A step recorded into a graph is the step
    of that t at every replay, so one that rounds at random cannot be recorded: its bits would be the same ones every time.)"""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, seed=0):
        if state_bits not in (8, 32):
            raise ValueError("state_bits is 8 or 32")
        if not (lr >= 0 and eps >= 0 and weight_decay >= 0 and 0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError("lr, eps and weight_decay are not below zero, betas are from 0 to below 1")
        self.state_bits, self.seed = state_bits, int(seed) & 0xffffffffffffffff
        self._groups, self._places, self._size, self._arrays = [], {}, 0, None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        params = self.param_groups[-1]["params"]
        device = next((p.device for g in self.param_groups for p in g["params"]), torch.device("cuda"))
        try:
            for p in params:
                if p.dtype not in (torch.float32, torch.bfloat16, torch.complex64):
                    raise TypeError("parameters are float32, bfloat16 or complex64")
                if not p.is_cuda or p.device != device:
                    raise ValueError("parameters must be on one GPU: this step has no host form")
                if not p.is_contiguous() or p.is_conj() or p.is_neg():
                    raise ValueError("parameters are contiguous in memory")
        except (TypeError, ValueError):
            self.param_groups.pop()
            raise
        self._grow(self._place(params), device)

    def _place(self, params):
        """Gives the parameters of a further group their places behind the others; where the next ones would begin."""
        first, size = [], self._size
        for p in params:
            n = p.numel() * (2 if p.is_complex() else 1)
            self._places[p] = size, n
            first.append(size)
            size += -(-n // BLOCK) * BLOCK
        self._groups.append(backend().AdamWGroup(params, first))
        return size

    def _grow(self, size, device):
        of = [torch.float32] * 2 if self.state_bits == 32 else [torch.uint8] * 2 + [torch.int16] * 2
        lengths = [size] * 2 + [size // BLOCK] * 2
        new = [torch.zeros(n, dtype=t, device=device) for t, n in zip(of, lengths)]
        if self._arrays is not None:
            for a, b in zip(new, self._arrays):
                a[:b.numel()] = b
        self._arrays, self._size = new, size

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        m, v, *tops = self._arrays
        mt, vt = tops if tops else (None, None)
        for group, of in zip(self._groups, self.param_groups):
            b1, b2 = of["betas"]
            group.step(m, v, mt, vt, self.state_bits, of["lr"], b1, b2, of["eps"], of["weight_decay"], self.seed)
        return loss

    def moments(self, p=None):
        """(m, v) of parameter p, shaped like it (complex: with a last dimension of 2), or of all parameters as two long tensors in which
        every parameter starts at a multiple of 256 elements.  32 bits: the optimizer's own memory; 8 bits: what the codes stand
        for, in bfloat16, which holds it exactly."""
        if p is None:
            return tuple(self._arrays) if self.state_bits == 32 else backend().adamw_moments(*self._arrays)
        first, n = self._places[p]
        end = -(-(first + n) // BLOCK) * BLOCK
        if self.state_bits == 32:
            m, v = (t[first:end] for t in self._arrays)
        else:
            m, v = backend().adamw_moments(*[t[first:end] for t in self._arrays[:2]], *[t[first // BLOCK:end // BLOCK] for t in self._arrays[2:]])
        shape = p.shape + (2,) if p.is_complex() else p.shape
        return m[:n].view(shape), v[:n].view(shape)

    def set_moments(self, m, v, steps):
        """Sets the moments of all parameters from two tensors as moments() gives them (8 bits: to the nearest values, which are those
        themselves for what moments() gave) and the steps taken, one number or one a parameter in the order of the groups."""
        m, v = (t.to(device=self._arrays[0].device, dtype=torch.float32).contiguous() for t in (m, v))
        if m.shape != (self._size,) or v.shape != (self._size,):
            raise ValueError("m and v have %d elements each" % self._size)
        if isinstance(steps, int):
            steps = [steps] * len(self._places)
        if len(steps) != len(self._places) or min(steps, default=0) < 0:
            raise ValueError("as many steps as parameters are needed, none below zero")
        if self.state_bits == 32:
            self._arrays[0].copy_(m)
            self._arrays[1].copy_(v)
        else:
            backend().adamw_set_moments(*self._arrays, m, v)
        at = 0
        for group in self._groups:
            k = len(group.steps)
            group.steps = list(steps[at:at + k])
            at += k

    def __getstate__(self):   # (of copies and pickles; the groups that hold the places in memory are made again)
        return dict(super().__getstate__(), state_bits=self.state_bits, seed=self.seed, _arrays=self._arrays, steps=[list(g.steps) for g in self._groups])

    def __setstate__(self, state):
        state = dict(state)
        steps = state.pop("steps", None)
        super().__setstate__(state)
        if steps is None:         # (what Optimizer.load_state_dict sets: hyperparameters)
            return
        self._groups, self._places, self._size = [], {}, 0
        for group, k in zip(self.param_groups, steps):
            self._size = self._place(group["params"])
            self._groups[-1].steps = k

    def state_dict(self):
        d = super().state_dict()
        d["state"] = {"arrays": [t.clone() for t in self._arrays], "steps": [list(g.steps) for g in self._groups], "state_bits": self.state_bits,
                      "seed": self.seed}
        return d

    def load_state_dict(self, state_dict):
        s = state_dict["state"]
        if s["state_bits"] != self.state_bits or [len(k) for k in s["steps"]] != [len(g.steps) for g in self._groups] or [
                t.shape for t in s["arrays"]] != [t.shape for t in self._arrays]:
            raise ValueError("the state belongs to other parameters or to other state_bits")
        super().load_state_dict(dict(state_dict, state={}))
        for a, b in zip(self._arrays, s["arrays"]):
            a.copy_(b)
        for g, k in zip(self._groups, s["steps"]):
            g.steps = list(k)
        self.seed = s["seed"]
