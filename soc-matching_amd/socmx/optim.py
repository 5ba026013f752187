"""AdamW over many tensors on the GPU, with states in 32 or in 8 bits (csrc/socmx_adamw.hip).

Beside the fused Adam of the training iteration (`socmx_adam_step_f32`: one flat float32 gradient, the reference's rule without
weight decay): decoupled weight decay, tensors wherever they lie, weights in 16 bits with float32 masters, and states of one byte each.
`make_optimizer(weight_decay=..., state_bits=...)` (socmx/train.py) and main.py's optim.weight_decay / optim.state_bits use it.
"""
import torch

from . import _lib
from ._lib import SocmxError

BLOCK = 256          # elements that share the two scales of 8-bit states


def scale_rows(n):
    """Rows of the (rows, 2) scales of a tensor of `n` elements with 8-bit states."""
    return -(-n // BLOCK)


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, steps, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, scales=None,
               masters=None):
    """One AdamW update of every tensor, in place:

        m = b1 m + (1-b1) g,  v = b2 v + (1-b2) g^2,  p = p (1 - lr wd) - lr / (1-b1^t) m / (sqrt(v) / sqrt(1-b2^t) + eps)

    params, grads: lists of dense tensors of ONE type (float32, bfloat16 or float16) on one GPU, contiguous or, with all that belongs to a
    parameter, of one other order of dimensions in memory.  exp_avgs, exp_avg_sqs: float32 tensors of the same sizes; with `scales`, 8-bit states: int8 and uint8 codes and a float32 (ceil(n / 256), 2) for each tensor of n
    elements (zeros are states of zero; `adamw_state_values` decodes).  masters: float32 weights the update works on, the 16-bit
    weights getting their rounding.  steps: (len(params),) float32 on the GPU, or a list of tensors of one float32 each: the updates so
    far, advanced here -- a captured call counts its replays.  No two tensors may share memory, but gradients among themselves; a
    tensor may be empty."""
    if torch.is_tensor(lr):
        raise SocmxError("adamw_step: lr is a number, got a tensor")
    binding = _lib.torch_binding()
    call = binding.adamw_step if torch.is_tensor(steps) else binding.adamw_step_counts
    call(params, grads, exp_avgs, exp_avg_sqs, steps, lr, betas[0], betas[1], eps, weight_decay, scales, masters)


def adamw_state_values(exp_avgs, exp_avg_sqs, scales):
    """The values 8-bit states stand for: two lists of float32 tensors, the first and the second moments."""
    return _lib.torch_binding().adamw_state_values(exp_avgs, exp_avg_sqs, scales)


class AdamW(torch.optim.Optimizer):
    """AdamW whose step is one call of `adamw_step` for each type of weights in a group (48 tensors a launch).

    state_bits: 32 (float32 states) or 8 (one byte a state, two float32 for 256 elements: a gradient that is not finite makes the states of all 256
    NaN from then on, and their weights with the next step).  master_weights: keep float32 weights for 16-bit
    parameters (a 16-bit weight does not see updates below 2^-9 of it).  The state is that of torch.optim.AdamW -- "step", "exp_avg",
    "exp_avg_sq" -- and, where there are any, "scale" and "master".  Parameters without a gradient are left alone.  The state of a
    parameter, its step count included, lives on the GPU and stays where it is, so step() can be captured in a graph once the state exists (one
    eager step); a learning rate is part of the capture.  load_state_dict makes new state tensors: capture again after it."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32, master_weights=True):
        if not lr >= 0.0 or not eps >= 0.0 or not weight_decay >= 0.0:
            raise SocmxError(f"AdamW: lr {lr}, eps {eps} and weight_decay {weight_decay} are not negative")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise SocmxError(f"AdamW: betas {tuple(betas)} outside [0, 1)")
        if state_bits not in (8, 32):
            raise SocmxError(f"AdamW: state_bits is 8 or 32, got {state_bits}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      master_weights=master_weights))

    def _new_state(self, p, group):
        if not p.is_cuda:
            raise SocmxError(f"AdamW: parameters on the GPU are needed, got {p.device} (there is no CPU path)")
        if torch.cuda.is_current_stream_capturing():
            raise SocmxError("AdamW: the state of a parameter would be created inside a capture: take one step before it")
        if p.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise SocmxError(f"AdamW: float32, bfloat16 or float16 parameters are needed, got {p.dtype}")
        if torch.empty_like(p).stride() != p.stride() and not p.is_contiguous():
            raise SocmxError(f"AdamW: a parameter is dense in memory, got strides {p.stride()} for {tuple(p.shape)}")
        st = self.state[p]
        st["step"] = torch.zeros((), dtype=torch.float32, device=p.device)
        kinds = (torch.float32, torch.float32) if group["state_bits"] == 32 else (torch.int8, torch.uint8)
        for name, kind in zip(("exp_avg", "exp_avg_sq"), kinds):
            st[name] = torch.zeros_like(p, dtype=kind, requires_grad=False)          # (dense, in p's order of dimensions)
        if group["state_bits"] == 8:
            st["scale"] = torch.zeros(scale_rows(p.numel()), 2, dtype=torch.float32, device=p.device)
        if group["master_weights"] and p.dtype != torch.float32:
            st["master"] = p.detach().to(torch.float32)
        return st

    @staticmethod
    def _laid_like(grad, p):
        if p.is_contiguous() and grad.is_contiguous() or grad.stride() == p.stride():
            return grad
        return torch.empty_like(p, requires_grad=False).copy_(grad)

    def load_state_dict(self, state_dict):
        """torch casts what it loads to the parameters' type: codes, masters and float32 states of 16-bit weights are taken as they are.
        A state of torch.optim.AdamW is taken too, without its amsgrad and maximize, which are refused."""
        for group in state_dict["param_groups"]:
            for name in ("amsgrad", "maximize"):
                if group.get(name):
                    raise SocmxError(f"AdamW: a state with {name} cannot be continued")
        super().load_state_dict(state_dict)
        for group in self.param_groups:
            for name, value in self.defaults.items():
                group.setdefault(name, value)
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(ids, (p for g in self.param_groups for p in g["params"])):
            for name, v in state_dict["state"].get(i, {}).items():
                kind = torch.float32 if name == "step" or torch.is_tensor(v) and v.is_floating_point() else None
                self.state[p][name] = torch.as_tensor(v).detach().clone().to(device=p.device, dtype=kind)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        found = {}                                 # (what is refused is refused before anything is updated)
        for k, group in enumerate(self.param_groups):
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise SocmxError("AdamW: a sparse gradient")
                st = self.state.get(p) or self._new_state(p, group)
                found.setdefault((k, p.dtype, p.device, "scale" in st, "master" in st), []).append((p, st))
        for (k, _, _, small, master), some in found.items():
            group = self.param_groups[k]
            adamw_step([p for p, _ in some], [self._laid_like(p.grad, p) for p, _ in some], [st["exp_avg"] for _, st in some],
                       [st["exp_avg_sq"] for _, st in some], [st["step"] for _, st in some], lr=group["lr"], betas=group["betas"],
                       eps=group["eps"], weight_decay=group["weight_decay"], scales=[st["scale"] for _, st in some] if small else None,
                       masters=[st["master"] for _, st in some] if master else None)
        return loss
