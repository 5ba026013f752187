"""Layer operators on the GPU: layer norm and the gated scan, with their gradients (csrc/socmx_layernorm.hip, csrc/socmx_scan.hip; the
tensors' side in csrc/socmx_torch.cpp).

They stand beside the linear / ReLU operators of `socmx.nets`: what a control network with normalised layers, or with a memory
along the trajectory, is built from.  No reference counterpart (the reference's networks have neither); the scan is the general
form of the decayed sums of reference SOC_matching/method.py:371-478, whose one trained rate is log_decay = -gamma dt.

Every call launches on the current stream of its tensors' device, allocates through torch's caching allocator (a captured call
uses the graph's own memory) and is bit-reproducible: no atomics.  There is no CPU path: CPU tensors raise SocmxError.

Gradients inside a captured graph: no autograd graph of the same leaves that was built on another stream may be alive (an output kept
from an eager iteration).  torch ties a leaf's gradient to the stream of its first graph and would wait for the capture there, which
ends the process when the capture is closed; a call that is captured while a leaf that leads to it is in that state raises SocmxError
instead.  (Leaves that are used behind the call are not seen by it.)

Derivatives are reverse-mode and first order: an input with a forward-mode tangent raises SocmxError, a second derivative raises RuntimeError.
A call under torch.jit.trace or make_fx raises SocmxError.
"""
import torch

from . import _lib
from ._lib import SocmxError

_binding = _lib.torch_binding


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of `x` (any number of dimensions; float32, bfloat16 or
    float16; rows may be strided).  weight, bias: (D,) of x's type or, both, float32; None is ones / zeros.  Statistics and sums
    are formed in float32, outputs are rounded once.  Differentiable in x, weight and bias."""
    return _binding().layer_norm(x, weight, bias, eps)


class LayerNorm(torch.nn.Module):
    """`layer_norm` over a last dimension of `dim` with trained weight (ones) and bias (zeros); `affine=False`: neither, `bias=False`: no
    bias."""

    def __init__(self, dim, eps=1e-5, affine=True, bias=True, device=None, dtype=None):
        super().__init__()
        self.dim, self.eps = int(dim), float(eps)
        kw = dict(device=device, dtype=dtype)
        self.weight = torch.nn.Parameter(torch.ones(self.dim, **kw)) if affine else None
        self.bias = torch.nn.Parameter(torch.zeros(self.dim, **kw)) if affine and bias else None

    def forward(self, x):
        if x.shape[-1] != self.dim:
            raise SocmxError(f"LayerNorm({self.dim}): the input's last dimension is {x.shape[-1]}")
        return layer_norm(x, self.weight, self.bias, self.eps)


def gated_scan(x, log_decay, initial=None, lengths=None, reverse=False):
    """The gated linear recurrence  h_t = exp(log_decay_t) h_{t-1} + x_t  along the first dimension of x (T, B, D); returns
    (h (T, B, D) of x's type, final state (B, D) float32).

    log_decay (T, B, G), of x's type or float32, G a divisor of D: gate j decays the D / G channels from j D / G on (G = D: one for each,
    G = 1: one for all).  It is the LOGARITHM of the decay: -gamma dt, or logsigmoid of a gate's logit; 0 keeps everything, -inf
    forgets everything before the step (the start of another sequence in a packed batch), infinities and NaN included.  x and
    log_decay may be strided or expanded in their first two dimensions.  initial (B, D) float32, or zeros.
    lengths (B,) int32: row b's steps are the first lengths[b] (0 to T; values outside are clipped); the steps behind them are not
    read, their h and gradients are 0 and the final state is the one before them.  reverse: from each row's last step to its
    first.  The state and all sums are float32 whatever x's type; a state that grows (log_decay above 0) beyond float32 is infinite or NaN, also
    where the growth of up to 256 steps together is beyond it and the state is not zero; an infinite one may become NaN under a log_decay
    from -1/4 to 0, the steps behind a row's length leave it as it is.  Differentiable in x, log_decay and initial."""
    return _binding().gated_scan(x, log_decay, initial, lengths, reverse)


def gated_scan_step(state, x, log_decay):
    """One step of `gated_scan` while a control is evaluated: state (B, D) float32 becomes exp(log_decay) state + x IN PLACE; returns it
    rounded to x's type, (B, D).  x (B, D), log_decay (B, G), neither in state's memory.  Not differentiable: inputs that require a gradient are
    refused where gradients are recorded."""
    return _binding().gated_scan_step(state, x, log_decay)
