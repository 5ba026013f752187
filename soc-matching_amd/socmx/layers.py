"""Layer operators on the GPU: layer norm and the gated scan, with their gradients (csrc/socmx_layernorm.hip, csrc/socmx_scan.hip).

They stand beside the linear / ReLU operators of `socmx.nets`: what a control network with normalised layers, or with a memory
along the trajectory, is built from.  No reference counterpart (the reference's networks have neither); the scan is the general
form of the decayed sums of reference SOC_matching/method.py:371-478, whose one trained rate is log_decay = -gamma dt.

Every call launches on the current stream of its tensors' device, allocates through torch's caching allocator (a captured call
uses the graph's own memory) and is bit-reproducible: no atomics.  There is no CPU path: CPU tensors raise SocmxError.

Gradients inside a captured graph: no autograd graph of the same leaves that was built on another stream may be alive (an output kept
from an eager iteration).  torch ties a leaf's gradient to the stream of its first graph and would wait for the capture there, which
ends the process when the capture is closed; a call that is captured in that state raises SocmxError instead.
"""
import ctypes as C

import torch

from . import _lib
from ._lib import SocmxError


def _type(t, what):
    kind = _lib.ELEMENT_TYPES.get(t.dtype)
    if kind is None:
        raise SocmxError(f"{what}: float32, bfloat16 or float16 is needed, got {t.dtype}")
    return kind


def _on_gpu(what, first, *others):
    if not first.is_cuda:
        raise SocmxError(f"{what}: tensors on the GPU are needed, got {first.device} (there is no CPU path)")
    for t in others:
        if t is not None and t.device != first.device:
            raise SocmxError(f"{what}: tensors on {first.device} and on {t.device}")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _guarded(out):
    """`out` of a Function that has just been applied.  Its leaves' gradient nodes carry the stream of the first call that met them
    (they live as long as any graph of the leaf does): a capture on another one is refused before its backward can wait there."""
    fn = out.grad_fn
    if fn is not None:
        here = _lib.stream_ptr(out.device)
        for node, _ in fn.next_functions:
            if type(node).__name__ == "AccumulateGrad":
                first = node.metadata.setdefault("socmx_stream", here)
                if first != here and torch.cuda.is_current_stream_capturing():
                    raise SocmxError("an autograd graph of the same leaf, built on another stream, is alive: drop what keeps it (the outputs "
                                     "of an eager iteration) before capturing")
    return out


# ---- layer norm ------------------------------------------------------------------------------------------------------------
def _rows(t):
    """`t` as rows of its last dimension, each dense, at one distance from the next: a view where its strides allow it."""
    cols = t.shape[-1]
    r = t if t.dim() == 2 else t.reshape(-1, cols)
    if cols > 1 and r.stride(1) != 1:
        r = r.contiguous()
    return r


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        r = _rows(x)
        rows, cols = r.shape
        dev = x.device
        y = torch.empty(x.shape, dtype=x.dtype, device=dev)
        grads = any(ctx.needs_input_grad)
        stats = torch.empty(2, rows, dtype=torch.float32, device=dev) if grads else None
        wtype = next((t.dtype for t in (weight, bias) if t is not None), x.dtype)
        weight, bias = (t if t is None or t.is_contiguous() else t.contiguous() for t in (weight, bias))
        if rows:
            with _lib.on_device(dev):
                _lib.check(_lib.lib().socmx_layer_norm_fwd(
                    _lib.ELEMENT_TYPES[x.dtype], _lib.ELEMENT_TYPES[wtype], r.data_ptr(), rows, cols, r.stride(0), _ptr(weight),
                    _ptr(bias), eps, y.data_ptr(), stats.data_ptr() if grads else None,
                    stats.data_ptr() + 4 * rows if grads else None, _lib.stream_ptr(dev)), "socmx_layer_norm_fwd")
        if grads:
            ctx.save_for_backward(x, weight, stats)
            ctx.wtype = wtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        r, d = _rows(x), _rows(dy)
        rows, cols = r.shape
        dev = x.device
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        kind = _lib.ELEMENT_TYPES[x.dtype]
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
        make = torch.empty if rows else torch.zeros
        dw = make(cols, dtype=ctx.wtype, device=dev) if need_w else None
        db = make(cols, dtype=ctx.wtype, device=dev) if need_b else None
        if rows:
            L = _lib.lib()
            ws = (torch.empty(L.socmx_layer_norm_bwd_workspace_floats(kind, rows, cols), dtype=torch.float32, device=dev)
                  if need_w or need_b else None)
            with _lib.on_device(dev):
                _lib.check(L.socmx_layer_norm_bwd(
                    kind, _lib.ELEMENT_TYPES[ctx.wtype], r.data_ptr(), rows, cols, r.stride(0), d.data_ptr(), d.stride(0),
                    _ptr(weight), stats.data_ptr(), stats.data_ptr() + 4 * rows, _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws),
                    _lib.stream_ptr(dev)), "socmx_layer_norm_bwd")
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of `x` (any number of dimensions; float32, bfloat16 or
    float16; rows may be strided).  weight, bias: (D,) of x's type or, both, float32; None is ones / zeros.  Statistics and sums
    are formed in float32, outputs are rounded once.  Differentiable in x, weight and bias."""
    what = "layer_norm"
    if x.dim() < 1 or x.shape[-1] < 1:
        raise SocmxError(f"{what}: the last dimension is empty or missing, got shape {tuple(x.shape)}")
    _on_gpu(what, x, weight, bias)
    _type(x, what)
    cols = x.shape[-1]
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and tuple(t.shape) != (cols,):
            raise SocmxError(f"{what}: {name} is ({cols},) for this input, got {tuple(t.shape)}")
        if t is not None and t.dtype not in (x.dtype, torch.float32):
            raise SocmxError(f"{what}: {name} is of the input's type {x.dtype} or float32, got {t.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise SocmxError(f"{what}: weight and bias of two types, {weight.dtype} and {bias.dtype}")
    if not float(eps) >= 0.0:
        raise SocmxError(f"{what}: eps {eps} is negative")
    return _guarded(_LayerNorm.apply(x, weight, bias, float(eps)))


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


# ---- gated scan --------------------------------------------------------------------------------------------------------------
def _dense_last(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _like(t, dtype=None):
    """A new tensor of `t`'s shape with steps outside rows, or rows outside steps, as in `t`: whichever it has further apart."""
    T, B, D = t.shape
    kw = dict(dtype=dtype or t.dtype, device=t.device)
    if t.stride(0) < t.stride(1):
        return torch.empty(B, T, D, **kw).transpose(0, 1)
    return torch.empty(T, B, D, **kw)


def _descriptor(x, a, lengths, reverse):
    return _lib.Scan(type=_lib.ELEMENT_TYPES[x.dtype], gate_type=_lib.ELEMENT_TYPES[a.dtype], T=x.shape[0], B=x.shape[1],
                     D=x.shape[2], G=a.shape[2], reverse=int(reverse), x_stride_t=x.stride(0), x_stride_b=x.stride(1),
                     gate_stride_t=a.stride(0), gate_stride_b=a.stride(1), lengths=_ptr(lengths))


def _sizes(scan):
    n = [C.c_int64() for _ in range(3)]
    _lib.check(_lib.lib().socmx_gated_scan_sizes(C.byref(scan), *(C.byref(v) for v in n)), "socmx_gated_scan_sizes")
    return [v.value for v in n]


def _floats(n, device):
    return torch.empty(n, dtype=torch.float32, device=device) if n else None


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, a, initial, lengths, reverse):
        dev = x.device
        x, a = _dense_last(x), _dense_last(a)
        T, B, D = x.shape
        h = _like(x)
        final = torch.empty(B, D, dtype=torch.float32, device=dev)
        scan = _descriptor(x, a, lengths, reverse)
        n_states, n_ws, _ = _sizes(scan)
        grads = any(ctx.needs_input_grad[:3])
        states, ws = _floats(n_states if grads else 0, dev), _floats(n_ws, dev)
        first = initial if initial is None or initial.is_contiguous() else initial.contiguous()
        with _lib.on_device(dev):
            _lib.check(_lib.lib().socmx_gated_scan_fwd(C.byref(scan), x.data_ptr(), a.data_ptr(), _ptr(first), h.data_ptr(),
                                                       h.stride(0), h.stride(1), final.data_ptr(), _ptr(states), _ptr(ws),
                                                       _lib.stream_ptr(dev)), "socmx_gated_scan_fwd")
        if grads:
            ctx.set_materialize_grads(False)
            ctx.save_for_backward(x, a, states, lengths)
            ctx.reverse = reverse
        return h, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dfinal):
        x, a, states, lengths = ctx.saved_tensors
        dev = x.device
        T, B, D = x.shape
        scan = _descriptor(x, a, lengths, ctx.reverse)
        ws = _floats(_sizes(scan)[2], dev)
        if dh is not None:
            dh = _dense_last(dh)
        if dfinal is not None:
            dfinal = dfinal.contiguous()
        dx, da = _like(x), _like(a)
        dinitial = torch.empty(B, D, dtype=torch.float32, device=dev) if ctx.needs_input_grad[2] else None
        with _lib.on_device(dev):
            _lib.check(_lib.lib().socmx_gated_scan_bwd(
                C.byref(scan), x.data_ptr(), a.data_ptr(), states.data_ptr(), _ptr(dh), dh.stride(0) if dh is not None else 0,
                dh.stride(1) if dh is not None else 0, _ptr(dfinal), dx.data_ptr(), dx.stride(0), dx.stride(1), da.data_ptr(),
                da.stride(0), da.stride(1), _ptr(dinitial), _ptr(ws), _lib.stream_ptr(dev)), "socmx_gated_scan_bwd")
        return dx, da, dinitial, None, None


def _check_scan(what, x, log_decay, state, dims):
    if x.dim() != dims or log_decay.dim() != dims:
        raise SocmxError(f"{what}: x and log_decay have {dims} dimensions, got {tuple(x.shape)} and {tuple(log_decay.shape)}")
    _on_gpu(what, x, log_decay, state)
    _type(x, what)
    if log_decay.dtype not in (x.dtype, torch.float32):
        raise SocmxError(f"{what}: log_decay is of x's type {x.dtype} or float32, got {log_decay.dtype}")
    D, G = x.shape[-1], log_decay.shape[-1]
    if tuple(log_decay.shape[:-1]) != tuple(x.shape[:-1]):
        raise SocmxError(f"{what}: log_decay {tuple(log_decay.shape)} does not go with x {tuple(x.shape)} (expand() shares a gate between "
                         "steps or rows)")
    if D < 1 or G < 1 or D % G:
        raise SocmxError(f"{what}: {G} gates do not divide {D} channels")


def gated_scan(x, log_decay, initial=None, lengths=None, reverse=False):
    """The gated linear recurrence  h_t = exp(log_decay_t) h_{t-1} + x_t  along the first dimension of x (T, B, D); returns
    (h (T, B, D) of x's type, final state (B, D) float32).

    log_decay (T, B, G), of x's type or float32, G a divisor of D: gate j decays the D / G channels from j D / G on (G = D: one for each,
    G = 1: one for all).  It is the LOGARITHM of the decay: -gamma dt, or logsigmoid of a gate's logit; 0 keeps everything, -inf
    forgets everything before the step (the start of another sequence in a packed batch), infinities and NaN included.  x and
    log_decay may be strided or expanded in their first two dimensions.  initial (B, D) float32, or zeros.
    lengths (B,) int32: row b's steps are the first lengths[b] (0 to T; values outside are clipped); the steps behind them are not
    read, their h and gradients are 0 and the final state is the one before them.  reverse: from each row's last step to its
    first.  The state and all sums are float32 whatever x's type.  Differentiable in x, log_decay and initial."""
    what = "gated_scan"
    _check_scan(what, x, log_decay, initial, 3)
    T, B, D = x.shape
    if initial is not None and (tuple(initial.shape) != (B, D) or initial.dtype != torch.float32):
        raise SocmxError(f"{what}: initial is ({B}, {D}) float32, got {tuple(initial.shape)} {initial.dtype}")
    if lengths is not None:
        _on_gpu(what, x, lengths)
        if tuple(lengths.shape) != (B,) or lengths.dtype != torch.int32:
            raise SocmxError(f"{what}: lengths is ({B},) int32, got {tuple(lengths.shape)} {lengths.dtype}")
        lengths = lengths.contiguous()
    if T == 0 or B == 0:
        # (no step, or no row: the state is what it was)
        return x + 0, initial + 0 if initial is not None else torch.zeros(B, D, dtype=torch.float32, device=x.device)
    h, final = _GatedScan.apply(x, log_decay, initial, lengths, bool(reverse))
    return _guarded(h), final


@torch.no_grad()
def gated_scan_step(state, x, log_decay):
    """One step of `gated_scan` while a control is evaluated: state (B, D) float32 becomes exp(log_decay) state + x IN PLACE; returns it
    rounded to x's type, (B, D).  x (B, D), log_decay (B, G).  Not differentiable."""
    what = "gated_scan_step"
    _check_scan(what, x, log_decay, state, 2)
    B, D = x.shape
    if tuple(state.shape) != (B, D) or state.dtype != torch.float32 or (D > 1 and state.stride(1) != 1):
        raise SocmxError(f"{what}: state is ({B}, {D}) float32 with dense rows, got {tuple(state.shape)} {state.dtype} strides {state.stride()}")
    if state.requires_grad:
        raise SocmxError(f"{what}: state is updated in place and must not require a gradient")
    if B > 1 and state.stride(0) < D:
        raise SocmxError(f"{what}: the rows of state overlap (stride {state.stride(0)})")
    x, log_decay = _dense_last(x), _dense_last(log_decay)
    h = torch.empty(B, D, dtype=x.dtype, device=x.device)
    if B:
        with _lib.on_device(x.device):
            _lib.check(_lib.lib().socmx_gated_scan_step(
                _lib.ELEMENT_TYPES[x.dtype], _lib.ELEMENT_TYPES[log_decay.dtype], B, D, log_decay.shape[1], x.data_ptr(), x.stride(0),
                log_decay.data_ptr(), log_decay.stride(0), state.data_ptr(), state.stride(0), h.data_ptr(),
                _lib.stream_ptr(x.device)), "socmx_gated_scan_step")
    return h
