"""Cases for the operators of a recurrent layer's training step: layer norm, the gated scan, AdamW.

`run(state)` makes ONE pass through an operator.  With `own` false it is the operator's plain form in elementary torch
operations; with `own` true it is the call a user makes of this package.  `exact` is the operator's definition in 64 bits.

  norm    y = (x - mean) / sqrt(var + eps) * weight + bias over the last dimension; training: also d x, d weight, d bias
  scan    h_t = exp(log_decay_t) h_{t-1} + x_t along the first dimension of (T, B, D), a gate per D / G channels;
          training: also d x, d log_decay, d initial; "step": one time step on a state that stays
  adamw   decoupled weight decay, states in 32 bits or in 8 bits per block of 256 elements
"""
import math
import os
import random
import sys

import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
EPS = 1e-5
BLOCK = 256
HYPER = dict(lr=3e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "soc-matching_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from socmx import layers, optim
    return layers, optim


# ---- cases -------------------------------------------------------------------------------------------------------------
def _norm(name, rows, cols, dtype, wtype, mode, pad=0):
    return dict(name=name, op="norm", rows=rows, cols=cols, dtype=dtype, wtype=wtype, mode=mode, pad=pad)


def _scan(name, T, B, D, G, dtype, gtype, mode, reverse=False, ragged=False, resets=False, layout="time"):
    return dict(name=name, op="scan", T=T, B=B, D=D, G=G, dtype=dtype, gtype=gtype, mode=mode, reverse=reverse, ragged=ragged,
                resets=resets, layout=layout)


def _adamw(name, tensors, elements, dtype, bits, master=False):
    return dict(name=name, op="adamw", tensors=tensors, elements=elements, dtype=dtype, bits=bits, master=master)


def listed():
    return [
        # one step's batch of 128 rows through a 256-wide layer while a control is evaluated: latency
        _norm("norm forward 128x256", 128, 256, "float32", "float32", "forward"),
        # training on every row of 128 trajectories of 201 points, the control network's widest layer
        _norm("norm train 25728x256", 201 * 128, 256, "float32", "float32", "train"),
        # a wide layer in 16 bits with 32-bit weights
        _norm("norm train 8192x4096 bf16", 8192, 4096, "bfloat16", "float32", "train"),
        # odd sizes, rows cut out of a wider buffer, everything in fp16
        _norm("norm train 4111x1601 fp16", 4111, 1601, "float16", "float16", "train", pad=7),
        # serving: one new time step of 128 rows of a 256-wide recurrent control
        _scan("scan step 128x256", 1, 128, 256, 256, "float32", "float32", "step"),
        # decayed sums back from the terminal time along the trajectories of a d = 10 problem, one decay a step
        _scan("scan train 201x128x10", 201, 128, 10, 1, "float32", "float32", "train", reverse=True),
        # a padded batch of sequences in 16 bits, a gate for 64 channels, batch first in memory
        _scan("scan train 4096x8x2048 bf16", 4096, 8, 2048, 32, "bfloat16", "float32", "train", ragged=True, layout="batch"),
        # one very long trajectory, every channel its own gate, with resets where packed pieces begin
        _scan("scan train 65536x1x640", 65536, 1, 640, 640, "float32", "float32", "train", resets=True),
        # the parameters of the d = 10 control network
        _adamw("adamw control network", 18, 170562, "float32", 32),
        # a large model in 32 bits, its tensors packed in flat buffers at odd offsets
        _adamw("adamw 100 tensors 96M", 100, 96_000_000, "float32", 32),
        # a large model in bf16 with 32-bit master weights and 8-bit states
        _adamw("adamw 24 tensors 96M 8 bit", 24, 96_000_000, "bfloat16", 8, master=True),
        # a small model of odd tensors with 8-bit states
        _adamw("adamw 20 tensors 1M 8 bit", 20, 1_000_003, "float32", 8),
    ]


def _spread(rng, low, high):
    """A whole number spread over the logarithm of the range."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("norm", "scan", "adamw"))
    dtype = rng.choice(tuple(_TYPES))
    if op == "norm":
        cols = _spread(rng, 5, 16384)     # (with two columns d x is 1e-5 of its terms: nothing to compare)
        rows = _spread(rng, 1, min(65536, 33_000_000 // cols))
        c = _norm("", rows, cols, dtype, rng.choice((dtype, "float32")), rng.choice(("forward", "train", "train")),
                  rng.choice((0, 0, rng.randrange(1, 9))))
    elif op == "scan":
        mode = rng.choice(("forward", "train", "train", "step"))
        heads = rng.choice((1, _spread(rng, 1, 64)))
        per = rng.choice((1, _spread(rng, 1, 128)))
        D, G = heads * per, heads
        B = _spread(rng, 1, 256)
        T = 1 if mode == "step" else _spread(rng, 1, max(2, min(32768, 30_000_000 // (B * D))))
        c = _scan("", T, B, D, G, dtype, rng.choice((dtype, "float32")), mode, mode != "step" and rng.random() < 0.5,
                  mode != "step" and rng.random() < 0.4, rng.random() < 0.4, "time" if mode == "step" else rng.choice(("time", "batch")))
    else:
        bits = rng.choice((8, 32))
        elements = _spread(rng, 1000, 40_000_000)
        c = _adamw("", rng.randrange(1, 28 if bits == 8 else 120), elements, dtype, bits, dtype != "float32" and rng.random() < 0.6)
    del c["name"]
    return c


# ---- inputs ------------------------------------------------------------------------------------------------------------
def _sizes(case):
    """The sizes of an optimiser's tensors: of very different lengths, most of them odd, the same for every seed."""
    n, total = case["tensors"], case["elements"]
    if (n, total) == (18, 170562):     # weights and biases of the nine layers of the d = 10 control network, widths 256, 128, 64
        layers = ((11, 256), (256, 128), (128, 64), (11, 10), (256, 256), (128, 128), (64, 128), (128, 256), (256, 10))
        return [v for i, o in layers for v in (i * o, o)]
    r = random.Random(n * 1000003 + total)
    w = [math.exp(r.uniform(0.0, 4.0)) for _ in range(n)]
    return [max(1, int(total * v / sum(w))) for v in w]


def _offsets(sizes, to):
    """Offsets of tensors in a flat buffer, each rounded up to `to` elements, and the buffer's length."""
    at, out = 0, []
    for n in sizes:
        out.append(at)
        at += -(-n // to) * to
    return out, at


def _lengths(T, B):
    """Lengths of a padded batch: an empty one, one of a single step, a full one, the others between."""
    return [(0, 1, T)[b] if b < 3 and B > 3 else max(0, T - (b * T) // (2 * B)) for b in range(B)]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    s = dict(case=dict(case))
    rand = lambda *shape: torch.randn(shape, generator=gen, device=dev)   # noqa: E731
    if case["op"] == "norm":
        t, wt, R, C = _TYPES[case["dtype"]], _TYPES[case["wtype"]], case["rows"], case["cols"]
        # activations: channels of different scale around a common offset
        x = (rand(R, C + case["pad"]) * torch.exp(0.5 * rand(C + case["pad"])) + 0.7).to(t)
        s["x"] = x[:, :C].detach()
        s["weight"], s["bias"] = (1 + 0.2 * rand(C)).to(wt), (0.1 * rand(C)).to(wt)
        if case["mode"] == "train":
            s["dy"] = rand(R, C).to(t)
            for k in ("x", "weight", "bias"):
                s[k].requires_grad_()
    elif case["op"] == "scan":
        t, gt = _TYPES[case["dtype"]], _TYPES[case["gtype"]]
        T, B, D, G = (case[k] for k in ("T", "B", "D", "G"))

        def laid(v, kind):
            v = v.to(kind)
            return v.transpose(0, 1).contiguous().transpose(0, 1).detach() if case["layout"] == "batch" else v

        s["x"] = laid(rand(T, B, D), t)
        # memories of one step to some hundreds of them
        a = -torch.exp(1.5 * rand(T, B, G) - 2.5)
        if case["resets"]:
            a = a.masked_fill(torch.rand((T, B, 1), generator=gen, device=dev) < 1 / 512, -math.inf)
        s["log_decay"] = laid(a, gt)
        s["initial"] = rand(B, D)
        if case["mode"] == "step":
            s["x"], s["log_decay"] = s["x"][0], s["log_decay"][0]
        else:
            s["lengths"] = torch.tensor(_lengths(T, B), dtype=torch.int32, device=dev) if case["ragged"] else None
        if case["mode"] == "train":
            s["dh"], s["dfinal"] = laid(rand(T, B, D), t), rand(B, D)
            for k in ("x", "log_decay", "initial"):
                s[k].requires_grad_()
    else:
        t, sizes = _TYPES[case["dtype"]], _sizes(case)
        off, n = _offsets(sizes, BLOCK if case["bits"] == 8 else 1)
        cut = lambda v: [v[o:o + k] for o, k in zip(off, sizes)]   # noqa: E731
        s["sizes"], s["offsets"] = sizes, off
        used = torch.zeros(n, device=dev)
        for o, k in zip(off, sizes):
            used[o:o + k] = 1
        # weights of a few hundredths; gradients whose scale differs from region to region
        w = 0.05 * rand(n) * used
        region = 1e-3 * torch.exp(rand(-(-n // BLOCK))).repeat_interleave(BLOCK)[:n]
        g = region * rand(n) * used
        s["param"], s["grad"] = w.to(t), g.to(t)
        s["params"], s["grads"] = cut(s["param"]), cut(s["grad"])
        s["master"] = w.clone() if case["master"] else None
        s["masters"] = cut(s["master"]) if case["master"] else None
        s["steps"] = torch.full((len(sizes),), 20.0, device=dev)
        if case["bits"] == 32:
            s["m"], s["v"], s["scale"], s["scales"] = 0.3 * region * rand(n) * used, (region * (0.2 + rand(n).abs())).square() * used, None, None
        else:
            s["m"] = ((45 * rand(n)).round().clamp(-127, 127) * used).to(torch.int8)
            s["v"] = ((130 + 40 * rand(n)).round().clamp(1, 255) * used).to(torch.uint8)
            top = region[::BLOCK]
            s["scale"] = torch.stack([2 * top, (3 * top).square()], dim=1).contiguous()
            s["scales"] = [s["scale"][o // BLOCK:o // BLOCK - (-k // BLOCK)] for o, k in zip(off, sizes)]
        s["ms"], s["vs"] = cut(s["m"]), cut(s["v"])
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------
def _plain_norm(s):
    c, t, wt = s["case"], s["x"].dtype, s["weight"].dtype
    x, w, b = s["x"].detach().float(), s["weight"].detach().float(), s["bias"].detach().float()
    d = x - x.mean(dim=1, keepdim=True)
    r = torch.rsqrt((d * d).mean(dim=1, keepdim=True) + EPS)
    n = d * r
    y = (n * w + b).to(t)
    if c["mode"] == "forward":
        return y
    dy = s["dy"].float()
    g = dy * w
    dx = r * (g - g.mean(dim=1, keepdim=True) - n * (g * n).mean(dim=1, keepdim=True))
    return y, dx.to(t), (dy * n).sum(dim=0).to(wt), dy.sum(dim=0).to(wt)


def _prefix(a, x):
    """h_t = a_t h_{t-1} + x_t along the first dimension: pairs of steps joined, then pairs of pairs, and so on."""
    T, reach = x.shape[0], 1
    a = a.expand_as(x)
    while reach < T:
        x = torch.cat([x[:reach], x[reach:] + a[reach:] * x[:-reach]])
        a = torch.cat([a[:reach], a[reach:] * a[:-reach]])
        reach *= 2
    return x


def _plain_scan(s):
    c, t, gt = s["case"], s["x"].dtype, s["log_decay"].dtype
    B, D, G = c["B"], c["D"], c["G"]
    if c["mode"] == "step":
        a = torch.exp(s["log_decay"].float()).reshape(B, G, 1)
        s["initial"].copy_((a * s["initial"].reshape(B, G, D // G)).reshape(B, D) + s["x"].float())
        return s["initial"].to(t), s["initial"]
    T = c["T"]
    x = s["x"].detach().float().reshape(T, B, G, D // G)
    a = torch.exp(s["log_decay"].detach().float()).reshape(T, B, G, 1)
    h0 = s["initial"].detach().reshape(B, G, D // G)
    at = torch.arange(T, device=x.device).reshape(T, 1, 1, 1)
    n = (s["lengths"].long() if s["lengths"] is not None else torch.full((B,), T, device=x.device)).reshape(1, B, 1, 1)
    live = at < n
    x, a = torch.where(live, x, torch.zeros_like(x)), torch.where(live, a, torch.zeros_like(a))
    first = live & (at == (n - 1 if c["reverse"] else 0))      # the step that reads `initial`
    last = live & (at == (0 if c["reverse"] else n - 1))
    turn = (lambda v: v.flip(0)) if c["reverse"] else (lambda v: v)
    shift = lambda v: torch.cat([torch.zeros_like(v[:1]), v[:-1]])   # noqa: E731
    h = turn(_prefix(turn(a), turn(x + first * a * h0)))
    h = torch.where(live, h, torch.zeros_like(h))
    final = torch.where(n[0] > 0, (last * h).sum(dim=0), h0)
    if c["mode"] == "forward":
        return h.reshape(T, B, D).to(t), final.reshape(B, D)
    before = turn(shift(turn(h))) + first * h0                  # h_{t-1} as each step saw it
    dfinal = s["dfinal"].reshape(B, G, D // G)
    dh = torch.where(live, s["dh"].float().reshape(T, B, G, D // G), torch.zeros_like(h)) + last * dfinal
    back = (lambda v: v) if c["reverse"] else (lambda v: v.flip(0))
    g = back(_prefix(shift(back(a)), back(dh)))
    g = torch.where(live, g, torch.zeros_like(g))
    da = (a * before * g).sum(dim=3)
    d0 = torch.where(n[0] > 0, (first * a * g).sum(dim=0), dfinal)
    return h.reshape(T, B, D).to(t), final.reshape(B, D), g.reshape(T, B, D).to(t), da.to(gt), d0.reshape(B, D)


def _thresholds(s, n, step):
    """The two thresholds in (0, 1) of every element: a 32-bit mix of its place in its tensor and the step, cut in halves."""
    dev, low = s["param"].device, 0xFFFFFFFF
    off = torch.tensor(s["offsets"] + [n], device=dev)
    i = torch.arange(n, device=dev) - off[:-1].repeat_interleave(off.diff())
    z = (i * 0x9E3779B1 + step.long() * 0xBB67AE85) & low
    z = z ^ (z >> 16)
    z = (z * 0x6A09E667) & low
    z = z ^ (z >> 15)
    z = (z * 0x9E3779B1) & low
    z = z ^ (z >> 16)
    return ((z & 0xFFFF).double() + 0.5) / 65536, ((z >> 16).double() + 0.5) / 65536


def _code(value, scale, power, top, u):
    """The level c of top^power with value / scale * top^power between c^power and (c + 1)^power, one up where u says so."""
    r = value * torch.where(scale > 0, float(top ** power) / scale, torch.zeros_like(scale))
    c = (r.sqrt().sqrt() if power == 4 else r.sqrt()).floor().clamp(max=top)
    low = _power(c, power)
    return (c + (r - low > u * (_power(c + 1, power) - low)).double()).clamp(max=top)


def _power(c, power):
    """Whole numbers' squares and fourth powers, without the last digit that a library's power may lose."""
    return (c * c) * (c * c) if power == 4 else c * c


def _plain_adamw(s):
    c, (b1, b2) = s["case"], HYPER["betas"]
    s["steps"] += 1
    step = s["steps"][0].double()
    size, root = HYPER["lr"] / (1 - b1 ** step), torch.sqrt(1 - b2 ** step)
    p, g = s["master"] if c["master"] else s["param"].float(), s["grad"].float()
    if c["bits"] == 32:
        m, v = s["m"].mul_(b1).add_(g * (1 - b1)), s["v"].mul_(b2).add_(g * g * (1 - b2))
    else:
        # which of two levels a state becomes hangs on its last digits: 64 bits, as long as they are not levels
        n, wide = s["param"].numel(), lambda v: v.repeat_interleave(BLOCK)   # noqa: E731
        S = s["scale"].double()
        k, g = s["m"].double(), g.double()
        m = b1 * (k * k.abs() * wide(S[:, 0] / 127 ** 2)) + (1 - b1) * g
        v = b2 * (_power(s["v"].double(), 4) * wide(S[:, 1] / 255 ** 4)) + (1 - b2) * (g * g)
        s["scale"].copy_(torch.stack([m.abs().reshape(-1, BLOCK).amax(dim=1), v.reshape(-1, BLOCK).amax(dim=1)], dim=1))
        S = s["scale"].double()
        um, uv = _thresholds(s, n, step)
        s["m"].copy_(_code(m.abs(), wide(S[:, 0]), 2, 127, um) * m.sign())
        s["v"].copy_(torch.maximum(_code(v, wide(S[:, 1]), 4, 255, uv), (v > 0).double()))
        m, v = m.float(), v.float()
    p = p * (1 - HYPER["lr"] * HYPER["weight_decay"]) - size.float() * m / (v.sqrt() / root.float() + HYPER["eps"])
    s["param"].copy_(p)
    if c["master"]:
        s["master"].copy_(p)
    if c["bits"] == 32:
        return _adamw_outputs(s, s["m"], s["v"])
    k = s["m"].double()
    m, v = (k * k.abs() * wide(S[:, 0] / 127 ** 2)).float(), (_power(s["v"].double(), 4) * wide(S[:, 1] / 255 ** 4)).float()
    return _adamw_outputs(s, *([v[o:o + k] for o, k in zip(s["offsets"], s["sizes"])] for v in (m, v)))


def _adamw_outputs(s, m, v):
    return dict(param=s["param"], master=s["master"], m=m, v=v, scale=s["scale"], steps=s["steps"])


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if not own:
        with torch.no_grad():
            return {"norm": _plain_norm, "scan": _plain_scan, "adamw": _plain_adamw}[c["op"]](s)
    layers, optim = _package()
    if c["op"] == "norm":
        y = layers.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS)
        return (y,) + torch.autograd.grad(y, [s["x"], s["weight"], s["bias"]], s["dy"]) if c["mode"] == "train" else y
    if c["op"] == "scan":
        if c["mode"] == "step":
            return layers.gated_scan_step(s["initial"], s["x"], s["log_decay"]), s["initial"]
        h, final = layers.gated_scan(s["x"], s["log_decay"], s["initial"], lengths=s["lengths"], reverse=c["reverse"])
        if c["mode"] == "forward":
            return h, final
        return (h, final) + torch.autograd.grad([h, final], [s["x"], s["log_decay"], s["initial"]], [s["dh"], s["dfinal"]])
    optim.adamw_step(s["params"], s["grads"], s["ms"], s["vs"], s["steps"], scales=s["scales"], masters=s["masters"], **HYPER)
    if c["bits"] == 32:
        return _adamw_outputs(s, s["m"], s["v"])
    return _adamw_outputs(s, *optim.adamw_state_values(s["ms"], s["vs"], s["scales"]))


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "norm":
        n, e, w = case["rows"] * case["cols"], _BYTES[case["dtype"]], case["cols"] * _BYTES[case["wtype"]]
        if case["mode"] == "forward":
            return dict(bytes=2 * n * e + 2 * w, flops=8 * n)
        return dict(bytes=4 * n * e + 4 * w, flops=22 * n)
    if case["op"] == "scan":
        T, B, D, G = (case[k] for k in ("T", "B", "D", "G"))
        steps = sum(_lengths(T, B)) if case["ragged"] else T * B     # steps that are read; every step is written
        e, ge = D * _BYTES[case["dtype"]], G * _BYTES[case["gtype"]]
        if case["mode"] == "train":
            return dict(bytes=2 * (steps + T * B) * e + (steps + T * B) * ge + 5 * B * D * 4, flops=steps * (8 * D + G))
        return dict(bytes=(steps + T * B) * e + steps * ge + 2 * B * D * 4, flops=steps * (2 * D + G))
    n, e = sum(_sizes(case)), _BYTES[case["dtype"]]
    moved = 2 * e + (8 if case["master"] else e)           # gradient in, weight out; master, or weight, in and out
    if case["bits"] == 32:
        return dict(bytes=n * (moved + 16), flops=14 * n)
    return dict(bytes=n * (moved + 4 + 8) + 16 * n // BLOCK, flops=60 * n)     # the states' values go out too


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------
def _exact_norm(s):
    x, w, b = (s[k].detach().double().requires_grad_() for k in ("x", "weight", "bias"))
    with torch.enable_grad():
        y = (x - x.mean(dim=-1, keepdim=True)) / (x.var(dim=-1, unbiased=False, keepdim=True) + EPS).sqrt() * w + b
    if s["case"]["mode"] == "forward":
        return y.detach()
    return (y.detach(),) + torch.autograd.grad(y, [x, w, b], s["dy"].double())


def _exact_scan(s):
    """Step after step; each sequence on its own clock, so that a padded batch needs no masks in the recurrence itself."""
    c = s["case"]
    B, D, G = c["B"], c["D"], c["G"]
    spread = lambda v: v.repeat_interleave(D // G, dim=-1)   # noqa: E731
    h = s["initial"].detach().double().clone()
    if c["mode"] == "step":
        h = spread(s["log_decay"].double().exp()) * h + s["x"].double()
        return h, h
    T = c["T"]
    x, a = s["x"].detach().double(), s["log_decay"].detach().double().exp()
    n = s["lengths"].tolist() if s["lengths"] is not None else [T] * B
    count = torch.tensor(n, device=x.device)
    rows = torch.arange(B, device=x.device)

    def place(k):
        """Where each row's step number k is, and which rows have one."""
        return (count - 1 - k if c["reverse"] else torch.full_like(count, k)).clamp(0, T - 1), (k < count).unsqueeze(1)

    out, seen = torch.zeros_like(x), []
    for k in range(max(n)):
        t, on = place(k)
        if c["mode"] == "train":
            seen.append(h)
        h = torch.where(on, spread(a[t, rows]) * h + x[t, rows], h)
        out[t, rows] = torch.where(on, h, out[t, rows])
    if c["mode"] == "forward":
        return out, h
    dh, g = s["dh"].double(), s["dfinal"].double().clone()
    dx, da = torch.zeros_like(x), torch.zeros_like(a)
    for k in reversed(range(max(n))):
        t, on = place(k)
        total = g + dh[t, rows]
        at = a[t, rows]
        dx[t, rows] = torch.where(on, total, dx[t, rows])
        da[t, rows] = torch.where(on, at * (total * seen[k]).reshape(B, G, D // G).sum(dim=2), da[t, rows])
        g = torch.where(on, spread(at) * total, g)
    return out, h, dx, da, g


def _exact_adamw(s):
    c, (b1, b2), lr, eps = s["case"], HYPER["betas"], HYPER["lr"], HYPER["eps"]
    n = s["param"].numel()
    t = float(s["steps"][0]) + 1
    g = s["grad"].double()
    p = (s["master"] if c["master"] else s["param"]).double()
    scale = None
    if c["bits"] == 32:
        m, v = s["m"].double(), s["v"].double()
    else:
        signed = torch.arange(-127, 128, device=g.device, dtype=torch.float64)
        levels = [(signed * signed.abs()) / 127 ** 2, (torch.arange(256, device=g.device, dtype=torch.float64) / 255) ** 4]
        S = s["scale"].double().repeat_interleave(BLOCK, dim=0)
        m, v = levels[0][s["m"].long() + 127] * S[:, 0], levels[1][s["v"].long()] * S[:, 1]
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    p = p * (1 - lr * HYPER["weight_decay"]) - lr / (1 - b1 ** t) * m / ((v / (1 - b2 ** t)).sqrt() + eps)
    if c["bits"] == 8:
        scale = torch.stack([m.abs().reshape(-1, BLOCK).amax(dim=1), v.reshape(-1, BLOCK).amax(dim=1)], dim=1).float()
        S = scale.double().repeat_interleave(BLOCK, dim=0)
        u = _thresholds(s, n, torch.tensor(t, device=g.device))

        def near(value, S, levels, u):
            grid = levels[levels >= 0]
            share = torch.where(S > 0, value / S, torch.zeros_like(S))
            low = (torch.searchsorted(grid, share, right=True) - 1).clamp(0, len(grid) - 2)
            up = (share - grid[low]) / (grid[low + 1] - grid[low]) > u
            return grid, low + up.long()

        grid, k = near(m.abs(), S[:, 0], levels[0], u[0])
        m = m.sign() * grid[k] * S[:, 0]
        grid, k = near(v, S[:, 1], levels[1], u[1])
        v = grid[torch.maximum(k, (v > 0).long())] * S[:, 1]
        m, v = ([w[o:o + k] for o, k in zip(s["offsets"], s["sizes"])] for w in (m, v))
        scale = scale.double()
    return dict(param=p, master=p if c["master"] else None, m=m, v=v, scale=scale, steps=s["steps"].double() + 1)


def exact(case, seed):
    with torch.no_grad():
        return {"norm": _exact_norm, "scan": _exact_scan, "adamw": _exact_adamw}[case["op"]](prepare(case, seed))
