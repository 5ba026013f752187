"""Layer norm, gated scan and AdamW at the edges of what a program does with them: torch's other modes, padded rows whose state is
infinite, gradients of gradients, rows far from zero, memory that is shared, graphs that outlive a change.

Oracles are plain formulas in 64 bits; tolerances count roundings in units of U = 2^-24, as in test_gpu_layers.py.
"""
import gc
import math

import pytest
import torch

from socmx import layers, optim
from socmx._lib import SocmxError
from test_gpu_layers import BF16, DEV, F16, F32, HYPER, U, close, gen, half, new_states, scan_case, scan_check, tiny

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_adamw_step_outlives_steps_with_missing_gradients(bits):
    """Replays of a captured step mixed with eager steps in which a parameter has no gradient: counts, states and weights are those of the
    same steps made one by one."""
    sizes, g = (1000, 37, 300), gen(51)
    start, grads = [torch.randn(n, generator=g) for n in sizes], [[torch.randn(n, generator=g) for n in sizes] for _ in range(12)]

    def setup():
        ps = [torch.nn.Parameter(t.to(DEV)) for t in start]
        buffers = [torch.zeros(n, device=DEV) for n in sizes]
        return ps, buffers, optim.AdamW(ps, lr=1e-2, weight_decay=0.1, state_bits=bits)
    # (None: all three; k: parameter k has no gradient in this step)
    plan = [None, None, 1, None, None, 0, 2, None, 1, None, None, None]
    ps, buffers, opt = setup()
    cs, held, copt = setup()

    def eager(ps, buffers, opt, row, missing):
        for i, (p, b, q) in enumerate(zip(ps, buffers, row)):
            b.copy_(q)
            p.grad = None if i == missing else b
        opt.step()
    graph, side, spare = None, torch.cuda.Stream(), []
    for k, (row, missing) in enumerate(zip(grads, plan)):
        eager(ps, buffers, opt, row, missing)
        if missing is not None or k == 0 or k == 4:
            eager(cs, held, copt, row, missing)
        else:
            for p, b, q in zip(cs, held, row):
                b.copy_(q)
                p.grad = b
            if graph is None:
                side.wait_stream(torch.cuda.current_stream())
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    copt.step()
            graph.replay()
        torch.cuda.synchronize()
        spare.append(torch.full((128,), 7.0, device=DEV))      # (takes what has been given back to the allocator)
        for p, c in zip(ps, cs):
            assert torch.equal(p, c), k
            for name, v in opt.state[p].items():
                assert torch.equal(v, copt.state[c][name]), (k, name)
    assert all(bool((t == 7).all()) for t in spare)
    assert [float(copt.state[c]["step"]) for c in cs] == [11.0, 10.0, 11.0]


def test_adamw_step_counts_each_where_it_lies():
    """More tensors than one launch counts (256), their counts in any order in one buffer: the same bits as with one tensor of counts."""
    n, g = 300, gen(52)
    make = lambda: [torch.randn(3 + i % 5, generator=gen(i)).to(DEV) for i in range(n)]   # noqa: E731
    grads = [torch.randn(p.shape, generator=g).to(DEV) for p in make()]
    runs = []
    for each in (False, True):
        ps = make()
        m, v, _, _ = new_states([p.numel() for p in ps], F32, 32, False, ps)
        steps = torch.arange(n, device=DEV).float()
        buffer = torch.full((2 * n,), -1.0, device=DEV)
        buffer[1::2] = steps.flip(0)
        counts = [buffer[2 * (n - 1 - i) + 1] for i in range(n)]
        optim.adamw_step(ps, grads, m, v, counts if each else steps, **HYPER)
        assert torch.equal(torch.stack(counts), torch.arange(n, device=DEV).float() + 1) if each else torch.equal(steps, torch.arange(n, device=DEV).float() + 1)
        assert bool((buffer[::2] == -1).all())
        runs.append(ps + m + v)
    assert all(torch.equal(p, q) for p, q in zip(*runs))
    one = torch.zeros((), device=DEV)
    f = lambda: torch.zeros(10, device=DEV)   # noqa: E731
    ok = dict(params=[f(), f()], grads=[f(), f()], exp_avgs=[f(), f()], exp_avg_sqs=[f(), f()], lr=1e-3)
    for bad in ([one, one], [one], [one, f()], [one, torch.zeros(())], [one, one.to(F16)]):
        with pytest.raises(SocmxError):
            optim.adamw_step(steps=bad, **ok)
    assert float(one) == 0.0


def test_forward_mode_derivatives_are_refused():
    """A dual tensor's tangent is not dropped: the call raises, with and without gradients recorded."""
    import torch.autograd.forward_ad as fwad
    x, a, state = torch.randn(4, 2, 6, device=DEV), -torch.rand(4, 2, 3, device=DEV), torch.zeros(2, 6, device=DEV)
    w = torch.ones(6, device=DEV)
    for grad in (False, True):
        with fwad.dual_level(), torch.set_grad_enabled(grad):
            dual = lambda t: fwad.make_dual(t, torch.ones_like(t))   # noqa: E731
            for call in (lambda: layers.layer_norm(dual(x)), lambda: layers.layer_norm(x, dual(w), w), lambda: layers.layer_norm(x, w, dual(w)),
                         lambda: layers.gated_scan(dual(x), a), lambda: layers.gated_scan(x, dual(a)), lambda: layers.gated_scan(x, a, dual(state)),
                         lambda: layers.gated_scan_step(state, dual(x[0]), a[0]), lambda: layers.gated_scan_step(state, x[0], dual(a[0])),
                         lambda: layers.gated_scan_step(dual(state), x[0], a[0])):
                with pytest.raises(SocmxError, match="forward-mode"):
                    call()
            layers.layer_norm(x)                               # (a plain tensor while a level is open)
    x.requires_grad_()
    for y in (layers.layer_norm(x), layers.gated_scan(x, a)[0], layers.gated_scan(x, a)[1]):
        with fwad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):          # (from the engine: without its class)
            torch.autograd.grad(y, x, fwad.make_dual(torch.ones_like(y), torch.ones_like(y)))
    assert not bool(state.any())


def test_tracing_is_refused():
    """torch.jit.trace sees allocations and no kernel: its function would return memory that nobody has written."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, a = torch.randn(4, 2, 6, device=DEV), -torch.rand(4, 2, 3, device=DEV)
    for f, args in ((lambda x: layers.layer_norm(x), (x,)), (lambda x, a: layers.gated_scan(x, a)[0], (x, a)),
                    (lambda x, a: layers.gated_scan_step(torch.zeros(2, 6, device=DEV), x[0], a[0]), (x, a))):
        with pytest.raises(SocmxError, match="trac"):
            torch.jit.trace(f, args, check_trace=False)
        with pytest.raises(SocmxError, match="trac"):
            make_fx(f)(*args)
        f(*args)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("n,T", [(20, 21), (20, 40), (16, 40), (16, 700), (130, 131), (130, 700), (300, 5000)])
@pytest.mark.parametrize("G", [8, 2, 1])
@pytest.mark.parametrize("reverse", [False, True])
def test_gated_scan_padding_keeps_an_infinite_state(kind, n, T, G, reverse):
    """A state that is infinite after a row's last step, and a gradient that is when it arrives there, are what they are in a batch without
    padding.  (Decays of 1/e: infinity times them is infinity.)"""
    D = 8 if G < 8 else G
    x, _, initial, dh, dfinal = scan_case(n, 2, D, G, n + T, kind)
    a = torch.full((n, 2, G), -1.0)
    last = 0 if reverse else n - 1
    x[last, 0, 0], x[last, 1, D - 1] = math.inf, -math.inf
    dfinal[0, 1], dfinal[1, 0] = math.inf, -math.inf

    def run(x, a, dh, lengths):
        ts = [t.to(DEV).requires_grad_() for t in (x, a, initial)]
        h, final = layers.gated_scan(*ts, lengths=lengths, reverse=reverse)
        return [h[:n], final] + [t[:n] for t in torch.autograd.grad([h, final], ts, [dh.to(DEV), dfinal.to(DEV)])]
    wide = lambda t: torch.cat([t, torch.full((T - n,) + t.shape[1:], math.nan, dtype=t.dtype)])   # noqa: E731
    want = run(x, a, dh, None)
    got = run(wide(x), wide(a), wide(dh), torch.tensor([n, n], dtype=torch.int32, device=DEV))
    assert float(want[1][0, 0]) == math.inf and float(want[1][1, D - 1]) == -math.inf and not bool(want[1].isnan().any())
    for p, q in zip(got, want):
        assert torch.equal(p.isnan(), q.isnan()) and torch.equal(p.isinf(), q.isinf())
        p, q = p.nan_to_num(posinf=1.0, neginf=-1.0).double(), q.nan_to_num(posinf=1.0, neginf=-1.0).double()
        assert float((p - q).abs().max()) <= 64 * U * float(q.abs().max())


@pytest.mark.parametrize("order", ["time", "batch"])
def test_gated_scan_results_may_be_changed_in_place(order):
    """Whatever the layout of x: h and the final state are tensors of their own."""
    x, a, initial, dh, _ = (t.to(DEV) for t in scan_case(30, 3, 8, 2, 5))
    if order == "batch":
        x = x.transpose(0, 1).contiguous().transpose(0, 1)
    x.requires_grad_()
    extra = torch.ones(8, device=DEV, requires_grad=True)
    want, = torch.autograd.grad(layers.gated_scan(x, a, initial)[0], x, 2 * dh)
    h, final = layers.gated_scan(x, a, initial)
    assert h._base is None and final._base is None
    h *= 2
    final += 1
    h += extra
    got, ge = torch.autograd.grad(h, [x, extra], dh)
    assert torch.equal(got, want)
    close(ge, dh.double().sum((0, 1)), 90 * U * dh.abs().double().sum((0, 1)))
    h, _ = layers.gated_scan(x.detach(), a, initial)
    h += extra                                                 # (no gradients recorded by the scan itself)
    assert h.requires_grad and h.transpose(0, 1).is_contiguous() is (order == "batch")


def test_a_second_derivative_is_refused_on_every_way_to_the_inputs():
    """Also where the upstream gradient is a constant and an input had to be laid out afresh, and by way of the initial state."""
    g = gen(17)
    base, decay = torch.randn(2, 8, 5, generator=g).to(DEV).requires_grad_(), (-torch.rand(2, 4, 5, generator=g)).to(DEV).requires_grad_()
    init = torch.randn(2, 8, generator=g).to(DEV).requires_grad_()
    far = lambda t: t.permute(2, 0, 1)   # noqa: E731  (steps, rows, channels, the steps next to each other in memory)
    cases = [(far(base), far(decay), None), (far(base), far(decay).contiguous(), init), (far(base).contiguous(), far(decay), init),
             (far(base.detach()), far(decay.detach()).requires_grad_(), init), (far(base).contiguous(), far(decay.detach()), init)]
    for x, a, first in cases:
        ins = [t for t in (x, a, first) if t is not None and t.requires_grad]
        h, final = layers.gated_scan(x, a, first)
        for grad in torch.autograd.grad(h.sum() + final.sum(), ins, create_graph=True):
            assert grad.requires_grad
            for t in ins:
                with pytest.raises(RuntimeError, match="not differentiable"):
                    torch.autograd.grad(h.sum() + grad.square().sum(), t, retain_graph=True)
    wide = torch.randn(16, generator=g).to(DEV).requires_grad_()
    x = torch.randn(3, 8, generator=g).to(DEV)
    w = wide[::2]
    y = layers.layer_norm(x, w)
    grad, = torch.autograd.grad(y.sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(y.sum() + grad.square().sum(), wide)
    x = torch.randn(8, 3, generator=g).to(DEV).requires_grad_()
    y = layers.layer_norm(x.t(), w)
    grad, = torch.autograd.grad(y.sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(y.sum() + grad.square().sum(), x)
    # one derivative, by either way, is what it was
    ref = torch.autograd.grad(layers.gated_scan(far(base), far(decay), init)[0].square().sum(), [base, decay, init])
    far_dense = torch.autograd.grad(layers.gated_scan(far(base).contiguous(), far(decay).contiguous(), init)[0].square().sum(), [base, decay, init])
    assert all(torch.equal(p, q) for p, q in zip(ref, far_dense))


def far_rows_oracle(x, w, b, eps, dy):
    """Outputs in 64 bits with their tolerances' float32 parts, for rows far from zero that hardly vary.

    Nothing here scales with |mean| / deviation in the first order.  With m the float32 next to the mean (off by E <= k U mean|x|, k additions one
    after the other), x - m is exact (x and m within a factor of 2), the mean of x - m is formed with an error of k U mean|x - m|, where
    mean|x - m| <= mean|x - mu| + E; what is left of a variance shifted by E^2 is off by (k + 2) U (var + E^2)."""
    x, dy, w, b = (t.double() for t in (x, dy, w, b))
    D, R = x.shape[1], x.shape[0]
    mu = x.mean(1, keepdim=True)
    var = (x - mu).square().mean(1, keepdim=True)
    r = 1 / (var + eps).sqrt()
    n = (x - mu) * r
    g = dy * w
    s, q = g.mean(1, keepdim=True), (g * n).mean(1, keepdim=True)
    dx = r * (g - s - n * q)
    k = 32 + D / 1024
    E = k * U * x.abs().mean(1, keepdim=True)
    shift = 1 + E * E * r * r
    dn = U * (k * r * ((x - mu).abs().mean(1, keepdim=True) + E) + (2 * k * shift + 8) * n.abs() + 2 * r * E)
    tol_y = w.abs() * dn + 4 * U * ((n * w).abs() + b.abs())
    G, GN = g.abs().mean(1, keepdim=True), (g * n).abs().mean(1, keepdim=True)
    # the sums of g (n + c) and of g, c the part of the mean that is taken off afterwards, |c| <= E r
    dq = (g.abs() * dn).mean(1, keepdim=True) + (k + 2) * U * (GN + E * r * G)
    tol_dx = r * (4 * U * g.abs() + (k + 2) * U * G + n.abs() * dq + dn * q.abs() + 4 * U * (n * q).abs() + (2 * k * shift + 8) * U * (g - s - n * q).abs())
    m = 64 + R / 256
    return [(n * w + b, tol_y), (dx, tol_dx), ((dy * n).sum(0), (dy.abs() * dn).sum(0) + m * U * (dy * n).abs().sum(0)),
            (dy.sum(0), m * U * dy.abs().sum(0))]


@pytest.mark.parametrize("offset,spread", [(100.0, 1e-3), (1000.0, 1e-2), (-3e4, 1.0)])
@pytest.mark.parametrize("rows,cols", [(40, 24), (40, 256), (30, 500), (40, 1601), (20, 4100), (6, 16384), (5, 20001)])
def test_layer_norm_of_rows_that_hardly_vary(offset, spread, rows, cols):
    """The part of the mean that one float32 does not hold, the same for a whole row, is in no output and no gradient."""
    g = gen(rows + cols)
    x = offset + spread * torch.randn(rows, cols, generator=g)
    w, b = 1 + 0.3 * torch.randn(cols, generator=g), torch.randn(cols, generator=g)
    dy = 1 + torch.randn(rows, cols, generator=g)
    ts = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    y = layers.layer_norm(*ts)
    got = [y] + list(torch.autograd.grad(y, ts, dy.to(DEV)))
    for t, (want, tol) in zip(got, far_rows_oracle(x, w, b, 1e-5, dy)):
        close(t, want, tol + half(F32) * want.abs() + tiny(F32))
    for i in (1, 2):                                           # each gradient alone: the same bits
        alone = [t.detach().requires_grad_(j == i - 1) for j, t in enumerate(ts)]
        assert torch.equal(torch.autograd.grad(layers.layer_norm(*alone), alone[i - 1], dy.to(DEV))[0], got[i])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind,master", [(F32, False), (BF16, True), (F16, True)])
@pytest.mark.parametrize("lr,decay", [(1e-5, 1e-2), (1e-3, 5e-5), (1e-4, 4e-4), (3e-4, 1e-2)])
def test_adamw_decay_of_a_small_share(bits, kind, master, lr, decay):
    """lr wd far below 1, no gradient: the float32 weight is p - lr wd p with ONE rounding, half a step of the weight, and what the product
    lr wd p is off by, 2 U of itself.  (A factor 1 - lr wd in float32 is off by up to 2^-25: a fifth of a decay of 1e-7.)"""
    g = gen(41)
    p = (1 + torch.rand(3000, generator=g)).to(kind)
    w = p.float() + (2 ** -10 * torch.rand(3000, generator=g) if master else 0)
    ps, ws = p.to(DEV), w.to(DEV)
    m, v, scales, _ = new_states([3000], kind, bits, False, [ps])
    optim.adamw_step([ps], [torch.zeros_like(ps)], m, v, torch.zeros(1, device=DEV), lr=lr, weight_decay=decay, scales=scales,
                     masters=[ws] if master else None)
    want = w.double() * (1 - lr * decay)
    step = 2.0 ** (torch.floor(torch.log2(want)) - 24)         # half the distance of float32 numbers there
    close(ws if master else ps, want, step + 2 * U * lr * decay * w.double() + 1e-15)
    if master:
        assert torch.equal(ps, ws.to(kind))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("decay", [0.0, 0.1])
def test_adamw_leaves_infinite_weights_infinite(bits, decay):
    p = torch.tensor([math.inf, -math.inf, 1.0, math.nan], device=DEV)
    m, v, scales, _ = new_states([4], F32, bits, False, [p])
    optim.adamw_step([p], [torch.full((4,), 0.5, device=DEV)], m, v, torch.zeros(1, device=DEV), lr=1e-2, weight_decay=decay, scales=scales)
    assert float(p[0]) == math.inf and float(p[1]) == -math.inf and 0.9 < float(p[2]) < 1.0 and math.isnan(float(p[3]))


def test_gated_scan_step_refuses_a_state_that_shares_memory():
    """Elements that are read while others write them would be a race."""
    x, a = torch.randn(3, 8, device=DEV), -torch.rand(3, 2, device=DEV)
    wide = torch.zeros(3, 40, device=DEV)
    state = wide[:, 4:12]
    flat = wide.view(-1)
    meet = lambda x, a: pytest.raises(SocmxError, match="shares memory")   # noqa: E731
    for xs, As in ((state, a), (wide[:, 5:13], a), (wide[:, :8], a), (wide[:, 11:19], a), (x, wide[:, 2:6]), (x, wide[:, 11:13]),
                   (flat[51:59].expand(3, 8), a), (flat[44:52].expand(3, 8), a), (x, flat[91:92].expand(3, 1)), (flat.as_strided((3, 8), (9, 1), 77), a),
                   (wide.view(F16).as_strided((3, 8), (16, 1), 1), a), (x, flat[4:].as_strided((3, 8), (0, 1)))):
        with meet(xs, As):
            layers.gated_scan_step(state, xs, As)
    assert not bool(wide.any())
    wide[:, 12:20], wide[:, 2:4] = x, a
    h = layers.gated_scan_step(state, wide[:, 12:20], wide[:, 2:4])          # (between each other in one buffer, and apart)
    assert torch.equal(h, x) and torch.equal(wide[:, 4:12], x) and torch.equal(wide[:, 2:4], a) and not bool(wide[:, :2].any())
    one = torch.zeros(30, device=DEV)
    layers.gated_scan_step(one[:24].view(3, 8), one[24:].as_strided((3, 1), (1, 1)).expand(3, 8).contiguous(), one[24:27].view(3, 1))
    layers.gated_scan_step(one[6:30].view(3, 8), one[:6].view(3, 2).repeat_interleave(4, 1), one[:6].view(3, 2))
    layers.gated_scan_step(one[6:30].view(3, 8), one[:6].expand(3, 6).repeat(1, 2)[:, :8], one[5:6].expand(3, 1))
    layers.gated_scan_step(wide[:2, 4:12], flat[52:60].expand(2, 8), a[:2])


def test_gated_scan_step_refuses_inputs_that_want_a_gradient():
    """It is not dropped without a word."""
    x, a = torch.randn(3, 8, device=DEV), -torch.rand(3, 2, device=DEV)
    for ts in ((x.clone().requires_grad_(), a), (x, a.clone().requires_grad_())):
        state = torch.zeros(3, 8, device=DEV)
        with pytest.raises(SocmxError, match="gradient"):
            layers.gated_scan_step(state, *ts)
        assert not bool(state.any())
        with torch.no_grad():
            layers.gated_scan_step(state, *ts)
        assert torch.equal(state, x)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_refuses_memory_that_is_shared_in_part(bits):
    """Not the same first element only: any element that one tensor's update writes and another's reads or writes."""
    n = 600
    flat = torch.zeros(4 * n, device=DEV)
    f = lambda t=F32: torch.zeros(n, dtype=t, device=DEV)   # noqa: E731
    kinds = (F32, F32) if bits == 32 else (torch.int8, torch.uint8)

    def call(**kw):
        a = dict(params=[f(), f()], grads=[f(), f()], exp_avgs=[f(kinds[0]), f(kinds[0])], exp_avg_sqs=[f(kinds[1]), f(kinds[1])],
                 steps=torch.zeros(2, device=DEV), lr=1e-3)
        if bits == 8:
            a["scales"] = [torch.zeros(optim.scale_rows(n), 2, device=DEV) for _ in range(2)]
        optim.adamw_step(**{**a, **kw})
    call(params=[flat[:n], flat[n:2 * n]], grads=[flat[2 * n:3 * n], flat[2 * n + 1:3 * n + 1]])      # (gradients may overlap each other)
    small = torch.zeros(n, dtype=kinds[0], device=DEV)
    for bad in (dict(params=[flat[:n], flat[n - 1:2 * n - 1]]), dict(params=[flat[:n], f()], grads=[f(), flat[1:n + 1]]),
                dict(params=[flat[:n], f()], grads=[flat[:n], f()]), dict(params=[f(), flat[1:n + 1]], grads=[flat[:n], f()]),
                dict(params=[flat[:n], f()], steps=flat[n - 1:n + 1]), dict(grads=[flat[:n], f()], steps=flat[n - 1:n + 1]),
                dict(grads=[flat[:n], f()], steps=[flat[4], flat[3 * n]]), dict(exp_avgs=[small, small]),
                dict(steps=[flat[3], flat[3]])):
        with pytest.raises(SocmxError, match="another tensor's"):
            call(**bad)
    if bits == 8:
        scales = torch.zeros(2 * optim.scale_rows(n), 2, device=DEV)
        call(scales=[scales[:optim.scale_rows(n)], scales[optim.scale_rows(n):]])
        with pytest.raises(SocmxError, match="another tensor's"):
            call(scales=[scales[:optim.scale_rows(n)], scales[1:1 + optim.scale_rows(n)]])
        codes = torch.zeros(2 * n, dtype=torch.int8, device=DEV)
        with pytest.raises(SocmxError, match="another tensor's"):
            call(exp_avgs=[codes[:n], codes[n - 1:2 * n - 1]])
    assert not bool(flat.any())


@pytest.mark.parametrize("T,B", [(0, 3), (5, 0), (0, 0)])
def test_gated_scan_gradients_of_no_steps_and_no_rows(T, B):
    """Every input has a gradient: nothing for x and log_decay, the final state's for the initial one."""
    x, a = torch.zeros(T, B, 4, device=DEV, requires_grad=True), torch.zeros(T, B, 2, device=DEV, requires_grad=True)
    init = torch.ones(B, 4, device=DEV, requires_grad=True)
    h, final = layers.gated_scan(x, a, init)
    assert h.shape == (T, B, 4) and torch.equal(final, init) and (B == 0 or final.data_ptr() != init.data_ptr())
    up = torch.arange(4 * B, device=DEV).reshape(B, 4).float()
    gx, ga, g0 = torch.autograd.grad([h, final], [x, a, init], [torch.zeros_like(h), up])
    assert gx.shape == x.shape and ga.shape == a.shape and torch.equal(g0, up)
    h, final = layers.gated_scan(x, a)
    gx, ga = torch.autograd.grad(h.sum() + final.sum(), [x, a])
    assert gx.shape == x.shape and ga.shape == a.shape and final.shape == (B, 4) and not bool(final.any())


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_goes_on_from_a_state_of_torch(bits):
    """Parameters that torch has stepped go on in 32 bits, those that it has not get the new optimiser's states."""
    g = gen(61)
    ps = [torch.nn.Parameter(torch.randn(n, generator=g).to(DEV)) for n in (300, 41)]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    kw = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-6, weight_decay=0.1)
    ref = torch.optim.AdamW(ps, **kw)
    for p in ps[:1]:
        p.grad = torch.randn(p.shape, generator=g).to(DEV)
    ref.step()
    qs[0].data.copy_(ps[0])
    opt = optim.AdamW(qs, state_bits=bits)
    opt.load_state_dict(ref.state_dict())
    for _ in range(3):
        for p, q in zip(ps, qs):
            p.grad = torch.randn(p.shape, generator=g).to(DEV)
            q.grad = p.grad.clone()
        ref.step()
        opt.step()
    # 24 roundings on either side of each update, none longer than 3 lr (the codes of the parameter that is new to both differ in 8 bits)
    for p, q in zip(ps[:1 if bits == 8 else 2], qs):
        close(q, p.detach(), 2 * 3 * U * (3 * p.detach().abs().double().cpu() + 24 * 3e-2))
    assert [float(opt.state[q]["step"]) for q in qs] == [4.0, 3.0]
    assert opt.state[qs[0]]["exp_avg"].dtype == F32 and ("scale" in opt.state[qs[1]]) == (bits == 8)


@pytest.mark.parametrize("kind,bits", [(F32, 32), (F32, 8), (BF16, 8)])
def test_adamw_of_parameters_in_other_orders_in_memory(kind, bits):
    """A transposed weight and one with its channels last: the bits of the same memory as contiguous parameters, also with gradients laid out
    differently, through a saved state, and in step."""
    g = gen(71)
    base = [torch.randn(17, 40, generator=g).to(kind).to(DEV), torch.randn(3, 5, 7, 4, generator=g).to(kind).to(DEV)]
    turn = (lambda t: t.t(), lambda t: t.permute(0, 3, 1, 2))
    make = lambda ps: optim.AdamW(ps, lr=1e-2, weight_decay=0.1, state_bits=bits)   # noqa: E731
    plain = [torch.nn.Parameter(t.clone()) for t in base]
    turned = [torch.nn.Parameter(f(t.clone())) for f, t in zip(turn, base)]
    assert not any(p.is_contiguous() for p in turned)
    a, b = make(plain), make(turned)
    for k in range(4):
        for f, p, q in zip(turn, plain, turned):
            p.grad = torch.randn(p.shape, generator=g).to(kind).to(DEV)
            q.grad = f(p.grad.clone()) if k % 2 else f(p.grad).contiguous()
        a.step()
        b.step()
        if k == 1:
            state = b.state_dict()
            b = make(turned)
            b.load_state_dict(state)
    for f, p, q in zip(turn, plain, turned):
        assert torch.equal(f(p), q)
        for name, v in a.state[p].items():
            assert torch.equal(f(v) if v.dim() > 2 or name in ("exp_avg", "exp_avg_sq", "master") else v, b.state[q][name]), name
    t = lambda *s: torch.zeros(*s, device=DEV)   # noqa: E731
    for p, q in ((t(4, 6).t(), t(6, 4)), (t(6, 4), t(4, 6).t()), (t(4, 12)[:, ::2], t(4, 6)), (t(4, 1).expand(4, 6), t(4, 6)), (t(4, 6).t(), t(24))):
        with pytest.raises(SocmxError, match="laid out alike"):
            optim.adamw_step([p], [q], [t(p.shape)], [t(p.shape)], t(1), lr=1e-3)


def test_adamw_refuses_tangents():
    import torch.autograd.forward_ad as fwad
    f = lambda: torch.ones(10, device=DEV)   # noqa: E731
    ok = dict(params=[f()], grads=[f()], exp_avgs=[f()], exp_avg_sqs=[f()], steps=torch.zeros(1, device=DEV), lr=1e-3)
    with fwad.dual_level(), torch.no_grad():
        optim.adamw_step(**ok)
        for name in ("params", "grads", "exp_avgs", "exp_avg_sqs"):
            with pytest.raises(SocmxError, match="forward-mode"):
                optim.adamw_step(**{**ok, name: [fwad.make_dual(f(), f())]})


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("size", [1e-18, 1e-19])
def test_adamw_of_tiny_gradients_without_eps_in_codes(bits, size):
    """eps below 1e-10, states in 32 and in 8 bits: the first update is lr whatever the gradient's size.  v = 0.05 g^2 is 5e-38 at 1e-18 and, at
    1e-19, 5e-40, 3.6e5 of float32's smallest numbers: off by half of one in g g, its product and the sum, 4.2e-6 of v, half of that of its root."""
    p, q = torch.zeros(300, device=DEV), torch.full((300,), size, device=DEV)
    m, v, scales, _ = new_states([300], F32, bits, False, [p])
    optim.adamw_step([p], [q], m, v, torch.zeros(1, device=DEV), lr=1e-2, betas=(0.9, 0.95), eps=0.0, weight_decay=0.0, scales=scales)
    close(p, torch.full((300,), -1e-2).double(), 1e-2 * (30 * U + (2.1e-6 if size < 1e-18 else 0)))


def test_the_trainer_s_captured_iteration_with_adamw_is_the_eager_one():
    """Six iterations on the noise of the same device key, replayed and eager: the same losses and the same parameters up to what the two
    bodies' gradients differ by in their last bits.  (Both are stepped by the same kernel; an entry whose gradient nearly cancels moves by that
    difference over eps = 1e-4: 1e-5 of an update each, at most lr.)"""
    from test_host_cpu import build_sde
    from SOC_matching.method import SOC_Solver
    from socmx.rollout import PhiloxKey
    from socmx.train import Trainer, make_optimizer
    runs = []
    for graph in (False, True):
        torch.manual_seed(0)
        sde, aux = build_sde("tiny_double_well_d10", DEV)
        solver = SOC_Solver(sde, aux["x0"], None, T=aux["T"], num_steps=aux["K"], lmbd=aux["lmbd"], d=aux["d"], sigma=sde.sigma)
        solver.philox_key = PhiloxKey(torch.device(DEV), seed=77, offset=5)
        opt = make_optimizer(solver, nabla_V_lr=1e-3, M_lr=1e-3, weight_decay=0.05, state_bits=32)
        tr = Trainer(solver, opt, 16, normalization_const=0.8, hip_graph=graph, overlap_M_backward=False)
        steps = [tr.step() for _ in range(6)]
        tr.join()
        torch.cuda.synchronize()
        runs.append(([float(s["loss"]) for s in steps], {n: p.detach().clone() for n, p in sde.named_parameters()}, [s["mode"] for s in steps]))
    (le, pe, _), (lg, pg, modes) = runs
    assert "graph-replay" in modes
    assert all(abs(a - b) <= 2e-5 * abs(b) + 1e-7 for a, b in zip(lg, le)), (lg, le)
    for n in pe:
        close(pg[n], pe[n], 2e-5 * pe[n].abs().double().cpu() + 6 * 1e-5 * 1e-3 + 5e-7)


def test_adamw_refuses_before_it_updates_anything():
    """A parameter that the update has no form for, in the last group: the others stay as they are, and no state is left behind."""
    good = [torch.nn.Parameter(torch.ones(40, device=DEV)) for _ in range(2)]
    sparse = torch.nn.Embedding(5, 8, sparse=True, device=DEV)
    sparse(torch.tensor([1], device=DEV)).sum().backward()
    for bad in (torch.nn.Parameter(torch.ones(6, 8, device=DEV)[:, ::2]), torch.nn.Parameter(torch.ones(5, dtype=torch.float64, device=DEV)),
                torch.nn.Parameter(torch.ones(3, 1, device=DEV).expand(3, 4)), sparse.weight, torch.nn.Parameter(torch.ones(5))):
        if bad.grad is None:
            bad.grad = torch.ones_like(bad)
        opt = optim.AdamW([dict(params=good[:1]), dict(params=good[1:], lr=1.0), dict(params=[bad])])
        for p in good:
            p.grad = torch.ones_like(p)
        with pytest.raises(SocmxError):
            opt.step()
        assert all(bool((p == 1).all()) for p in good) and bad not in opt.state
        opt.param_groups[2]["params"] = []
        opt.step()
        assert all(float(opt.state[p]["step"]) == 1.0 for p in good)
        for p in good:
            p.data.fill_(1.0)


def test_a_capture_is_refused_for_every_leaf_that_leads_to_the_call():
    """Not only for leaves that are inputs themselves.  A leaf first used on a stream that the capture has joined is none of these."""
    d = 12
    net = torch.nn.Linear(d, d, device=DEV)
    x = torch.randn(5, 3, d, device=DEV)
    decay = torch.full((1, 1, 2), -0.5, device=DEV, requires_grad=True)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()

    def forward(which):
        y = torch.tanh(net(x)) * 2
        if which == "norm":
            return layers.layer_norm(y)
        return layers.gated_scan(x if which == "decay" else y, (decay * 2).expand(5, 3, 2))[0]
    for which in ("norm", "scan", "decay"):
        alive = forward(which)                                 # on the current stream
        side.wait_stream(torch.cuda.current_stream())
        with pytest.raises(SocmxError, match="alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                forward(which)                                 # (refused before there is a backward)
        del alive
        gc.collect()                                           # (frames of the refused call)
    params = list(net.parameters()) + [decay]

    def step(out):
        for p, q in zip(params, torch.autograd.grad(out, params, torch.ones_like(out))):
            p.grad = q
    want = forward("scan")
    step(want)
    eager, want = [p.grad.clone() for p in params], want.detach().clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):                              # (libraries set themselves up outside the capture)
        for _ in range(2):
            step(forward("scan"))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        other.wait_stream(side)
        with torch.cuda.stream(other):
            y = torch.tanh(net(x)) * 2                         # a branch of the capture
        side.wait_stream(other)
        out = layers.gated_scan(y, (decay * 2).expand(5, 3, 2))[0]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    del out, y
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(forward("scan"))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        forward("norm").sum().item()
        assert all(torch.allclose(p.grad, q, rtol=1e-5, atol=1e-6) for p, q in zip(params, eager))
