"""Layer norm, gated scan and AdamW on the GPU against plain implementations in 64 bits.

Tolerances are sums over the roundings of each path, in units of U = 2^-24 (half a step of float32) times the magnitudes that are
rounded, plus half a step of the output's type; they were set before the first run.
"""
import math

import numpy as np
import pytest
import torch

from socmx import layers, optim
from socmx._lib import SocmxError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """Half a step of the smallest numbers of a type: what rounding to a denormal may lose."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def close(got, want, tol):
    got, want, tol = got.detach().double().cpu(), want.double().cpu(), torch.as_tensor(tol).double().cpu()
    assert got.shape == want.shape, (got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / tol).nan_to_num(1e9).max()):.3g} of the tolerance"


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- layer norm --------------------------------------------------------------------------------------------------------------
def norm_oracle(x, w, b, eps, dy):
    """Outputs in 64 bits and their tolerances' float32 parts (without the outputs' own rounding)."""
    x, dy = x.double(), dy.double()
    w64 = w.double() if w is not None else torch.ones(x.shape[1], dtype=torch.float64)
    b64 = b.double() if b is not None else torch.zeros(x.shape[1], dtype=torch.float64)
    D, R = x.shape[1], x.shape[0]
    mu = x.mean(1, keepdim=True)
    r = 1 / ((x - mu).square().mean(1, keepdim=True) + eps).sqrt()
    n = (x - mu) * r
    g = dy * w64
    s, q = g.mean(1, keepdim=True), (g * n).mean(1, keepdim=True)
    dx = r * (g - s - n * q)
    # a sum over D: at most 16 terms a lane one after the other (rows beyond 16384: D / 1024), then 10 levels of a tree
    k = 32 + D / 1024
    # error of n: the mean's (k roundings of mean |x|, one of x - mean) times r, the variance's relative one (2 k) times n
    dn = U * (k * r * (x.abs().mean(1, keepdim=True) + (x - mu).abs()) + (2 * k + 8) * n.abs())
    # (the error of the mean shifts every x - mean alike: its share in the variance is second order)
    tol_y = w64.abs() * dn + 4 * U * ((n * w64).abs() + b64.abs())
    G, GN = g.abs().mean(1, keepdim=True), (g * n).abs().mean(1, keepdim=True)
    dq = (g.abs() * dn).mean(1, keepdim=True) + (k + 2) * U * GN
    tol_dx = r * (4 * U * g.abs() + (k + 2) * U * G + n.abs() * dq + dn * q.abs() + 4 * U * (n * q).abs() + (2 * k + 8) * U * (g - s - n * q).abs())
    m = 64 + R / 256          # additions a weight's gradient goes through, one after the other
    out = [(n * w64 + b64, tol_y), (dx, tol_dx), ((dy * n).sum(0), (dy.abs() * dn).sum(0) + m * U * (dy * n).abs().sum(0)),
           (dy.sum(0), m * U * dy.abs().sum(0))]
    return out


def norm_check(x, w, b, dy, eps=1e-5):
    """x, dy on the CPU, as a view of whatever strides they have there; compares all four outputs on the GPU."""
    def put(t):
        if t is None:
            return None
        base = torch.as_strided(t, (t.untyped_storage().nbytes() // t.element_size(),), (1,), 0).to(DEV)
        return torch.as_strided(base, t.shape, t.stride(), t.storage_offset()).detach()
    xs, ws, bs = put(x).requires_grad_(), *(None if t is None else t.to(DEV).requires_grad_() for t in (w, b))
    y = layers.layer_norm(xs, ws, bs, eps=eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    wants = [xs] + [t for t in (ws, bs) if t is not None]
    got = torch.autograd.grad(y, wants, put(dy))
    D = x.shape[-1]
    o = norm_oracle(x.reshape(-1, D), w, b, eps, dy.reshape(-1, D))
    with torch.no_grad():
        assert torch.equal(layers.layer_norm(xs, ws, bs, eps=eps), y)          # without statistics, and the same bits again
    checks = [(y, o[0], x.dtype), (got[0], o[1], x.dtype)] + [(t, v, t.dtype) for t, v in zip(got[1:], o[2:] if w is not None else o[3:])]
    for t, (want, tol), kind in checks:
        close(t.reshape(want.shape), want, tol + half(kind) * want.abs() + tiny(kind))
    again = torch.autograd.grad(layers.layer_norm(xs, ws, bs, eps=eps), wants, put(dy))
    assert all(torch.equal(p, q) for p, q in zip(got, again))                  # no atomics


@pytest.mark.parametrize("kind,wkind", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (1, 7), (65, 10), (130, 33), (77, 64), (9, 65), (33, 128), (1030, 200), (17, 256),
                                       (19, 257), (40, 512), (21, 1000), (12, 1024), (11, 1025), (9, 2049), (10, 4100), (3, 8200), (5, 16384),
                                       (4, 16385), (70, 20001)])
def test_layer_norm_sizes(kind, wkind, rows, cols):
    g = gen(rows * 7919 + cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(0.5 * torch.randn(cols, generator=g)) + 0.7).to(kind)
    w, b = (1 + 0.3 * torch.randn(cols, generator=g)).to(wkind), torch.randn(cols, generator=g).to(wkind)
    norm_check(x, w, b, torch.randn(rows, cols, generator=g).to(kind))


@pytest.mark.parametrize("kind", [F32, BF16])
def test_layer_norm_strides_dimensions_and_missing_parts(kind):
    g = gen(5)
    base = torch.randn(40, 3, 101, generator=g).to(kind)
    w, b = torch.randn(96, generator=g).to(kind), torch.randn(96, generator=g).to(kind)
    x = base[:, :, 3:99]                                    # rows at odd distances, each at an odd offset
    dy = torch.randn(40, 3, 96, generator=g).to(kind)
    norm_check(x, w, b, dy)
    norm_check(base[:, 1, 5:101], w, None, dy[:, 0])
    norm_check(x, None, b, dy)
    norm_check(x, None, None, dy)
    norm_check(x[0, 0], w, b, dy[0, 0])                     # one dimension
    norm_check(x.transpose(0, 1), w, b, dy.transpose(0, 1).contiguous())
    norm_check(x, w, b, torch.randn(96, generator=g).to(kind).expand(40, 3, 96))
    norm_check(torch.randn(96, generator=g).to(kind).expand(40, 3, 96), w, b, dy)
    norm_check(torch.randn(96, 40, generator=g).to(kind).t(), w, b, dy[:, 0])       # columns apart: laid out afresh


def test_layer_norm_only_the_gradients_that_are_asked_for():
    g = gen(6)
    x, w, b = torch.randn(50, 300, generator=g).to(DEV), torch.randn(300, generator=g).to(DEV), torch.randn(300, generator=g).to(DEV)
    dy = torch.randn(50, 300, generator=g).to(DEV)
    full = torch.autograd.grad(layers.layer_norm(*(t.requires_grad_() for t in (x, w, b))), [x, w, b], dy)
    for want in ((0,), (1,), (2,), (0, 2), (1, 2)):
        ts = [t.detach().requires_grad_(i in want) for i, t in enumerate((x, w, b))]
        got = torch.autograd.grad(layers.layer_norm(*ts), [ts[i] for i in want], dy)
        assert all(torch.equal(p, full[i]) for p, i in zip(got, want))


def test_layer_norm_of_no_rows():
    x, w = torch.zeros(0, 8, device=DEV, requires_grad=True), torch.ones(8, device=DEV, requires_grad=True)
    y = layers.layer_norm(x, w, w)
    assert y.shape == (0, 8)
    gx, gw = torch.autograd.grad(y, [x, w], torch.zeros(0, 8, device=DEV))
    assert gx.shape == (0, 8) and torch.equal(gw, torch.zeros(8, device=DEV))


def test_layer_norm_keeps_rows_apart():
    """A row of NaN or infinity spoils its own outputs and the weights' gradients, no other row; a constant row gives the bias."""
    g = gen(8)
    for cols in (10, 300, 3000, 20000):
        x = torch.randn(12, cols, generator=g)
        clean = layers.layer_norm(x.to(DEV))
        x[3, cols // 2] = math.nan
        x[7, 0] = math.inf
        x[9] = 2.5
        xs = x.to(DEV).requires_grad_()
        y = layers.layer_norm(xs)
        gx, = torch.autograd.grad(y, [xs], torch.ones_like(y))
        rest = [0, 1, 2, 4, 5, 6, 8, 10, 11]
        assert torch.equal(y[rest], clean[rest]) and bool(torch.isfinite(gx[rest]).all())
        assert bool(torch.isnan(y[3]).all()) and not bool(torch.isfinite(y[7]).any())
        assert float(y[9].detach().abs().max()) == 0.0 and bool(torch.isfinite(gx[9]).all())


def test_layer_norm_gradient_against_differences():
    g = gen(9)
    x, w, b = torch.randn(4, 12, generator=g), torch.randn(12, generator=g), torch.randn(12, generator=g)
    dy = torch.randn(4, 12, generator=g)
    ts = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    got = torch.autograd.grad(layers.layer_norm(*ts), ts, dy.to(DEV))

    def f(*t):
        x, w, b = t
        return float((dy.double() * ((x - x.mean(1, keepdim=True)) / (x.var(1, unbiased=False, keepdim=True) + 1e-5).sqrt() * w + b)).sum())
    for i, grad in enumerate(got):
        for j in (0, grad.numel() // 2, grad.numel() - 1):
            up, down = ([t.double().clone() for t in (x, w, b)] for _ in range(2))
            up[i].view(-1)[j] += 1e-5
            down[i].view(-1)[j] -= 1e-5
            # (differences: 1e-10 of the third derivative and 1e-11 of rounding; the kernel's float32: 1e-5 of terms of a few units)
            assert abs((f(*up) - f(*down)) / 2e-5 - float(grad.view(-1)[j])) < 1e-4


def test_layer_norm_module_and_refusals():
    m = layers.LayerNorm(24, device=DEV)
    x = torch.randn(5, 24, device=DEV)
    assert torch.equal(m(x), layers.layer_norm(x, m.weight, m.bias))
    assert set(m.state_dict()) == {"weight", "bias"} and not list(layers.LayerNorm(24, affine=False).parameters())
    assert len(list(layers.LayerNorm(24, bias=False).parameters())) == 1
    w = torch.ones(24, device=DEV)
    for bad in (lambda: m(x[:, :5]), lambda: layers.layer_norm(x, w[:5]), lambda: layers.layer_norm(x.double()),
                lambda: layers.layer_norm(x, w.to(F16)), lambda: layers.layer_norm(x.to(F16), w.to(F16), w), lambda: layers.layer_norm(x, w.cpu()),
                lambda: layers.layer_norm(x[:, :0]), lambda: layers.layer_norm(x[0, 0]), lambda: layers.layer_norm(x, eps=-1.0)):
        with pytest.raises(SocmxError):
            bad()


# ---- gated scan ---------------------------------------------------------------------------------------------------------------
def walk(a, x, start):
    """h_k = a_k h_{k-1} + x_k over the first dimension in 64 bits; a decay of 0 forgets."""
    h, out = start, []
    for k in range(x.shape[0]):
        h = torch.where(a[k] == 0, x[k], a[k] * h + x[k])
        out.append(h)
    return torch.stack(out)


# A decay below the normal float32 numbers counts as 0 (the device's exp flushes denormals): it is off by at most 2^-126, which adds
# 2^-126 |h_{t-1}| to a step and 2^-126 |h_{t-1} G_t| to a gate's gradient.  (The first run met one: exp(-96.9) = 8.5e-43, whose gradient
# -4.7e-42 came out as 0.)
FLUSH = 2.0 ** -126
STEP = 24        # roundings of one step, in U of the sum of magnitudes: q (5), its use (2), the joining of runs (2 + 7), sums of log decays


def scan_oracle(x, alpha, initial, lengths, reverse, dh, dfinal):
    """(h, final, dx, dalpha, dinitial), each with its tolerance's float32 part."""
    T, B, D = x.shape
    G = alpha.shape[2]
    per = D // G
    x, dh = x.double(), dh.double()
    a = alpha.double().exp().repeat_interleave(per, dim=2)
    init = initial.double() if initial is not None else torch.zeros(B, D, dtype=torch.float64)
    dfin = dfinal.double() if dfinal is not None else torch.zeros(B, D, dtype=torch.float64)
    n = [T] * B if lengths is None else [min(max(int(v), 0), T) for v in lengths]
    z = lambda *s: torch.zeros(*s, dtype=torch.float64)   # noqa: E731
    out = dict(h=z(T, B, D), final=init.clone(), dx=z(T, B, D), da=z(T, B, G), d0=dfin.clone())
    tol = {k: torch.zeros_like(v) for k, v in out.items()}
    for b in range(B):
        if n[b] == 0:
            continue
        turn = (lambda v: v.flip(0)) if reverse else (lambda v: v)
        X, A, DH = (turn(v[:n[b], b]) for v in (x, a, dh))
        h, hm = walk(A, X, init[b]), walk(A, X.abs(), init[b].abs())
        he = walk(A, STEP * U * hm + FLUSH * torch.cat([init[b].abs()[None], hm[:-1]]), torch.zeros(D, dtype=torch.float64))
        one = torch.ones(1, D, dtype=torch.float64)
        An, back = torch.cat([A[1:], one]), lambda v: v.flip(0)   # noqa: E731
        g = back(walk(back(An), back(DH), dfin[b]))
        gm = back(walk(back(An), back(DH.abs()), dfin[b].abs()))
        ge = back(walk(back(An), STEP * U * back(gm) + FLUSH * back(torch.cat([gm[1:], dfin[b].abs()[None]])), torch.zeros(D, dtype=torch.float64)))
        prev, pm, pe = (torch.cat([s[None], v[:-1]]) for s, v in ((init[b], h), (init[b].abs(), hm), (z(D), he)))
        prev, pm, pe = (torch.where(A == 0, torch.zeros_like(v), v) for v in (prev, pm, pe))
        fold = lambda v: v.reshape(n[b], G, per).sum(2)   # noqa: E731
        for name, v, e in (("h", h, he), ("dx", g, ge), ("da", fold(A * prev * g), fold(A * (pe * gm + pm * ge) + ((STEP + per) * U * A + FLUSH) * pm * gm))):
            out[name][:n[b], b], tol[name][:n[b], b] = turn(v), turn(e)
        out["final"][b], tol["final"][b] = h[-1], he[-1]
        out["d0"][b], tol["d0"][b] = A[0] * g[0], A[0] * (ge[0] + STEP * U * gm[0]) + FLUSH * gm[0]
        out["d0"][b] = torch.where(A[0] == 0, torch.zeros_like(g[0]), out["d0"][b])
    return out, tol


def scan_case(T, B, D, G, seed, kind=F32, gkind=F32, resets=0.0):
    g = gen(seed)
    x = torch.randn(T, B, D, generator=g).to(kind)
    a = -torch.exp(1.5 * torch.randn(T, B, G, generator=g) - 2.5)
    if resets:
        a = a.masked_fill(torch.rand(T, B, G, generator=g) < resets, -math.inf)
    return x, a.to(gkind), torch.randn(B, D, generator=g), torch.randn(T, B, D, generator=g).to(kind), torch.randn(B, D, generator=g)


def scan_check(x, a, initial, dh, dfinal, lengths=None, reverse=False, oracle=None):
    """x, a, dh as they are on the GPU (any strides)."""
    ts = [t.detach().requires_grad_() for t in (x, a)] + [None if initial is None else initial.to(DEV).requires_grad_()]
    L = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    wants = [t for t in ts if t is not None]

    def once():
        h, final = layers.gated_scan(*ts, lengths=L, reverse=reverse)
        outs, ups = [h, final], [dh, None if dfinal is None else dfinal.to(DEV)]
        pick = [i for i, u in enumerate(ups) if u is not None]
        return [h, final] + list(torch.autograd.grad([outs[i] for i in pick], wants, [ups[i] for i in pick]))
    got = once()
    assert got[0].dtype == x.dtype and got[1].dtype == F32 and got[3].dtype == a.dtype
    want, tol = oracle or scan_oracle(*(t.detach().cpu() for t in (x, a)), initial, lengths, reverse, dh.cpu(), dfinal)
    for t, name in zip(got, ("h", "final", "dx", "da", "d0")):
        close(t, want[name], tol[name] + half(t.dtype) * want[name].abs() + tiny(t.dtype))
    with torch.no_grad():
        h, final = layers.gated_scan(*ts, lengths=L, reverse=reverse)
    assert torch.equal(h, got[0]) and torch.equal(final, got[1])
    assert all(torch.equal(p, q) for p, q in zip(got, once()))
    return got


TYPES = [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)]


@pytest.mark.parametrize("kind,gkind", TYPES)
@pytest.mark.parametrize("T,B,D,G", [(1, 1, 1, 1), (2, 3, 5, 5), (7, 2, 6, 1), (8, 1, 64, 64), (64, 2, 12, 3), (65, 3, 10, 10), (129, 5, 33, 11),
                                     (200, 130, 4, 4), (63, 300, 64, 64), (70, 40, 512, 8), (66, 70, 256, 1), (40, 3, 2048, 2)])
@pytest.mark.parametrize("reverse", [False, True])
def test_gated_scan_sizes(kind, gkind, T, B, D, G, reverse):
    x, a, initial, dh, dfinal = scan_case(T, B, D, G, T * 31 + B * 7 + D, kind, gkind, resets=0.02)
    scan_check(x.to(DEV), a.to(DEV), initial, dh.to(DEV), dfinal, reverse=reverse)


@pytest.mark.parametrize("kind,gkind", [(F32, F32), (BF16, F32)])
@pytest.mark.parametrize("T,B,D,G", [(2000, 1, 64, 64), (1500, 2, 30, 5), (1025, 1, 3, 1), (1300, 1, 700, 1)])
@pytest.mark.parametrize("reverse", [False, True])
def test_gated_scan_long_time_in_chunks(kind, gkind, T, B, D, G, reverse):
    x, a, initial, dh, dfinal = scan_case(T, B, D, G, T + D, kind, gkind, resets=0.002)
    lengths = [T, 700][:B]
    scan_check(x.to(DEV), a.to(DEV), initial, dh.to(DEV), dfinal, lengths=lengths, reverse=reverse)


@pytest.mark.parametrize("kind,T,B,D,G", [(F32, 4500, 2, 600, 600), (BF16, 4500, 1, 4096, 16), (F32, 5000, 1, 20, 20), (BF16, 5000, 1, 20, 4)])
def test_gated_scan_through_several_groups_of_chunks(kind, T, B, D, G):
    """Enough steps that the state is handed on from group to group of chunks, for few channels and for many."""
    x, a, initial, dh, dfinal = scan_case(T, B, D, G, T + D + G, kind, F32, resets=0.0005)
    scan_check(x.to(DEV), a.to(DEV), initial, dh.to(DEV), dfinal, reverse=D == 600)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("T,D,G", [(1, 3, 3), (70, 16, 4), (150, 9, 1), (130, 8, 8)])
def test_gated_scan_padded_batches(T, D, G, reverse):
    """Lengths of 0, 1, all, odd ones, and ones outside 0..T; what lies behind them is not read (NaN) and gets zeros."""
    lengths = [0, 1, T, T // 2, T - 1, -3, T + 5, min(T, 64), min(T, 65)]
    B = len(lengths)
    x, a, initial, dh, dfinal = scan_case(T, B, D, G, T + D)
    oracle = scan_oracle(x, a, initial, lengths, reverse, dh, dfinal)
    for b, n in enumerate(lengths):
        for t in (x, a, dh):
            t[max(n, 0):, b] = math.nan
    got = scan_check(x.to(DEV), a.to(DEV), initial, dh.to(DEV), dfinal, lengths=lengths, reverse=reverse, oracle=oracle)
    for b, n in enumerate(lengths):
        for i in (0, 2, 3):
            assert bool((got[i][max(n, 0):, b] == 0).all())
    assert torch.equal(got[1][0].cpu(), initial[0]) and torch.equal(got[4][0].cpu(), dfinal[0])


@pytest.mark.parametrize("kind,gkind", [(F32, F32), (BF16, F32), (F16, F16)])
def test_gated_scan_strides(kind, gkind):
    T, B, D, G = 90, 6, 32, 8
    x, a, initial, dh, dfinal = scan_case(T, B, D, G, 3, kind, gkind)
    oracle = scan_oracle(x, a, initial, None, False, dh, dfinal)
    swap = lambda t: t.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)   # noqa: E731

    def wide(t):
        big = torch.full((T, B, t.shape[2] + 5), math.nan, dtype=t.dtype, device=DEV)
        big[:, :, 3:3 + t.shape[2]] = t.to(DEV)
        return big[:, :, 3:3 + t.shape[2]]                                    # odd offsets, odd distances
    far = lambda t: t.permute(2, 0, 1).contiguous().to(DEV).permute(1, 2, 0)  # noqa: E731  (channels apart: laid out afresh)
    for how in (swap, wide, far):
        scan_check(how(x), how(a), initial, how(dh), dfinal, oracle=oracle)
    h, _ = layers.gated_scan(swap(x), a.to(DEV))
    assert h.transpose(0, 1).is_contiguous()                                  # laid out as x is
    scan_check(x.to(DEV), a.to(DEV), None, dh.to(DEV), dfinal)
    scan_check(x.to(DEV), a.to(DEV), initial, dh.to(DEV), None)
    # one decay a step for all rows, one input a row for all steps, one gradient for all
    shared = a[:, :1].to(DEV).expand(T, B, G)
    same = x[:1].to(DEV).expand(T, B, D)
    scan_check(same, shared, initial, dh[:1, :1].to(DEV).expand(T, B, D), dfinal)


def test_gated_scan_gradients_through_one_output_only():
    x, a, initial, dh, dfinal = scan_case(80, 3, 8, 2, 4)
    ts = [t.to(DEV).requires_grad_() for t in (x, a, initial)]
    _, final = layers.gated_scan(*ts)
    got = torch.autograd.grad(final, ts, dfinal.to(DEV))
    want, tol = scan_oracle(x, a, initial, None, False, torch.zeros_like(dh), dfinal)
    for t, name in zip(got, ("dx", "da", "d0")):
        close(t, want[name], tol[name] + half(F32) * want[name].abs() + tiny(F32))


def test_gated_scan_forgets_at_a_decay_of_zero():
    """-inf, and decays so low that exp gives 0, cut the sequence: infinities and NaN in front of the cut stay there."""
    T, B, D = 150, 2, 5
    x, a, initial, dh, dfinal = scan_case(T, B, D, D, 11)
    cut = [10, 63, 64, 65, 128]
    a[cut] = -math.inf
    a[cut[1]] = -1000.0
    clean = [t.cpu() for t in layers.gated_scan(x.to(DEV), a.to(DEV), initial.to(DEV))]
    x[9], x[62], x[127, 0, 0] = math.inf, math.nan, -math.inf
    ts = [t.to(DEV).requires_grad_() for t in (x, a)]
    h, final = layers.gated_scan(*ts)
    h, final = h.cpu(), final.cpu()
    for lo, hi in ((10, 62), (63, 64), (64, 65), (65, 127), (128, 150)):
        assert torch.equal(h[lo:hi], clean[0][lo:hi]), (lo, hi)
    assert torch.equal(final, clean[1])
    # the gradient of the last piece alone reaches no earlier one, and the gates at the cuts get none
    out, _ = layers.gated_scan(*ts)
    gx, ga = torch.autograd.grad(out[128:].sum(), ts)
    assert bool((gx[:128] == 0).all()) and bool((ga[cut] == 0).all()) and bool(torch.isfinite(ga[129:]).all())


@pytest.mark.parametrize("kind,gkind", [(F32, F32), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("T,D,G", [(40, 96, 3), (150, 192, 3), (129, 192, 2), (33, 128, 1), (300, 320, 2), (20, 1280, 1), (140, 768, 4)])
@pytest.mark.parametrize("reverse", [False, True])
def test_gated_scan_shared_gates_in_whole_rows_of_lanes(kind, gkind, T, D, G, reverse):
    lengths = [T, 0, 17, T - 1, 1]
    x, a, initial, dh, dfinal = scan_case(T, len(lengths), D, G, T + D + G, kind, gkind, resets=0.01)
    scan_check(x.to(DEV), a.to(DEV), initial, dh.to(DEV), dfinal, lengths=lengths, reverse=reverse)


def test_gated_scan_forgets_behind_any_decay():
    """Infinite and NaN decays in front of a cut, in the same run of steps, in another one and far before it, stay in front of it."""
    T, B, D = 700, 1, 4
    x, a, initial, _, _ = scan_case(T, B, D, D, 12)
    cut = [20, 100, 400, 690]
    a[cut] = -math.inf
    clean = [t.cpu() for t in layers.gated_scan(x.to(DEV), a.to(DEV), initial.to(DEV))]
    a[18], a[70], a[140] = math.inf, math.nan, math.inf
    h, final = (t.cpu() for t in layers.gated_scan(x.to(DEV), a.to(DEV), initial.to(DEV)))
    for lo, hi in ((0, 18), (20, 70), (100, 140), (400, T)):
        assert torch.equal(h[lo:hi], clean[0][lo:hi]), (lo, hi)
    assert torch.equal(final, clean[1])
    for lo, hi in ((18, 20), (70, 100), (140, 400)):
        assert not bool(torch.isfinite(h[lo:hi]).any()), (lo, hi)


def test_gated_scan_products_of_decays_beyond_float32():
    """No single decay forgets, but those of a run multiply to less than 2^-126: NaN stays NaN.  They multiply to more than the
    largest number: a state of zero stays zero, in either direction of the derivative."""
    T = 900
    x = torch.zeros(T, 1, 3, device=DEV)
    x[5, 0, 0] = math.nan
    h, final = layers.gated_scan(x, torch.full((T, 1, 3), -10.0, device=DEV))
    assert bool(h[5:, 0, 0].isnan().all()) and bool(final[0, 0].isnan()) and bool((h[..., 1:] == 0).all())
    a = torch.full((T, 1, 3), 3.0, device=DEV)
    a[-1] = -math.inf
    x = torch.zeros(T, 1, 3, device=DEV)
    x[-1] = 2.0
    ts = [t.requires_grad_() for t in (x, a)]
    h, final = layers.gated_scan(*ts)
    assert bool((h[:-1] == 0).all()) and bool((h[-1] == 2).all())
    gx, ga = torch.autograd.grad(final.sum(), ts)
    assert bool((gx[:-1] == 0).all()) and bool((gx[-1] == 1).all()) and bool((ga == 0).all())


def test_gated_scan_long_memory_is_exact():
    """A constant decay with a memory of 20000 steps: rounding exp(alpha) to float32 would be off by up to 20000 2^-25 = 6e-4 of the
    steady state; a gate kept as exp(alpha) - 1 leaves one rounding a step, in either direction."""
    T = 60000
    alpha = float(np.float32(-1.0 / 20000))
    x = torch.ones(T, 1, 2, device=DEV)
    a = torch.full((1, 1, 1), alpha, device=DEV).expand(T, 1, 2)
    _, final = layers.gated_scan(x, a)
    want = (1 - math.exp(alpha * T)) / -math.expm1(alpha)
    assert abs(float(final[0, 0]) - want) < 5e-5 * want


def test_gated_scan_gradient_against_differences():
    x, a, initial, dh, dfinal = scan_case(20, 2, 4, 2, 12)
    ts = [t.to(DEV).requires_grad_() for t in (x, a, initial)]
    got = torch.autograd.grad(layers.gated_scan(*ts, reverse=True), ts, [dh.to(DEV), dfinal.to(DEV)])

    def f(x, a, initial):
        h = walk(a.exp().repeat_interleave(2, dim=2).flip(0), x.flip(0), initial)
        return float((h.flip(0) * dh.double()).sum() + (h[-1] * dfinal.double()).sum())
    for i, grad in enumerate(got):
        for j in (0, grad.numel() // 2, grad.numel() - 1):
            up, down = ([t.double().clone() for t in (x, a, initial)] for _ in range(2))
            up[i].view(-1)[j] += 1e-5
            down[i].view(-1)[j] -= 1e-5
            assert abs((f(*up) - f(*down)) / 2e-5 - float(grad.reshape(-1)[j])) < 1e-4


@pytest.mark.parametrize("kind,gkind", TYPES)
@pytest.mark.parametrize("B,D,G", [(1, 1, 1), (3, 10, 1), (130, 256, 256), (7, 96, 12)])
def test_gated_scan_step_follows_the_scan(kind, gkind, B, D, G):
    T = 5
    x, a, initial, dh, dfinal = scan_case(T, B, D, G, B + D, kind, gkind, resets=0.1)
    want, tol = scan_oracle(x, a, initial, None, False, dh, dfinal)
    wide = torch.full((B, D + 3), 7.0, device=DEV)
    state = wide[:, 1:1 + D]                                   # a state that is a part of a wider buffer
    state.copy_(initial)
    xs, As = x.to(DEV), a.to(DEV)
    for t in range(T):
        h = layers.gated_scan_step(state, xs[t], As[t])
        close(h, want["h"][t], tol["h"][t] + half(kind) * want["h"][t].abs() + tiny(kind))
    close(state, want["final"], tol["final"] + half(F32) * want["final"].abs())
    assert bool((wide[:, 0] == 7).all()) and bool((wide[:, 1 + D:] == 7).all())


def test_gated_scan_of_no_steps_and_no_rows():
    x = torch.zeros(0, 3, 4, device=DEV, requires_grad=True)
    init = torch.ones(3, 4, device=DEV, requires_grad=True)
    h, final = layers.gated_scan(x, torch.zeros(0, 3, 2, device=DEV), init)
    assert h.shape == (0, 3, 4) and torch.equal(final, init)
    assert torch.equal(torch.autograd.grad(final.sum(), init)[0], torch.ones(3, 4, device=DEV))
    h, final = layers.gated_scan(torch.zeros(5, 0, 4, device=DEV), torch.zeros(5, 0, 4, device=DEV))
    assert h.shape == (5, 0, 4) and final.shape == (0, 4)
    assert layers.gated_scan_step(torch.zeros(0, 4, device=DEV), torch.zeros(0, 4, device=DEV), torch.zeros(0, 2, device=DEV)).shape == (0, 4)


def test_gated_scan_refusals():
    x, a, init = torch.zeros(4, 2, 6, device=DEV), torch.zeros(4, 2, 3, device=DEV), torch.zeros(2, 6, device=DEV)
    n = torch.zeros(2, dtype=torch.int32, device=DEV)
    s = lambda *v, **k: (lambda: layers.gated_scan(*v, **k))   # noqa: E731
    t = lambda *v: (lambda: layers.gated_scan_step(*v))   # noqa: E731
    for bad in (s(x[0], a[0]), s(x, a[:3]), s(x, a[:, :1]), s(x, a[:, :, :0]), s(x, torch.zeros(4, 2, 4, device=DEV)), s(x.double(), a),
                s(x, a.to(F16)), s(x.to(BF16), a.to(F16)), s(x, a.cpu()), s(x, a, init[:1]), s(x, a, init.to(F16)), s(x, a, init.cpu()),
                s(x, a, lengths=n[:1]), s(x, a, lengths=n.long()), s(x, a, lengths=n.cpu()),
                t(init[:1], x[0], a[0]), t(init.to(F16), x[0], a[0]), t(init.t().contiguous().t(), x[0], a[0]),
                t(init[:1].expand(2, 6), x[0], a[0]), t(init.clone().requires_grad_(), x[0], a[0]), t(init, x, a)):
        with pytest.raises(SocmxError):
            bad()


def test_a_second_derivative_is_refused():
    """Not silently left out: differentiating a gradient raises."""
    x = torch.randn(5, 2, 8, device=DEV, requires_grad=True)
    a = -torch.rand(5, 2, 4, device=DEV)
    for y in (layers.layer_norm(x), layers.gated_scan(x, a)[0]):
        g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="not differentiable"):
            torch.autograd.grad(g.sum(), x, retain_graph=True)
        with pytest.raises(RuntimeError, match="not differentiable"):
            torch.autograd.grad((g * x).sum(), x)


# ---- AdamW -------------------------------------------------------------------------------------------------------------------
def mix(i, step):
    """The two thresholds of element i at this step (csrc/socmx_adamw.hip)."""
    low = np.uint64(0xFFFFFFFF)
    with np.errstate(over="ignore"):
        z = (i.astype(np.uint64) * np.uint64(0x9E3779B1) + np.uint64(step) * np.uint64(0xBB67AE85)) & low
        z ^= z >> np.uint64(16)
        z = (z * np.uint64(0x6A09E667)) & low
        z ^= z >> np.uint64(15)
        z = (z * np.uint64(0x9E3779B1)) & low
        z ^= z >> np.uint64(16)
    return ((z & np.uint64(0xFFFF)).astype(np.float64) + 0.5) / 65536, ((z >> np.uint64(16)).astype(np.float64) + 0.5) / 65536


class Plain:
    """AdamW on one tensor in 64 bits; 8-bit states by the definition."""

    def __init__(self, p, bits, hyper):
        self.p, self.bits, self.h, self.t = p.astype(np.float64).reshape(-1), bits, hyper, 0
        n = self.p.size
        self.m, self.v, self.em, self.ev, self.eup = (np.zeros(n) for _ in range(5))
        self.cm, self.cv, self.S = np.zeros(n, np.int64), np.zeros(n, np.int64), np.zeros((-(-n // 256), 2), np.float32)

    def decode(self):
        S = self.S.astype(np.float64).repeat(256, axis=0)[:self.p.size]
        # (in the definition's order: which of two f32 a maximum becomes can hang on the last bit)
        return (self.cm * np.abs(self.cm)) * (S[:, 0] * (1 / 127 ** 2)), self.cv ** 4 * (S[:, 1] * (1 / 255 ** 4))

    def code(self, x, S, power, top, u):
        with np.errstate(divide="ignore", invalid="ignore"):
            r = np.where(S > 0, x * (top ** power * (1 / np.where(S > 0, S, 1))), 0)
        levels = np.arange(top + 1, dtype=np.float64) ** power
        c = np.clip(np.searchsorted(levels, r, side="right") - 1, 0, top - 1)
        place = (r - levels[c]) / (levels[c + 1] - levels[c])
        assert np.min(np.abs(place - u)) > 1e-11            # no code hangs on the last digits of this oracle
        return c + (place > u)

    def step(self, g, rounded=None):
        b1, b2 = self.h["betas"]
        self.t += 1
        g = g.astype(np.float64).reshape(-1)
        m, v = (self.m, self.v) if self.bits == 32 else self.decode()
        if self.bits == 32:
            # float32 states, a step: a constant's, a product's and a sum's rounding on each term, and what the step before left
            # (the first form of this took the newest m for the magnitude: an average of large gradients that cancel is off by more)
            self.em = b1 * self.em + 4 * U * (b1 * np.abs(m) + (1 - b1) * np.abs(g))
            self.ev = b2 * self.ev + 5 * U * (b2 * v + (1 - b2) * g * g)
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * (g * g)
        root = np.sqrt(v / (1 - b2 ** self.t)) + self.h["eps"]
        up = self.h["lr"] / (1 - b1 ** self.t) * m / root
        self.p = self.p * (1 - self.h["lr"] * self.h["weight_decay"]) - up
        # the update: its own 24 roundings, and the states' errors through m / root (d root = dv / 2v of it at most)
        self.eup = 24 * U * np.abs(up) + self.h["lr"] / (1 - b1 ** self.t) * self.em / root + np.abs(up) * self.ev / (2 * v + 1e-60)
        if self.bits == 32:
            self.m, self.v = m, v
            return
        n = self.p.size
        pad = -(-n // 256) * 256 - n
        block = lambda x: np.abs(np.pad(x, (0, pad))).reshape(-1, 256).max(1).astype(np.float32)   # noqa: E731
        self.S = np.stack([block(m), block(v)], axis=1)
        S = self.S.astype(np.float64).repeat(256, axis=0)[:n]
        um, uv = mix(np.arange(n), self.t)
        self.cm = (np.sign(m) * self.code(np.abs(m), S[:, 0], 2, 127, um)).astype(np.int64)
        self.cv = np.maximum(self.code(v, S[:, 1], 4, 255, uv), v > 0).astype(np.int64)


HYPER = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-6, weight_decay=0.1)
SIZES = [1, 3, 255, 256, 257, 1000, 4096, 4097, 0, 10007]


def new_states(sizes, kind, bits, master, params):
    dt = (F32, F32) if bits == 32 else (torch.int8, torch.uint8)
    m, v = ([torch.zeros(n, dtype=t, device=DEV) for n in sizes] for t in dt)
    scales = [torch.zeros(optim.scale_rows(n), 2, device=DEV) for n in sizes] if bits == 8 else None
    masters = [p.float() for p in params] if master else None
    return m, v, scales, masters


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind,master", [(F32, False), (BF16, False), (BF16, True), (F16, False), (F16, True)])
def test_adamw_step_many_tensors(kind, master, bits):
    """Five steps over tensors of many sizes cut out of one buffer at odd offsets, more of them than one launch takes."""
    g = gen(bits + master)
    sizes = SIZES * 6
    flat = lambda: torch.zeros(sum(sizes) + 1, dtype=kind, device=DEV)   # noqa: E731
    cut = lambda t: [v for v in t[1:].split(sizes)]   # noqa: E731
    params, grads = cut(flat()), cut(flat())
    for p in params:
        p.copy_(0.1 * torch.randn(p.shape, generator=g))
    ms, vs, scales, masters = new_states(sizes, kind, bits, master, params)
    steps = torch.zeros(len(sizes), device=DEV)
    plain = [Plain(p.float().cpu().numpy(), bits, HYPER) for p in params]
    left = [0] * len(sizes)
    for t in range(5):
        for p, q, o in zip(params, grads, plain):
            q.copy_(torch.randn(q.shape, generator=g) * torch.exp(2 * torch.randn(q.shape, generator=g)) * 1e-2)
            if not master:
                o.p = p.double().cpu().numpy().copy()       # (each step from the weights as they were rounded)
        old = [o.p.copy() for o in plain]
        optim.adamw_step(params, grads, ms, vs, steps, scales=scales, masters=masters, **HYPER)
        for i, (q, o) in enumerate(zip(grads, plain)):
            if sizes[i] == 0:
                continue
            o.step(q.float().cpu().numpy())
            T = torch.from_numpy
            if bits == 8:
                assert np.array_equal(scales[i].cpu().numpy(), o.S), (t, i)
                assert np.array_equal(ms[i].cpu().numpy(), o.cm) and np.array_equal(vs[i].cpu().numpy(), o.cv), (t, i)
            else:
                close(ms[i], T(o.m), o.em + 1e-38)
                close(vs[i], T(o.v), o.ev + 1e-38)
            # p: the rounding of the decay, its product and the difference; with masters the errors of all steps so far
            left[i] = (left[i] if master else 0) + U * 3 * (np.abs(old[i]) + np.abs(o.p)) + o.eup
            tol = left[i]
            if master:
                close(masters[i], T(o.p), tol)
                assert torch.equal(params[i], masters[i].to(kind))
            else:
                close(params[i], T(o.p), tol + half(kind) * np.abs(o.p) + tiny(kind))
    assert torch.equal(steps.cpu(), torch.full((len(sizes),), 5.0))


def test_adamw_steps_are_counted_for_each_tensor():
    p = [torch.ones(10, device=DEV), torch.ones(20, device=DEV)]
    q = [t.clone() for t in p]
    m, v, _, _ = new_states([10, 20], F32, 32, False, p)
    steps = torch.tensor([0.0, 99.0], device=DEV)
    optim.adamw_step(p, q, m, v, steps, **HYPER)
    assert steps.tolist() == [1.0, 100.0]
    b1, b2 = HYPER["betas"]
    for t, w in ((1, p[0]), (100, p[1])):
        up = HYPER["lr"] / (1 - b1 ** t) * (1 - b1) / (math.sqrt((1 - b2) / (1 - b2 ** t)) + HYPER["eps"])
        close(w, torch.full_like(w, 1.0).double() * (1 - HYPER["lr"] * HYPER["weight_decay"]) - up, 30 * U)


def test_adamw_8_bit_averages_keep_their_mean():
    """300 steps of noise: the mean second moment of 16384 elements.  A step moves it by 0.1 %, a twentieth of a level: rounding to
    the nearest level would leave it where it was.  The thresholds spread an element by about 12 %, the mean by 0.1 %."""
    n, g = 16384, torch.Generator(device=DEV).manual_seed(1)
    p = torch.zeros(n, device=DEV)
    m, v, scales, _ = new_states([n], F32, 8, False, [p])
    steps, wide = torch.zeros(1, device=DEV), torch.zeros(n, device=DEV)
    for t in range(300):
        q = torch.randn(n, generator=g, device=DEV) * (1.0 if t < 150 else 0.3)
        optim.adamw_step([p], [q], m, v, steps, lr=0.0, scales=scales)
        wide = 0.999 * wide + 0.001 * q * q
    got = optim.adamw_state_values(m, v, scales)[1][0]
    assert abs(float(got.mean() / wide.mean()) - 1) < 0.01


def test_adamw_state_values_and_blocks_that_are_not_finite():
    n = 1000
    p, q = torch.ones(n, device=DEV), torch.randn(n, generator=gen(2)).to(DEV)
    q[300] = math.nan
    q[800] = math.inf
    m, v, scales, _ = new_states([n], F32, 8, False, [p])
    steps = torch.zeros(1, device=DEV)
    optim.adamw_step([p], [q], m, v, steps, scales=scales, **HYPER)
    mv, vv = optim.adamw_state_values(m, v, scales)
    for t in (mv[0], vv[0]):
        assert bool(torch.isnan(t[256:512]).all()) and bool(torch.isnan(t[768:]).all())
        assert bool(torch.isfinite(t[:256]).all()) and bool(torch.isfinite(t[512:768]).all())
    good = torch.isfinite(q)
    assert bool(torch.isfinite(p[good]).all()) and bool(torch.isnan(p[300]))
    fine = torch.arange(n, device=DEV)
    fine = (fine < 256) | ((fine >= 512) & (fine < 768))
    S = scales[0].double().repeat_interleave(256, dim=0)[:n]
    c = m[0].double()
    close(mv[0][fine], (c * c.abs() * S[:, 0] / 127 ** 2)[fine], U * mv[0][fine].abs())
    close(vv[0][fine], ((v[0].double() / 255) ** 4 * S[:, 1])[fine], U * vv[0][fine].abs())
    assert bool((v[0][good & fine & (q != 0)] > 0).all())                   # a positive second moment never becomes 0


def test_adamw_zero_gradients():
    for bits in (32, 8):
        p = torch.full((300,), 2.0, device=DEV)
        m, v, scales, _ = new_states([300], F32, bits, False, [p])
        optim.adamw_step([p], [torch.zeros(300, device=DEV)], m, v, torch.zeros(1, device=DEV), scales=scales, **HYPER)
        close(p, torch.full((300,), 2.0 * (1 - HYPER["lr"] * HYPER["weight_decay"])).double(), 4 * U * 2)
        assert not bool(m[0].any()) and not bool(v[0].any())


def test_adamw_refusals():
    p = torch.ones(10, device=DEV)
    s = torch.zeros(1, device=DEV)
    f = lambda n, t=F32: torch.zeros(n, dtype=t, device=DEV)   # noqa: E731
    ok = dict(params=[p], grads=[f(10)], exp_avgs=[f(10)], exp_avg_sqs=[f(10)], steps=s, lr=1e-3)
    codes = dict(exp_avgs=[f(10, torch.int8)], exp_avg_sqs=[f(10, torch.uint8)], scales=[torch.zeros(1, 2, device=DEV)])
    optim.adamw_step(**ok)
    optim.adamw_step(**{**ok, **codes})
    for bad in (dict(grads=[f(9)]), dict(grads=[f(10, F16)]), dict(exp_avgs=[f(11)]), dict(exp_avg_sqs=[f(10, F16)]), dict(steps=f(2)),
                dict(steps=f(1, F16)), dict(steps=s.cpu()), dict(grads=[f(20)[::2]]), dict(params=[f(10, torch.float64)]), dict(masters=[f(10)]),
                dict(betas=(1.0, 0.9)), dict(lr=torch.tensor(1e-3)), dict(grads=[f(10).cpu()]), {**codes, "scales": [f(2)]},
                {**codes, "exp_avgs": [f(10)]}, dict(params=[p, p], grads=[f(10)] * 2, exp_avgs=[f(10), f(10)], exp_avg_sqs=[f(10), f(10)], steps=f(2))):
        with pytest.raises(SocmxError):
            optim.adamw_step(**{**ok, **bad})


def optimiser_run(make, kind, n_steps=6, skip=None):
    g = gen(21)
    params = [torch.nn.Parameter((0.1 * torch.randn(s, generator=g)).to(kind).to(DEV)) for s in ((17, 9), (300,), (1,), (40, 3, 5))]
    opt = make([dict(params=params[:2]), dict(params=params[2:], lr=3e-3, weight_decay=0.0)])
    for t in range(n_steps):
        for i, p in enumerate(params):
            grad = torch.randn(p.shape, generator=g).to(kind).to(DEV)
            p.grad = None if skip == (t, i) else grad
        opt.step()
    return params, opt


def test_adamw_class_follows_the_rule_of_torch():
    kw = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-6, weight_decay=0.1)
    for skip in (None, (2, 1)):
        a, opt = optimiser_run(lambda g: optim.AdamW(g, **kw), F32, skip=skip)
        b, ref = optimiser_run(lambda g: torch.optim.AdamW(g, **kw), F32, skip=skip)
        for p, q in zip(a, b):
            # 24 roundings of each of six updates, none of which is longer than 3 lr (both sides have them)
            close(p, q.detach(), 2 * 6 * U * (3 * q.detach().abs().double().cpu() + 24 * 3e-2))
            assert float(opt.state[p]["step"]) == float(ref.state[q]["step"])


@pytest.mark.parametrize("kind,bits", [(F32, 8), (BF16, 32), (BF16, 8)])
def test_adamw_class_state_travels(kind, bits):
    """A run that is saved and loaded in the middle ends with the same bits."""
    make = lambda g: optim.AdamW(g, lr=1e-2, state_bits=bits)   # noqa: E731
    a, opt = optimiser_run(make, kind)
    g = gen(99)
    grads = [[torch.randn(p.shape, generator=g).to(kind).to(DEV) for p in a] for _ in range(3)]
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    other = make([dict(params=b[:2]), dict(params=b[2:])])
    import io
    f = io.BytesIO()
    torch.save(opt.state_dict(), f)
    f.seek(0)
    other.load_state_dict(torch.load(f, weights_only=True))
    for ps, o in ((a, opt), (b, other)):
        for row in grads:
            for p, q in zip(ps, row):
                p.grad = q
            o.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        for k, v in opt.state[p].items():
            assert torch.equal(v, other.state[q][k]) and v.dtype == other.state[q][k].dtype, k
    assert opt.state[a[0]]["exp_avg"].dtype == (F32 if bits == 32 else torch.int8)
    assert ("master" in opt.state[a[0]]) == (kind != F32)


def test_adamw_class_captured_steps_are_counted():
    kw = dict(lr=1e-2, weight_decay=0.1, state_bits=8)
    g = gen(31)
    start, grads = torch.randn(1000, generator=g), torch.randn(8, 1000, generator=g)

    def setup():
        p = torch.nn.Parameter(start.to(DEV))
        p.grad = torch.zeros(1000, device=DEV)
        return p, optim.AdamW([p], **kw)
    p, opt = setup()
    for q in grads:
        p.grad.copy_(q)
        opt.step()
    c, copt = setup()
    fresh = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with pytest.raises(SocmxError, match="before it"):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(fresh, stream=side):
            copt.step()
    c, copt = setup()
    c.grad.copy_(grads[0])
    copt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        copt.step()
    for q in grads[1:]:
        c.grad.copy_(q)
        graph.replay()
        torch.cuda.synchronize()
        torch.zeros(64, device=DEV).add_(1)                     # (the program's own work between replays)
    assert torch.equal(p, c) and float(copt.state[c]["step"]) == 8.0
    for k, v in opt.state[p].items():
        assert torch.equal(v, copt.state[c][k])


# ---- together ----------------------------------------------------------------------------------------------------------------
class Recurrent(torch.nn.Module):
    """A control with a memory along the trajectory: norm, gates and inputs, scan, norm, read-out."""

    def __init__(self, d, width, gates, norm, scan):
        super().__init__()
        self.inner, self.gate, self.out = (torch.nn.Linear(i, o, bias=False) for i, o in ((d, width), (d, gates), (width, d)))
        self.w1, self.b1 = torch.nn.Parameter(torch.ones(d)), torch.nn.Parameter(torch.zeros(d))
        self.w2, self.b2 = torch.nn.Parameter(torch.ones(width)), torch.nn.Parameter(torch.zeros(width))
        self.h0 = torch.nn.Parameter(torch.zeros(1, width))
        self.norm, self.scan = norm, scan

    def forward(self, x):
        n = self.norm(x, self.w1, self.b1)
        h, _ = self.scan(self.inner(n), torch.nn.functional.logsigmoid(self.gate(n)), self.h0.expand(x.shape[1], -1))
        return self.out(self.norm(h, self.w2, self.b2))


def plain_norm(x, w, b):
    return (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt() * w + b


def plain_scan(x, a, h0):
    a = a.exp().repeat_interleave(x.shape[2] // a.shape[2], dim=2)
    h, out = h0, []
    for t in range(x.shape[0]):
        h = a[t] * h + x[t]
        out.append(h)
    return torch.stack(out), h


def together(seed=3):
    torch.manual_seed(seed)
    net = Recurrent(10, 96, 8, layers.layer_norm, layers.gated_scan).to(DEV)
    x = torch.randn(51, 16, 10, generator=gen(seed)).to(DEV)
    target = torch.randn(51, 16, 10, generator=gen(seed + 1)).to(DEV)
    return net, x, target


def test_a_recurrent_layer_s_gradients():
    net, x, target = together()
    torch.manual_seed(3)
    ref = Recurrent(10, 96, 8, plain_norm, plain_scan).double()
    loss = (net(x) - target).square().mean()
    want = (ref(x.double().cpu()) - target.double().cpu()).square().mean()
    got = torch.autograd.grad(loss, list(net.parameters()))
    exp = torch.autograd.grad(want, list(ref.parameters()))
    assert abs(float(loss) - float(want)) < 1e-5 * float(want)
    for (name, _), p, q in zip(net.named_parameters(), got, exp):
        # float32 throughout: sums over 816 rows of terms whose factors carry some tens of roundings
        assert float((p.double().cpu() - q).norm()) <= 2e-4 * float(q.norm()) + 1e-9, name


@pytest.mark.parametrize("bits", [32, 8])
def test_a_recurrent_layer_s_training_step_captured(bits):
    """Norm, scan, their gradients and AdamW in one graph, replayed: the same bits as the steps run one by one.  While an eager graph of
    the same parameters from another stream is alive the capture is refused."""
    def step(net, opt, x, target):
        params = list(net.parameters())
        out = net(x)                                           # (no library sum over many blocks in the graph: d loss / d out by hand)
        for p, g in zip(params, torch.autograd.grad(out, params, 2 * (out.detach() - target) / out.numel())):
            p.grad = g
        opt.step()

    def setup():
        net, x, target = together()
        return net, optim.AdamW(net.parameters(), lr=1e-2, state_bits=bits), x, target
    net, opt, x, target = setup()
    for _ in range(6):
        step(net, opt, x, target)
    cap, copt, x, target = setup()
    alive = (cap(x) - target).square().mean()                  # an eager graph of the same leaves
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(cap, copt, x, target)
    torch.cuda.current_stream().wait_stream(side)
    with pytest.raises(SocmxError, match="alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            cap(x)                                             # (refused before any backward)
    assert float(alive) > 0
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(cap, copt, x, target)
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        (net(x) - target).square().mean().item()               # (eager work between the replays)
    for (name, p), q in zip(net.named_parameters(), cap.parameters()):
        assert torch.equal(p, q), name


def test_other_streams_and_two_calls_at_once():
    """Two streams run the operators at the same time on inputs of their own: the same bits as one after the other."""
    cases = []
    for seed in (1, 2):
        x, a, initial, dh, dfinal = scan_case(1200, 1, 60, 60, seed)
        cases.append([t.to(DEV).requires_grad_() for t in (x, a, initial)] + [dh.to(DEV), dfinal.to(DEV)])

    def once(x, a, initial, dh, dfinal):
        h, final = layers.gated_scan(layers.layer_norm(x), a, initial)
        return [h, final] + list(torch.autograd.grad([h, final], [x, a, initial], [dh, dfinal]))
    want = [once(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [None, None]
    for _ in range(5):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i] = once(*c)
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(w, g))


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_the_trainer_with_adamw(graph, bits):
    """make_optimizer(weight_decay, state_bits) through Trainer.step, eager and replayed: every parameter is stepped and stays finite, and in 32
    bits, on the same noise, they follow torch's AdamW on the same groups."""
    from test_host_cpu import build_sde
    from SOC_matching.method import SOC_Solver
    from socmx.train import Trainer, make_optimizer

    def run(own):
        torch.manual_seed(0)
        sde, aux = build_sde("tiny_double_well_d10", DEV)
        solver = SOC_Solver(sde, aux["x0"], None, T=aux["T"], num_steps=aux["K"], lmbd=aux["lmbd"], d=aux["d"], sigma=sde.sigma)
        opt = make_optimizer(solver, nabla_V_lr=1e-3, M_lr=1e-3, weight_decay=0.05, state_bits=bits)
        assert type(opt) is optim.AdamW
        if not own:
            opt = torch.optim.AdamW([{k: v for k, v in g.items() if k in ("params", "lr", "weight_decay")} for g in opt.param_groups],
                                    eps=opt.param_groups[0]["eps"])
        tr = Trainer(solver, opt, aux["B"], normalization_const=0.8, hip_graph=graph and own)
        modes = []
        for _ in range(6):
            if not graph:
                solver.noise_in = aux["noise"]                 # (a rollout consumes it: without it two runs of one optimiser differ)
            modes.append(tr.step()["mode"])
        tr.join()
        torch.cuda.synchronize()
        return sde, opt, modes
    sde, opt, modes = run(True)
    if graph:
        assert "graph-replay" in modes, modes
    counts = {float(st["step"]) for st in opt.state.values()}
    assert counts == {6.0}, counts
    assert all(bool(torch.isfinite(p).all()) for p in sde.parameters())
    if bits == 32 and not graph:
        ref, _, _ = run(False)
        for (name, p), q in zip(sde.named_parameters(), ref.parameters()):
            # six steps of at most 1e-3 each, whose gradients agree to about 1e-4: where a gradient is near nothing the direction is free
            assert float((p - q).abs().max()) <= 6 * 1e-3 * 0.05 + 1e-6 * float(q.abs().max()), name


def test_gated_scan_in_chunks_captured():
    """A sequence of several chunks, forward and backward in one graph, replayed with other inputs: every replay equals the eager call."""
    cases = [[t.to(DEV) for t in scan_case(1500, 2, 96, 3, seed, BF16, F32, resets=0.002)] for seed in range(4)]
    lengths = torch.tensor([1500, 1111], dtype=torch.int32, device=DEV)

    def once(x, a, initial, dh, dfinal):
        ts = [t.detach().requires_grad_() for t in (x, a, initial)]
        h, final = layers.gated_scan(*ts, lengths=lengths)
        return [h.detach(), final.detach()] + list(torch.autograd.grad([h, final], ts, [dh, dfinal]))
    want = [[t.clone() for t in once(*c)] for c in cases]
    held = [t.clone() for t in cases[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = once(*held)
    for i in (0, 1, 2, 3, 1, 0):
        for t, c in zip(held, cases[i]):
            t.copy_(c)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want[i])), i
        assert all(torch.equal(p, q) for p, q in zip(once(*cases[3 - i]), want[3 - i])), i


@pytest.mark.parametrize("kind", [F32, BF16])
def test_rows_further_apart_than_32_bits_count(kind):
    """Rows 2^31 elements and more apart, as in a slice of a large buffer."""
    far = 2 ** 31 + 640
    big = torch.zeros(2 * far + 4096, dtype=kind, device=DEV)
    x, a, initial, dh, dfinal = scan_case(150, 3, 16, 2, 77, kind, F32)
    wide = big.as_strided((150, 3, 16), (20, far, 1))
    wide.copy_(x)
    scan_check(wide, a.to(DEV), initial, dh.to(DEV), dfinal)
    rows = big.as_strided((3, 1000), (far, 1))
    rows.copy_(dh.reshape(-1)[:3000].reshape(3, 1000))
    w, b = torch.ones(1000, device=DEV), torch.zeros(1000, device=DEV)
    assert torch.equal(layers.layer_norm(rows, w, b), layers.layer_norm(rows.contiguous(), w, b))


def test_adamw_8_bit_beyond_32_bit_offsets():
    """The last 1000 of 2^32 + 1000 elements get the codes of the first 1000 of a small tensor: thresholds repeat after 2^32 elements."""
    n, tail = 2 ** 32 + 1000, 1000
    g = gen(3)
    grad, start = (0.1 * torch.randn(tail, generator=g)).to(BF16), torch.randn(tail, generator=g).to(BF16)
    p, q = (torch.zeros(n, dtype=BF16, device=DEV) for _ in range(2))
    m, v, scales, _ = new_states([n], BF16, 8, False, [p])
    ps, qs = start.to(DEV), grad.to(DEV)
    ms, vs, small, _ = new_states([tail], BF16, 8, False, [ps])
    p[-tail:], q[-tail:] = ps, qs
    steps = [torch.zeros(1, device=DEV) for _ in range(2)]
    for _ in range(2):
        optim.adamw_step([p], [q], m, v, steps[0], scales=scales, **HYPER)
        optim.adamw_step([ps], [qs], ms, vs, steps[1], scales=small, **HYPER)
    for wide, narrow in ((p, ps), (m[0], ms[0]), (v[0], vs[0])):
        assert torch.equal(wide[-tail:], narrow) and not bool(wide[:tail].any()) and not bool(wide[2 ** 31:2 ** 31 + tail].any())
    assert torch.equal(scales[0][-4:], small[0])


def test_what_is_written_in_place_is_seen_by_autograd():
    w = torch.ones(4, device=DEV, requires_grad=True)
    state, one = torch.ones(2, 4, device=DEV), torch.ones(2, 4, device=DEV)
    y = (w * state).sum()
    layers.gated_scan_step(state, one, one)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()
    y = (w * w).sum()
    with torch.no_grad():
        optim.adamw_step([w], [torch.ones_like(w)], *new_states([4], F32, 32, False, [w])[:2], torch.zeros(1, device=DEV), lr=1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


def test_adamw_refuses_shared_states():
    f = lambda t=F32: torch.zeros(10, dtype=t, device=DEV)   # noqa: E731
    one = f()
    ok = dict(params=[f(), f()], grads=[one, one], exp_avgs=[f(), f()], exp_avg_sqs=[f(), f()], steps=torch.zeros(2, device=DEV), lr=1e-3)
    optim.adamw_step(**ok)                                     # (a gradient is only read: it may be shared)
    for bad in (dict(exp_avgs=[one, one]), dict(exp_avgs=[one, f()], exp_avg_sqs=[f(), one]), dict(exp_avg_sqs=ok["params"])):
        with pytest.raises(SocmxError, match="another tensor's"):
            optim.adamw_step(**{**ok, **bad})


@pytest.mark.parametrize("size", [1e-18, 1e-20])
def test_adamw_of_tiny_gradients_without_eps(size):
    """The first update is lr whatever the gradient's size.  v = 5e-42 at 1e-20 is 3600 of float32's smallest numbers: g g, its product and
    the sum are off by half of one each, 2e-4 of v, half of that of its root."""
    p, g = torch.zeros(300, device=DEV), torch.full((300,), size, device=DEV)
    m, v, _, _ = new_states([300], F32, 32, False, [p])
    optim.adamw_step([p], [g], m, v, torch.zeros(1, device=DEV), lr=1e-2, betas=(0.9, 0.95), eps=0.0, weight_decay=0.0)
    close(p, torch.full((300,), -1e-2).double(), 1e-2 * (30 * U + (2.1e-4 if size < 1e-19 else 0)))
