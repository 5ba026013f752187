"""Layer operators and AdamW without a GPU: what they refuse, and what the C entry points check before any launch."""
import ctypes as C

import pytest
import torch

from socmx import _lib, layers, optim
from socmx._lib import SocmxError


def _scan(**kw):
    d = dict(type=0, gate_type=0, T=4, B=2, D=6, G=3)
    d.update(kw)
    return _lib.Scan(**d)


def _adamw(rows):
    flat = [w for row in rows for w in row]
    return (C.c_int64 * len(flat))(*flat)


def test_cpu_tensors_are_refused():
    x = torch.zeros(3, 4, 6)
    with pytest.raises(SocmxError, match="no CPU path"):
        layers.layer_norm(x)
    with pytest.raises(SocmxError, match="no CPU path"):
        layers.gated_scan(x, x)
    with pytest.raises(SocmxError, match="no CPU path"):
        layers.gated_scan_step(x[0], x[0], x[0])
    p = torch.zeros(5)
    with pytest.raises(SocmxError, match="no CPU path"):
        optim.adamw_step([p], [p], [p], [p], torch.zeros(1), lr=1e-3)
    with pytest.raises(SocmxError, match="no CPU path"):
        optim.adamw_state_values([p.to(torch.int8)], [p.to(torch.uint8)], [torch.zeros(1, 2)])
    q = torch.nn.Parameter(torch.zeros(5))
    q.grad = torch.ones(5)
    with pytest.raises(SocmxError, match="no CPU path"):
        optim.AdamW([q]).step()


@pytest.mark.parametrize("kw", [dict(lr=-1.0), dict(eps=-1.0), dict(weight_decay=-0.1), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)),
                                dict(state_bits=16), dict(lr=float("nan"))])
def test_adamw_refuses_hyper_parameters(kw):
    with pytest.raises(SocmxError):
        optim.AdamW([torch.nn.Parameter(torch.zeros(2))], **kw)


def test_adamw_step_refuses_lists_of_different_lengths():
    p = torch.zeros(5)
    with pytest.raises(SocmxError, match="1 params and 2 grads"):
        optim.adamw_step([p], [p, p], [p], [p], torch.zeros(1), lr=1e-3)
    with pytest.raises(SocmxError, match="masters"):
        optim.adamw_step([p], [p], [p], [p], torch.zeros(1), lr=1e-3, masters=[])
    optim.adamw_step([], [], [], [], torch.zeros(0), lr=1e-3)            # nothing to do


def test_layer_norm_entry_checks():
    L = _lib.lib()
    ok = [0, 0, 1, 4, 8, 8, None, None, 1e-5, 1, None, None, None]

    def call(**kw):
        a = list(ok)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return L.socmx_layer_norm_fwd(*a)
    assert call(_2=None) == -1 and call(_9=None) == -1 and call(_10=1) == -1         # x, y, mean without rstd
    assert call(_0=3) == -3 and call(_0=1, _1=2) == -3 and call(_0=0, _1=1) == -3    # types
    assert call(_3=0) == -2 and call(_4=0) == -2 and call(_4=(1 << 24) + 1) == -2    # sizes
    assert L.socmx_layer_norm_bwd(0, 0, 1, 4, 8, 8, 1, 8, None, 1, 1, None, None, None, None, None) == -1   # nothing wanted
    assert L.socmx_layer_norm_bwd(0, 0, 1, 4, 8, 8, 1, 8, None, 1, 1, None, 1, None, None, None) == -4      # no workspace
    assert L.socmx_layer_norm_bwd(0, 0, 1, 4, 8, 8, 1, 8, None, None, 1, 1, None, None, None, None) == -1
    assert L.socmx_layer_norm_bwd_workspace_floats(0, 0, 8) == 0
    for rows, cols in ((1, 1), (7, 10), (25728, 256), (100, 16384), (100, 20000), (3, 1 << 24)):
        n = L.socmx_layer_norm_bwd_workspace_floats(1, rows, cols)
        assert n % (2 * cols) == 0 and 1 <= n // (2 * cols) <= 512


def test_gated_scan_entry_checks():
    L = _lib.lib()
    n = [C.c_int64() for _ in range(3)]
    refs = [C.byref(v) for v in n]
    assert L.socmx_gated_scan_sizes(None, *refs) == -1
    assert L.socmx_gated_scan_sizes(C.byref(_scan()), refs[0], refs[1], None) == -1
    for bad in (dict(T=0), dict(B=0), dict(D=0), dict(G=0), dict(G=4), dict(T=(1 << 30) + 1), dict(B=1 << 20, D=1 << 13, G=1)):
        assert L.socmx_gated_scan_sizes(C.byref(_scan(**bad)), *refs) == -2, bad
    for bad in (dict(type=3), dict(type=0, gate_type=1), dict(type=2, gate_type=1), dict(type=-1)):
        assert L.socmx_gated_scan_sizes(C.byref(_scan(**bad)), *refs) == -3, bad
    assert L.socmx_gated_scan_sizes(C.byref(_scan()), *refs) == 0
    assert n[0].value >= 2 * 6 and n[1].value == 0 and n[2].value == 0               # short: one launch, no workspace
    s = _scan()
    assert L.socmx_gated_scan_fwd(C.byref(s), None, 1, None, 1, 0, 0, None, None, None, None) == -1
    assert L.socmx_gated_scan_bwd(C.byref(s), 1, 1, None, None, 0, 0, None, 1, 0, 0, 1, 0, 0, None, None, None) == -1
    # few channels, long time: chunks, whose runs need a workspace; a gate wider than a wave needs one in the backward
    s = _scan(T=100000, B=1, D=64, G=64)
    assert L.socmx_gated_scan_sizes(C.byref(s), *refs) == 0 and n[1].value > 0 and n[2].value > 0
    assert L.socmx_gated_scan_fwd(C.byref(s), 1, 1, None, 1, 0, 0, None, None, None, None) == -4
    assert L.socmx_gated_scan_bwd(C.byref(s), 1, 1, 1, None, 0, 0, None, 1, 0, 0, 1, 0, 0, None, None, None) == -4
    s = _scan(T=4, B=1, D=1000, G=1)
    assert L.socmx_gated_scan_sizes(C.byref(s), *refs) == 0 and n[2].value >= 4
    assert L.socmx_gated_scan_bwd(C.byref(s), 1, 1, 1, None, 0, 0, None, 1, 0, 0, 1, 0, 0, None, None, None) == -4
    assert L.socmx_gated_scan_step(0, 0, 2, 6, 4, 1, 6, 1, 3, 1, 6, 1, None) == -2
    assert L.socmx_gated_scan_step(0, 1, 2, 6, 3, 1, 6, 1, 3, 1, 6, 1, None) == -3
    assert L.socmx_gated_scan_step(0, 0, 2, 6, 3, 1, 6, 1, 3, None, 6, 1, None) == -1


def test_adamw_entry_checks():
    L = _lib.lib()
    hyper = (1e-3, 0.9, 0.999, 1e-8, 0.01)
    row = (1, 1, 1, 1, 1, 0, 10)
    call = lambda row=row, type=0, bits=32, n=1, steps=1, ws=1, hyper=hyper: L.socmx_adamw_step(   # noqa: E731
        type, bits, _adamw([row]), n, steps, ws, *hyper, None)
    assert call(steps=None) == -1 and call(ws=None) == -1 and L.socmx_adamw_step(0, 32, None, 1, 1, 1, *hyper, None) == -1
    assert call(type=3) == -3 and call(bits=16) == -3 and call(row=(1, 1, 1, 1, 0, 1, 10)) == -3            # f32 with a master
    assert call(n=0) == -2 and call(row=row[:6] + (-1,)) == -2
    assert call(hyper=(1e-3, 1.0, 0.999, 1e-8, 0.0)) == -2 and call(hyper=(1e-3, 0.9, float("nan"), 1e-8, 0.0)) == -2
    for i in range(4):
        assert call(row=row[:i] + (0,) + row[i + 1:]) == -1
    assert call(row=(1, 1, 1, 1, 0, 0, 10), bits=8) == -1                                                    # 8 bits without scales
    assert L.socmx_adamw_state_values(None, 1, None) == -1
    assert L.socmx_adamw_state_values(_adamw([(1, 1, 1, 1, 1, 10)]), 0, None) == -2
    assert L.socmx_adamw_state_values(_adamw([(1, 1, 0, 1, 1, 10)]), 1, None) == -1


def test_make_optimizer_takes_adamw_only_when_asked():
    from test_host_cpu import build_sde
    from SOC_matching.method import SOC_Solver
    from socmx.train import make_optimizer
    sde, aux = build_sde("tiny_double_well_d10", "cpu")
    solver = SOC_Solver(sde, aux["x0"], None, T=aux["T"], num_steps=aux["K"], lmbd=aux["lmbd"], d=aux["d"], sigma=sde.sigma)
    assert type(make_optimizer(solver)) is torch.optim.Adam
    opt = make_optimizer(solver, weight_decay=0.1)
    assert type(opt) is torch.optim.AdamW
    decays = {id(p): g["weight_decay"] for g in opt.param_groups for p in g["params"]}
    assert decays[id(sde.gamma)] == 0.0
    assert decays[id(sde.nabla_V.down_0[0].weight)] == 0.1 and decays[id(sde.M.sigmoid_layers[0].weight)] == 0.1
    lrs = {id(p): g["lr"] for g in opt.param_groups for p in g["params"]}
    ref = {id(p): g["lr"] for g in make_optimizer(solver).param_groups for p in g["params"]}
    assert lrs == ref
    with pytest.raises(ValueError, match="8 bits"):
        make_optimizer(solver, state_bits=8)
    for bits in (0, 16):
        with pytest.raises(ValueError, match="8 or 32"):
            make_optimizer(solver, state_bits=bits)


def test_the_configuration_has_the_adamw_keys_off():
    from socmx.config import load_config
    cfg = load_config()
    assert cfg.optim.weight_decay == 0.0 and cfg.optim.state_bits is None
    cfg = load_config(["optim.weight_decay=0.05", "optim.state_bits=8"])
    assert cfg.optim.weight_decay == 0.05 and cfg.optim.state_bits == 8
