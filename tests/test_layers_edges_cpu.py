"""Layer operators and AdamW at the edges, without a GPU: torch's other modes, what an optimiser keeps, what the C entry points check."""
import ctypes as C

import pytest
import torch

from socmx import _lib, layers, optim
from socmx._lib import SocmxError


def _adamw(rows):
    flat = [w for row in rows for w in row]
    return (C.c_int64 * len(flat))(*flat)


def test_adamw_keeps_step_counts_where_they_are(monkeypatch):
    """A captured step holds the addresses of the counts: a step in which a parameter has no gradient must not move them."""
    calls = []

    class Binding:
        def adamw_step_counts(self, params, grads, ms, vs, steps, *rest):
            calls.append([s.data_ptr() for s in steps])
            for s in steps:
                s += 1
    monkeypatch.setattr(_lib, "torch_binding", lambda: Binding())
    params = [torch.nn.Parameter(torch.zeros(n)) for n in (3, 5, 7)]
    opt = optim.AdamW(params)
    for p in params:
        opt.state[p] = dict(step=torch.zeros(()), exp_avg=torch.zeros(p.shape), exp_avg_sq=torch.zeros(p.shape))
    held = [opt.state[p]["step"] for p in params]
    for missing in (None, 1, None, 0, None):
        for i, p in enumerate(params):
            p.grad = None if i == missing else torch.ones(p.shape)
        opt.step()
        assert all(opt.state[p]["step"] is s for p, s in zip(params, held))
    at = [s.data_ptr() for s in held]
    assert calls == [at, [at[0], at[2]], at, at[1:], at]
    assert [float(s) for s in held] == [4.0, 4.0, 5.0]


def test_adamw_step_counts_entry_checks():
    L = _lib.lib()
    hyper = (1e-3, 0.9, 0.999, 1e-8, 0.01)
    row = (1, 1, 1, 1, 1, 0, 10)
    counts = lambda *v: (C.c_int64 * len(v))(*v)   # noqa: E731
    assert L.socmx_adamw_step_counts(0, 32, _adamw([row]), 1, None, 1, *hyper, None) == -1
    assert L.socmx_adamw_step_counts(0, 32, _adamw([row, row]), 2, counts(1, 0), 1, *hyper, None) == -1
    assert L.socmx_adamw_step_counts(0, 16, _adamw([row]), 1, counts(1), 1, *hyper, None) == -3
    assert L.socmx_adamw_step_counts(0, 32, _adamw([row]), 0, counts(1), 1, *hyper, None) == -2
    p = torch.zeros(5)
    with pytest.raises(SocmxError, match="1 params and 2 steps"):
        optim.adamw_step([p], [p], [p], [p], [p, p], lr=1e-3)
    with pytest.raises(SocmxError, match="no CPU path"):
        optim.adamw_step([p], [p], [p], [p], [torch.zeros(())], lr=1e-3)


def test_forward_mode_derivatives_are_refused():
    import torch.autograd.forward_ad as fwad
    x, a = torch.zeros(4, 2, 6), torch.zeros(4, 2, 3)
    p = torch.zeros(5)
    with fwad.dual_level():
        dual = lambda t: fwad.make_dual(t, torch.ones_like(t))   # noqa: E731
        for call in (lambda: layers.layer_norm(dual(x)), lambda: layers.layer_norm(x, bias=dual(x[0, 0])), lambda: layers.gated_scan(x, dual(a)),
                     lambda: layers.gated_scan(x, a, dual(x[0])), lambda: layers.gated_scan_step(x[0], dual(x[0]), a[0])):
            with pytest.raises(SocmxError, match="forward-mode"):
                call()
        with pytest.raises(SocmxError, match="no CPU path"):
            layers.layer_norm(x)


def test_tracing_is_refused():
    """(In front of every other check: on the CPU too the reason is the trace.)"""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, a, codes = torch.zeros(4, 2, 6), torch.zeros(4, 2, 3), torch.zeros(5, dtype=torch.int8)

    def adamw(x):
        optim.adamw_step([x], [x], [x], [x], torch.zeros(1), lr=1e-3)
        return x

    def values(x):
        return optim.adamw_state_values([codes], [codes.to(torch.uint8)], [torch.zeros(1, 2)])[0][0]
    for f, args in ((lambda x: layers.layer_norm(x), (x,)), (lambda x, a: layers.gated_scan(x, a)[0], (x, a)),
                    (lambda x, a: layers.gated_scan_step(x[0].clone(), x[0], a[0]), (x, a)), (adamw, (x,)), (values, (x,))):
        with pytest.raises(SocmxError, match="cannot be traced"):
            torch.jit.trace(f, args, check_trace=False)
        with pytest.raises(SocmxError, match="cannot be traced"):
            make_fx(f)(*args)


def test_adamw_refuses_what_a_launch_cannot_count():
    """A launch counts its threads in 32 bits: 2^24 - 1 workgroups of 256, 4096 elements each.  Refused before anything is launched."""
    L = _lib.lib()
    hyper = (1e-3, 0.9, 0.999, 1e-8, 0.01)
    most = 4096 * (2 ** 24 - 1)
    for n in (most + 1, 2 ** 37, 2 ** 40, 2 ** 62):
        assert L.socmx_adamw_step(0, 32, _adamw([(1, 1, 1, 1, 1, 0, 5), (1, 1, 1, 1, 1, 0, n)]), 2, 1, 1, *hyper, None) == -2
        assert L.socmx_adamw_state_values(_adamw([(1, 1, 1, 1, 1, n)]), 1, None) == -2


def test_adamw_takes_a_state_of_torch():
    """Its groups have no state_bits and no master_weights: the defaults of the optimiser that loads them.  What the rule does not have is refused."""
    params = [torch.nn.Parameter(torch.zeros(n)) for n in (3, 4)]
    params[0].grad = torch.ones(3)

    def torch_state(**kw):
        ref = torch.optim.AdamW(params, lr=1e-2, **kw)
        ref.step()
        return ref.state_dict()
    for bits in (32, 8):
        opt = optim.AdamW(params, lr=1e-3, state_bits=bits)
        opt.load_state_dict(torch_state())
        group, = opt.param_groups
        assert group["lr"] == 1e-2 and group["state_bits"] == bits and group["master_weights"] is True
        assert set(opt.state[params[0]]) == {"step", "exp_avg", "exp_avg_sq"} and params[1] not in opt.state
    before = optim.AdamW(params, lr=1e-3)
    for name in ("amsgrad", "maximize"):
        with pytest.raises(SocmxError, match=name):
            before.load_state_dict(torch_state(**{name: True}))
    assert before.param_groups[0]["lr"] == 1e-3 and not before.state
