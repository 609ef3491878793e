"""CPU: refusals and host logic of the training-step operators (layer normalisation, Newton-Schulz orthogonalisation, Muon)."""
import ctypes

import pytest
import torch


def _ns(nat, **kw):
    return nat.newton_schulz(**kw)


def _ptrs(*values):
    return (ctypes.c_void_p * len(values))(*values)


ONE = ctypes.c_void_p(4096)


def _norm_fwd(lib, x=ONE, xs=8, dt=0, w=None, b=None, wdt=0, rows=4, cols=8, eps=1e-5, y=ONE, mean=None, rstd=None):
    return lib.cnf_layer_norm_fwd(x, xs, dt, w, b, wdt, rows, cols, eps, y, mean, rstd, None)


@pytest.mark.parametrize("kw, words", [
    (dict(dt=3), b"unsupported types"), (dict(dt=-1), b"unsupported types"), (dict(dt=0, wdt=1), b"unsupported types"),
    (dict(dt=1, wdt=2), b"unsupported types"), (dict(rows=-1), b"rows >= 0"), (dict(cols=0), b"cols > 0"), (dict(cols=-3), b"cols > 0"),
    (dict(rows=1 << 40, cols=1 << 40), b"need rows"), (dict(xs=-8), b"row stride"), (dict(xs=1 << 60), b"row stride"),
    (dict(x=None), b"x must be given"), (dict(x=ctypes.c_void_p(4097)), b"aligned"), (dict(w=ctypes.c_void_p(4098)), b"aligned"),
    (dict(y=None), b"y must be given"), (dict(mean=ctypes.c_void_p(4097)), b"aligned"), (dict(eps=-1.0), b"eps"),
    (dict(eps=float("nan")), b"eps"), (dict(eps=float("inf")), b"eps")])
def test_layer_norm_fwd_refuses(kw, words):
    from gan_flow_amd import _native as nat
    lib = nat.load_library()
    assert _norm_fwd(lib, **kw) != 0 and words in lib.cnf_last_error()


def test_layer_norm_of_no_rows_enqueues_nothing():
    from gan_flow_amd import _native as nat
    lib = nat.load_library()
    assert _norm_fwd(lib, rows=0) == 0
    assert lib.cnf_layer_norm_workspace_bytes(0, 64) == 0 and lib.cnf_layer_norm_workspace_bytes(64, 0) == 0
    assert lib.cnf_layer_norm_workspace_bytes(1, 64) >= 2 * 64 * 4


def _norm_bwd(lib, dy=ONE, dys=8, x=ONE, xs=8, dt=0, w=None, wdt=0, mean=ONE, rstd=ONE, rows=4, cols=8, dx=ONE, dw=ONE, db=ONE, ws=ONE,
              bytes_=1 << 20):
    return lib.cnf_layer_norm_bwd(dy, dys, x, xs, dt, w, wdt, mean, rstd, rows, cols, dx, dw, db, ws, bytes_, None)


@pytest.mark.parametrize("kw, words", [
    (dict(dt=9), b"unsupported types"), (dict(dy=None), b"must be given"), (dict(mean=None), b"must be given"),
    (dict(rstd=None), b"must be given"), (dict(dys=-1), b"row stride"), (dict(dx=None, dw=None, db=None), b"nothing to compute"),
    (dict(dx=ctypes.c_void_p(4097)), b"aligned"), (dict(dw=ctypes.c_void_p(4098)), b"aligned"), (dict(ws=None), b"workspace"),
    (dict(bytes_=8), b"workspace"), (dict(ws=ctypes.c_void_p(4104)), b"workspace")])
def test_layer_norm_bwd_refuses(kw, words):
    from gan_flow_amd import _native as nat
    lib = nat.load_library()
    assert _norm_bwd(lib, **kw) != 0 and words in lib.cnf_last_error()


def _orth(nat, lib, g=None, ldg=8, out=None, ldo=8, dt=0, count=1, rows=4, cols=8, ns=None, ws=ONE, bytes_=1 << 30):
    g = _ptrs(4096) if g is None else g
    out = _ptrs(1 << 20) if out is None else out
    ns = _ns(nat) if ns is None else ns
    return lib.cnf_orthogonalize(g, ldg, out, ldo, dt, count, rows, cols, ctypes.byref(ns), ws, bytes_, None)


@pytest.mark.parametrize("kw, words", [
    (dict(dt=7), b"unsupported type"), (dict(count=0), b"count"), (dict(count=65), b"count"), (dict(rows=0), b"rows and cols"),
    (dict(cols=0), b"rows and cols"), (dict(rows=65537), b"rows and cols"), (dict(ldg=7), b"row stride"), (dict(ldo=-8), b"row stride"),
    (dict(ldg=1 << 60), b"row stride"), (dict(g=_ptrs(0)), b"NULL"), (dict(out=_ptrs(4098)), b"aligned"), (dict(ws=None), b"workspace"),
    (dict(bytes_=16), b"workspace"), (dict(ws=ctypes.c_void_p(4100)), b"workspace")])
def test_orthogonalize_refuses(kw, words):
    from gan_flow_amd import _native as nat
    lib = nat.load_library()
    assert _orth(nat, lib, **kw) != 0 and words in lib.cnf_last_error()


def test_newton_schulz_parameters_are_checked():
    from gan_flow_amd import _native as nat
    lib = nat.load_library()
    for steps in (0, -1, 17):
        with pytest.raises(nat.CnfError):
            _ns(nat, steps=steps)
        ns = _ns(nat)
        ns.steps = steps
        assert _orth(nat, lib, ns=ns) != 0 and b"steps" in lib.cnf_last_error()
    for eps in (0.0, -1e-7, float("nan"), float("inf")):
        assert _orth(nat, lib, ns=_ns(nat, eps=eps)) != 0 and b"eps" in lib.cnf_last_error()
    # polynomials that diverge: growth in one step, growth over the steps, NaN, and a gap between the ends of the interval
    for coef in ((9.0, 0.0, 0.0), (3.0, 0.0, 0.0), (float("nan"), 1.0, 1.0), (0.0, 100.0, -100.0), (1.0, 0.0, float("inf"))):
        assert _orth(nat, lib, ns=_ns(nat, coefficients=coef)) != 0 and b"diverge" in lib.cnf_last_error()
    with pytest.raises(nat.CnfError):
        _ns(nat, steps=3, coefficients=[(1.5, -0.5, 0.0)] * 2)
    with pytest.raises(nat.CnfError):
        _ns(nat, steps=3, coefficients=(1.5, -0.5))
    ns = _ns(nat, steps=2, coefficients=[(1.5, -0.5, 0.0), (3.4445, -4.7750, 2.0315)])
    assert (ns.a[0], ns.a[1], ns.b[0], ns.c[1]) == (1.5, 3.4445, -0.5, 2.0315)
    ns = _ns(nat)
    ns.reserved = 1
    assert _orth(nat, lib, ns=ns) != 0 and b"reserved" in lib.cnf_last_error()


def test_polynomial_bound_holds_on_a_grid():
    """Accepted coefficients keep every singular value in the range the pieces hold: scanned over 20 001 starting values."""
    from gan_flow_amd import _native as nat
    lib = nat.load_library()
    g = torch.Generator().manual_seed(5)
    for _ in range(300):
        coef = [tuple((torch.rand(3, generator=g, dtype=torch.float64) * 8 - 4).tolist()) for _ in range(4)]
        ns = _ns(nat, steps=4, coefficients=coef)
        accepted = _orth(nat, lib, ns=ns, bytes_=16) != 0 and b"workspace" in lib.cnf_last_error()   # (checked after the coefficients)
        u = torch.linspace(0, 1, 20001, dtype=torch.float64)
        worst = 0.0
        for a, b, c in coef:
            u = u * (a + b * u ** 2 + c * u ** 4)
            worst = max(worst, u.abs().max().item())
        if accepted:
            assert worst <= 7.5


@pytest.mark.parametrize("kw", [dict(lr=-1.0), dict(momentum=1.0), dict(momentum=-0.1), dict(weight_decay=-1.0), dict(scale=-1.0),
                                dict(lr=float("nan")), dict(lr=float("inf")), dict(nesterov=2), dict(reserved=1)])
def test_muon_step_refuses_hyper_parameters(kw):
    from gan_flow_amd import _native as nat
    lib = nat.load_library()
    o = nat.CnfMuonOpts(1e-3, 0.95, 0.1, 1.0, 1, 0)
    for k, v in kw.items():
        setattr(o, k, v)
    rc = lib.cnf_muon_step(_ptrs(4096), 8, _ptrs(1 << 20), 8, _ptrs(1 << 21), 8, 0, 1, 4, 8, ctypes.byref(o), ctypes.byref(_ns(nat)), None, ONE,
                           1 << 30, None)
    assert rc != 0 and b"invalid hyper-parameters" in lib.cnf_last_error()


def test_muon_step_refuses_the_same_matrix_twice():
    from gan_flow_amd import _native as nat
    lib = nat.load_library()
    o = nat.CnfMuonOpts(1e-3, 0.95, 0.1, 1.0, 1, 0)
    for p, m in ((_ptrs(4096, 4096), _ptrs(1 << 21, 1 << 22)), (_ptrs(4096, 8192), _ptrs(1 << 21, 1 << 21))):
        rc = lib.cnf_muon_step(p, 8, _ptrs(1 << 20, 1 << 20), 8, m, 8, 0, 2, 4, 8, ctypes.byref(o), ctypes.byref(_ns(nat)), None, ONE, 1 << 30, None)
        assert rc != 0 and b"same parameter" in lib.cnf_last_error()


def test_muon_step_refuses_a_momentum_that_is_something_else():
    from gan_flow_amd import _native as nat
    lib = nat.load_library()
    o = nat.CnfMuonOpts(1e-3, 0.95, 0.1, 1.0, 1, 0)
    for p, g, m in ((_ptrs(4096, 8192), _ptrs(1 << 20, 1 << 21), _ptrs(1 << 22, 1 << 20)), (_ptrs(4096, 8192), _ptrs(1 << 20, 1 << 21), _ptrs(8192, 1 << 22))):
        rc = lib.cnf_muon_step(p, 8, g, 8, m, 8, 0, 2, 4, 8, ctypes.byref(o), ctypes.byref(_ns(nat)), None, ONE, 1 << 30, None)
        assert rc != 0 and b"also a gradient or a parameter" in lib.cnf_last_error()


def test_orthogonalize_refuses_one_output_for_two_matrices():
    from gan_flow_amd import _native as nat
    lib = nat.load_library()
    rc = lib.cnf_orthogonalize(_ptrs(4096, 8192), 8, _ptrs(1 << 20, 1 << 20), 8, 0, 2, 4, 8, ctypes.byref(_ns(nat)), ONE, 1 << 30, None)
    assert rc != 0 and b"same output" in lib.cnf_last_error()


def test_python_entry_points_refuse_host_tensors():
    from gan_flow_amd import CnfError
    from gan_flow_amd.lib.layers import LayerNorm, layer_norm
    from gan_flow_amd.lib.optim import Muon, muon_step, orthogonalize
    x = torch.randn(4, 8)
    with pytest.raises(CnfError, match="HIP device"):
        layer_norm(x)
    with pytest.raises(CnfError, match="HIP device"):
        LayerNorm(8)(x)
    with pytest.raises(CnfError, match="features"):
        LayerNorm(9)(x)
    with pytest.raises(CnfError):
        layer_norm(torch.tensor(1.0))
    with pytest.raises(CnfError, match="HIP device"):
        orthogonalize(x)
    with pytest.raises(CnfError, match="HIP device"):
        muon_step([x], [x], [x.clone()])
    with pytest.raises(CnfError, match="params"):
        muon_step([x], [], [x])
    with pytest.raises(ValueError, match="another optimizer"):
        Muon([torch.nn.Parameter(torch.zeros(4))])
    for bad in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(eps=0.0)):
        with pytest.raises(ValueError):
            Muon([torch.nn.Parameter(x)], **bad)
    with pytest.raises(CnfError):
        Muon([torch.nn.Parameter(x)], adjust_lr="other")
    with pytest.raises(CnfError):
        Muon([torch.nn.Parameter(x)], ns_steps=0)


def test_adjusted_scale():
    from gan_flow_amd.lib.optim import adjusted_scale
    assert adjusted_scale("original", 400, 100) == 2.0 and adjusted_scale("original", 100, 400) == 1.0
    assert adjusted_scale("match_rms_adamw", 100, 400) == pytest.approx(4.0) and adjusted_scale(0.5, 3, 3) == 0.5


def test_layer_norm_module_mirrors_its_arguments():
    from gan_flow_amd.lib.layers import LayerNorm
    m = LayerNorm(12, eps=1e-3)
    assert sorted(m.state_dict()) == ["bias", "weight"] and m.weight.shape == (12,) and "12" in repr(m)
    with torch.no_grad():
        m.weight.zero_(), m.bias.fill_(3.0)
    m.reset_parameters()
    assert m.weight.eq(1).all() and m.bias.eq(0).all()
    assert not list(LayerNorm(12, affine=False).parameters())


@pytest.mark.parametrize("rows, cols", [(130, 260), (260, 130), (512, 640), (700, 500), (1000, 500), (256, 1024), (1024, 4096)])
def test_a_matrix_is_iterated_the_same_way_in_every_stack(rows, cols):
    """Whether steps are taken together (which needs more workspace) is decided by the shape, not by the number of matrices."""
    from gan_flow_amd import _native as nat
    one = nat.matrix_workspace_bytes(1, rows, cols)
    assert [nat.matrix_workspace_bytes(n, rows, cols) for n in (2, 8, 40, 64)] == [n * one for n in (2, 8, 40, 64)]


@pytest.mark.parametrize("which", ["x", "weight", "bias"])
@pytest.mark.parametrize("grad", [True, False])
def test_layer_norm_refuses_dual_tensors(monkeypatch, which, grad):
    """A tangent is not dropped without a word (the kernel's call is replaced: the refusal comes from autograd)."""
    from torch.autograd import forward_ad
    from gan_flow_amd.lib.layers import layer_norm, normalization
    monkeypatch.setattr(normalization._native, "norm_forward", lambda x, w, b, eps, stats: (x.clone(), x.new_zeros(2, len(x)), x, w, x.dtype))
    args = dict(x=torch.randn(3, 8), weight=torch.ones(8), bias=torch.zeros(8))
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        layer_norm(**args)                                     # no tangent: nothing to refuse
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
            layer_norm(**args)


def test_orthogonalize_refuses_dual_tensors(monkeypatch):
    from torch.autograd import forward_ad
    from gan_flow_amd import CnfError
    from gan_flow_amd.lib import optim
    monkeypatch.setattr(optim._native, "_elem", lambda t, name, dtypes=None: t)
    monkeypatch.setattr(optim._native, "orthogonalize", lambda g, out, ns: out.copy_(g))
    g = torch.randn(3, 8)
    with forward_ad.dual_level():
        optim.orthogonalize(g)
        with pytest.raises(CnfError, match="tangent"):
            optim.orthogonalize(forward_ad.make_dual(g, torch.ones_like(g)))


def test_layer_norm_bwd_of_no_rows_without_weight_gradients_enqueues_nothing():
    from gan_flow_amd import _native as nat
    lib = nat.load_library()
    for dx in (None, ONE):
        assert _norm_bwd(lib, rows=0, dx=dx, dw=None, db=None, dy=None, x=None, mean=None, rstd=None, ws=None, bytes_=0) == 0


def test_muon_refuses_to_create_its_momenta_inside_a_capture(monkeypatch):
    from gan_flow_amd import CnfError
    from gan_flow_amd.lib import optim
    p = torch.nn.Parameter(torch.zeros(4, 8))
    p.grad = torch.ones(4, 8)
    taken = []
    monkeypatch.setattr(optim, "_side_by_side", lambda *lists: lists)
    monkeypatch.setattr(optim, "_update", lambda *a, **kw: taken.append(a))
    monkeypatch.setattr(optim, "_capturing", lambda t: True)
    opt = optim.Muon([p])
    with pytest.raises(CnfError, match="before the first one that is captured"):
        opt.step()
    assert not taken
    monkeypatch.setattr(optim, "_capturing", lambda t: False)
    opt.step()
    monkeypatch.setattr(optim, "_capturing", lambda t: True)
    opt.step()                                                 # the momenta exist
    assert len(taken) == 2


def test_every_group_of_muon_is_checked():
    from gan_flow_amd import CnfError
    from gan_flow_amd.lib.optim import Muon
    opt = Muon([torch.nn.Parameter(torch.zeros(4, 8))])
    for bad, error in ((dict(lr=-1.0), ValueError), (dict(lr=float("inf")), ValueError), (dict(momentum=1.0), ValueError), (dict(eps=0.0), ValueError),
                       (dict(adjust_lr=-0.5), ValueError), (dict(adjust_lr="other"), CnfError), (dict(ns_steps=0), CnfError),
                       (dict(weight_decay=float("nan")), ValueError)):
        with pytest.raises(error):
            opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(4, 8))], **bad))
    with pytest.raises(ValueError, match="another optimizer"):
        opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(4))]))
    assert len(opt.param_groups) == 1
    opt.param_groups[0]["lr"] = -1.0
    with pytest.raises(ValueError):
        opt.step()


@pytest.mark.parametrize("c", [0.0, 1e-300, -1e-300, 1e-18, -1e-18, 1e-16, 1e-15, -1e-14, 1e-9])
def test_a_hump_inside_the_interval_is_found_whatever_the_highest_coefficient(c):
    """50 u - 50 u^3 + c u^5 is 0 at both ends of [0, 1] and 19 between: it diverges."""
    from gan_flow_amd import _native as nat
    lib = nat.load_library()
    assert _orth(nat, lib, ns=_ns(nat, steps=1, coefficients=(50.0, -50.0, c)), bytes_=16) != 0 and b"diverge" in lib.cnf_last_error()
    assert _orth(nat, lib, ns=_ns(nat, steps=1, coefficients=(5.0, -5.0, c)), bytes_=16) != 0 and b"workspace" in lib.cnf_last_error()


def test_muon_says_that_a_flow_has_no_hidden_matrices():
    from gan_flow_amd import gu_ffjord
    from gan_flow_amd.lib.optim import MuonWithAdam
    with pytest.raises(ValueError, match="at least two hidden layers"):
        MuonWithAdam(gu_ffjord.build_model(2, (64,)))
    assert len(MuonWithAdam(gu_ffjord.build_model(2, (64, 64))).muon.param_groups[0]["params"]) == 1


def test_muon_loads_no_other_optimizers_state():
    from gan_flow_amd import gu_ffjord
    from gan_flow_amd.lib.optim import Muon, MuonWithAdam
    p = torch.nn.Parameter(torch.zeros(4, 8))
    mine = Muon([p], lr=0.03)
    mine.state[p]["momentum_buffer"] = torch.ones(4, 8)
    fresh = Muon([p])
    others = [torch.optim.SGD([p], lr=0.1, momentum=0.9), torch.optim.Adam([p])]
    if hasattr(torch.optim, "Muon"):
        others.append(torch.optim.Muon([p]))
    for other in others:
        if isinstance(other, torch.optim.Adam):
            other.state[p].update(exp_avg=torch.ones(4, 8), exp_avg_sq=torch.ones(4, 8), step=torch.tensor(1.0))
        else:
            other.state[p]["momentum_buffer"] = torch.ones(4, 8)
        with pytest.raises(ValueError, match="another optimizer"):
            fresh.load_state_dict(other.state_dict())
        assert not fresh.state
    fresh.load_state_dict(mine.state_dict())
    assert fresh.param_groups[0]["lr"] == 0.03 and fresh.state[p]["momentum_buffer"].eq(1).all()
    model = gu_ffjord.build_model(2, (64, 64))
    both = MuonWithAdam(model)
    with pytest.raises(ValueError, match="another optimizer"):
        both.load_state_dict(torch.optim.Adam(model.parameters()).state_dict())
    both.load_state_dict(both.state_dict())


def test_matrices_that_are_read_and_written_by_different_workgroups_are_refused():
    from gan_flow_amd import _native as nat
    lib = nat.load_library()
    A, B, C, D, E, F = (4096 * (i + 1) for i in range(6))
    o, ns = nat.CnfMuonOpts(1e-3, 0.95, 0.1, 1.0, 1, 0), ctypes.byref(_ns(nat))
    for g, words in (((B, C), b"gradient 0 is parameter 1"), ((C, A), b"gradient 1 is parameter 0"), ((B, A), b"is parameter")):
        rc = lib.cnf_muon_step(_ptrs(A, B), 8, _ptrs(*g), 8, _ptrs(E, F), 8, 0, 2, 4, 8, ctypes.byref(o), ns, None, ONE, 1 << 30, None)
        assert rc != 0 and words in lib.cnf_last_error()
    for g, out, words in (((A, B), (B, C), b"output of matrix 0 is matrix 1"), ((A, B), (B, A), b"is matrix"), ((A, B), (D, A), b"output of matrix 1 is matrix 0")):
        rc = lib.cnf_orthogonalize(_ptrs(*g), 8, _ptrs(*out), 8, 0, 2, 4, 8, ns, ONE, 1 << 30, None)
        assert rc != 0 and words in lib.cnf_last_error()


def test_layer_norm_refuses_what_has_no_features_or_no_tensors(monkeypatch):
    from gan_flow_amd import CnfError
    from gan_flow_amd.lib.layers import LayerNorm, layer_norm
    for x in (torch.empty(2, 3, 0), torch.empty(0), torch.empty(0, 0), torch.empty(2, 0, 3, 0)):
        with pytest.raises(CnfError):
            layer_norm(x)
    with pytest.raises(CnfError):
        LayerNorm(8)(torch.tensor(1.0))
    for args in (([1.0] * 8, None), (None, 1.0), (2.0, None)):
        with pytest.raises(CnfError):
            layer_norm(torch.randn(4, 8, requires_grad=True), *args)


def test_matrix_plan():
    from gan_flow_amd import CnfError
    from gan_flow_amd import _native as nat
    assert nat.matrix_plan(1, 64, 64) == (0, 0, 64, 64, 64) and nat.matrix_plan(3, 64, 5000)[:2] == (1, 0)
    for shape in ((1, 200, 300), (8, 1024, 512), (16, 1000, 1000)):
        assert nat.matrix_plan(*shape) == nat.matrix_plan(shape[0], shape[2], shape[1]) and nat.matrix_plan(*shape)[0] == 2
    for bad in ((0, 8, 8), (65, 8, 8), (1, 0, 8), (1, 8, 65537)):
        with pytest.raises(CnfError):
            nat.matrix_plan(*bad)


def test_newton_schulz_check_refuses_what_a_call_would():
    from gan_flow_amd import CnfError
    from gan_flow_amd import _native as nat
    from gan_flow_amd.lib.optim import Muon
    lib = nat.load_library()
    assert lib.cnf_newton_schulz_check(None) != 0 and b"NULL" in lib.cnf_last_error()
    assert lib.cnf_newton_schulz_check(ctypes.byref(_ns(nat))) == 0
    for kw, words in ((dict(coefficients=(9.0, 0.0, 0.0)), b"diverge"), (dict(eps=0.0), b"eps")):
        assert lib.cnf_newton_schulz_check(ctypes.byref(_ns(nat, **kw))) != 0 and words in lib.cnf_last_error()
    p = torch.nn.Parameter(torch.zeros(4, 8))
    opt = Muon([p])
    with pytest.raises(CnfError, match="diverge"):
        opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(4, 8))], ns_coefficients=(9.0, 0.0, 0.0)))
    with pytest.raises(CnfError, match="diverge"):
        Muon([p], ns_coefficients=(9.0, 0.0, 0.0))
    p.grad = torch.ones(4, 8)
    opt.param_groups[0].update(lr=1e300, adjust_lr=1e300)
    with pytest.raises(ValueError, match="hyper-parameters"):
        opt.step()
