"""GPU: the training iteration with Muon on the hidden matrices -- FusedTrainStep(optimizer="muon") against the autograd loop with
lib.optim.MuonWithAdam on the same solves, batches and initial weights; resume; failed solves; the driver's --optimizer muon.

The two loops' gradients agree to about 1e-5 relative (the adjoint's rounding).  Muon's polynomial lifts a deviation at most 3.4445^5 =
485-fold in a direction, so an update's entries (1 / sqrt(64) each, times lr = 0.02) differ by at most 485e-5 * 0.02 / 8 = 1.2e-5
a step; over the six steps taken here 1e-4 is allowed, in parameters and (relative) in the loss they give."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
MUON = dict(lr=0.02, momentum=0.9, weight_decay=0.01)


def _batches(n=6, rows=512):
    from gan_flow_amd.gu import make_gu
    data = make_gu(8, seed=3)
    return [data.get_sample(rows).to(DEV) for _ in range(n)]


def _model(blocks=1, dims=(64, 64, 64), **kw):
    from gan_flow_amd import gu_ffjord
    torch.manual_seed(5)
    return gu_ffjord.build_model(2, dims, num_blocks=blocks, **kw).to(DEV).train()


def _flat(model):
    return torch.cat([p.detach().reshape(-1) for n, p in model.named_parameters() if "sqrt_end_time" not in n])


@pytest.mark.parametrize("graph, blocks, dims, kw", [
    (True, 1, (64, 64, 64), {}), (False, 2, (64, 64, 64), {}), (True, 2, (48, 32, 40), {}), (True, 1, (64, 64, 64), dict(layer_type="ignore")),
    (True, 1, (256, 256, 256), {}), (False, 1, (64, 64, 64), dict(solver="rk4"))])
def test_fused_muon_step_matches_autograd_loop(graph, blocks, dims, kw):
    from gan_flow_amd import gu_ffjord
    from gan_flow_amd.lib.optim import MuonWithAdam, hidden_matrices
    batches = _batches()
    ref = _model(blocks, dims, **kw)
    opt = MuonWithAdam(ref, MUON, dict(lr=1e-3, weight_decay=1e-5))
    assert len(hidden_matrices(ref)) == 2 * blocks
    start = _flat(ref)
    want = []
    for x in batches:
        opt.zero_grad(set_to_none=True)
        loss = gu_ffjord.compute_loss(ref, x)
        loss.backward()
        opt.step()
        want.append(loss.item())
    model = _model(blocks, dims, **kw)
    step = gu_ffjord.FusedTrainStep(model, batches[0], lr=1e-3, weight_decay=1e-5, graph=graph, optimizer="muon", muon=MUON)
    assert torch.equal(_flat(model), start) and step.step_count == 0          # (the dry run before the capture left nothing behind)
    got = [step(x).item() for x in batches]
    step.check()
    assert step.step_count == len(batches)
    assert all(abs(a - b) <= 1e-4 * abs(a) for a, b in zip(want, got)), (want, got)
    assert (_flat(ref) - _flat(model)).abs().max().item() <= 1e-4
    for m, p in zip(step.momenta, hidden_matrices(ref)):
        buf = opt.muon.state[p]["momentum_buffer"]
        assert (m - buf).norm() <= 1e-3 * buf.norm()


def test_fused_muon_step_resumes():
    from gan_flow_amd import gu_ffjord
    batches = _batches(5)
    args = dict(lr=1e-3, weight_decay=1e-5, optimizer="muon", muon=MUON)
    a = _model()
    step = gu_ffjord.FusedTrainStep(a, batches[0], **args)
    for x in batches[:3]:
        step(x)
    step.check()
    saved = {k: v.clone() for k, v in a.state_dict().items()}, step.state_dict()
    for x in batches[3:]:
        step(x)
    step.check()
    b = _model()
    b.load_state_dict(saved[0])
    again = gu_ffjord.FusedTrainStep(b, batches[0], **args)
    again.load_state_dict(saved[1])
    for x in batches[3:]:
        again(x)
    again.check()
    assert torch.equal(_flat(a), _flat(b)) and again.step_count == 5
    with pytest.raises(ValueError, match="another optimizer"):
        gu_ffjord.FusedTrainStep(_model(), batches[0], graph=False).load_state_dict(saved[1])
    with pytest.raises(ValueError):
        gu_ffjord.FusedTrainStep(_model(), batches[0], graph=False, optimizer="sgd")
    with pytest.raises(ValueError):
        gu_ffjord.FusedTrainStep(_model(), batches[0], graph=False, muon=MUON)
    with pytest.raises(ValueError):
        gu_ffjord.FusedTrainStep(_model(), batches[0], graph=False, optimizer="muon", muon=dict(momentum=1.5))


def test_failed_solve_leaves_the_matrices_and_momenta_alone():
    from gan_flow_amd import CnfError, gu_ffjord
    batches = _batches(2)
    model = _model(2)
    step = gu_ffjord.FusedTrainStep(model, batches[0], graph=False, optimizer="muon", muon=MUON)
    step(batches[0])
    step.check()
    before = _flat(model), [m.clone() for m in step.momenta]
    bad = batches[1].clone()
    bad[7, 0] = float("nan")
    step(bad)
    with pytest.raises(CnfError):
        step.check()
    assert torch.equal(_flat(model), before[0]) and all(torch.equal(p, q) for p, q in zip(step.momenta, before[1]))


@pytest.mark.parametrize("fused", [1, 0])
def test_driver_trains_with_muon(tmp_path, fused):
    from gan_flow_amd import gu_ffjord
    common = ["--gu_num", "1", "--batch_size", "256", "--optimizer", "muon", "--eval_size", "2000", "--eval_logp_size", "2000",
              "--log_interval", "4", "--save", str(tmp_path), "--fused", str(fused)]
    model = gu_ffjord.main(common + ["--niters", "4"])
    first = _flat(model)
    model = gu_ffjord.main(common + ["--niters", "8", "--resume", str(tmp_path / "ffjord_checkpoint.pth")])
    ck = torch.load(tmp_path / "ffjord_checkpoint.pth", weights_only=True)
    assert ck["itr"] == 8 and torch.isfinite(_flat(model)).all() and not torch.equal(first, _flat(model))
    assert ("momenta" if fused else "muon") in ck["optimizer"]


def test_graphed_loop_with_muon_replays_the_eager_steps():
    from gan_flow_amd import gu_ffjord
    from gan_flow_amd.lib.optim import MuonWithAdam
    batches = _batches(5)
    adam = dict(lr=1e-3, capturable=True)
    ref = _model()
    opt = MuonWithAdam(ref, MUON, adam)
    for x in batches:
        opt.zero_grad()
        gu_ffjord.compute_loss(ref, x).backward()
        opt.step()
    model = _model()
    step = gu_ffjord.GraphedTrainStep(model, MuonWithAdam(model, MUON, adam), batches[0], warmup_batches=batches[:1])
    for x in batches[1:]:
        step(x)
    step.check()
    assert (_flat(ref) - _flat(model)).abs().max().item() <= 1e-4


def test_graphed_loop_without_a_warm_up_is_refused_for_muon():
    from gan_flow_amd import CnfError, gu_ffjord
    from gan_flow_amd.lib.optim import MuonWithAdam
    batches = _batches(1)
    model = _model()
    with torch.no_grad():                                      # (what the solves themselves read back once is there)
        gu_ffjord.compute_loss(model, batches[0])
    with pytest.raises(CnfError, match="before the first one that is captured"):
        gu_ffjord.GraphedTrainStep(model, MuonWithAdam(model, MUON, dict(lr=1e-3, capturable=True)), batches[0])


def test_fused_muon_step_says_that_a_flow_has_no_hidden_matrices():
    from gan_flow_amd import gu_ffjord
    with pytest.raises(ValueError, match="at least two hidden layers"):
        gu_ffjord.FusedTrainStep(_model(dims=(64,)), _batches(1)[0], optimizer="muon", muon=MUON)


def _compare(model_kw, muon, batches, coeffs=None, **step_kw):
    """The captured iteration against the autograd loop on the same batches, as above."""
    from gan_flow_amd import gu_ffjord
    from gan_flow_amd.lib.optim import MuonWithAdam
    ref = _model(**model_kw)
    opt = MuonWithAdam(ref, muon, dict(lr=1e-3, weight_decay=1e-5))
    want = []
    for x in batches:
        opt.zero_grad(set_to_none=True)
        loss = gu_ffjord.compute_loss(ref, x)
        if coeffs:
            loss = loss + gu_ffjord.get_regularization(ref, coeffs)
        loss.backward()
        opt.step()
        want.append(loss.item())
    model = _model(**model_kw)
    step = gu_ffjord.FusedTrainStep(model, batches[0], lr=1e-3, weight_decay=1e-5, optimizer="muon", muon=muon, reg_coeffs=coeffs, **step_kw)
    got = [step(x).item() for x in batches]
    step.check()
    assert all(abs(a - b) <= 1e-4 * abs(a) for a, b in zip(want, got)), (want, got)
    assert (_flat(ref) - _flat(model)).abs().max().item() <= 1e-4


@pytest.mark.parametrize("layer_type", ["concat_v2", "squash"])
def test_fused_muon_step_of_other_layer_types(layer_type):
    _compare(dict(layer_type=layer_type, dims=(64, 48, 64)), MUON, _batches())


@pytest.mark.parametrize("kw", [dict(nesterov=False), dict(adjust_lr="match_rms_adamw", lr=0.005), dict(ns_steps=3, ns_coefficients=[(4.0, -6.0, 2.5), (3.0, -3.5, 1.4),
                                (1.5, -0.5, 0.0)]), dict(adjust_lr=0.5, eps=1e-3)], ids=str)
def test_fused_muon_step_takes_muons_arguments(kw):
    _compare(dict(), dict(MUON, **kw), _batches(), spread=False)


def test_fused_muon_step_with_kinetic_regularisers():
    from gan_flow_amd.lib.layers.wrappers import cnf_regularization as creg
    _compare(dict(blocks=2, regularization_fns=(creg.l1_regularzation_fn, creg.l2_regularzation_fn)), MUON, _batches(), coeffs=[0.5, 0.25])


def test_fused_muon_step_with_a_device_sampler():
    from gan_flow_amd import gu_ffjord
    from gan_flow_amd.gu import make_gu
    runs = []
    for _ in range(2):
        model = _model()
        sampler = make_gu(8, seed=3, extend_dim=True).device_sampler(torch.device(DEV))
        step = gu_ffjord.FusedTrainStep(model, torch.zeros(512, 2, device=DEV), sampler=sampler, warmup=2, optimizer="muon", muon=MUON)
        losses = [step().item() for _ in range(5)]
        step.check()
        runs.append((losses, _flat(model)))
        assert step.step_count == 7
    assert runs[0][0] == runs[1][0] and torch.equal(runs[0][1], runs[1][1]) and torch.isfinite(runs[0][1]).all()
