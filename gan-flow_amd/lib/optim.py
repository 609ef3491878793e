"""The Muon optimiser for the matrices of a network: each update is the momentum with its singular values driven to one
by Newton-Schulz products (gan-flow_amd/csrc/cnf_muon.hip).  The reference trains with Adam only (the library's
cnf_adam_step); vectors, and whatever else is not a matrix, stay with it."""
import ctypes
import math

import torch
from torch.autograd import forward_ad

from .. import _native

DEFAULT_COEFFICIENTS = (3.4445, -4.7750, 2.0315)   # steep at 0 (3.44), hovers around 1: five steps lift 1e-2 .. 1 into 0.7 .. 1.2
# one call iterates as many matrices side by side as this much workspace holds (at least one): enough to fill the device
_WORKSPACE_BUDGET = 8 << 30


def _at_once(n, rows, cols):
    """How many of n matrices one call takes."""
    one = _native.matrix_workspace_bytes(1, rows, cols)
    if not one:
        raise _native.CnfError("matrices of 1..%d rows and columns (got %d x %d)" % (_native.MAX_MATRIX_DIM, rows, cols))
    return max(1, min(n, _native.MAX_MATRICES, _WORKSPACE_BUDGET // one))


def orthogonalize(g, steps=5, coefficients=DEFAULT_COEFFICIENTS, eps=1e-7):
    """X = g / (|g|_F + eps), then `steps` times X <- a X + (b X X^T + c (X X^T)^2) X, for every matrix of g (..., rows, cols);
    fp32, fp16 or bf16, returned in g's type.  coefficients: (a, b, c), or one such triple per step.  Matrices of zeros
    stay zero.  Not differentiable (dual tensors of forward mode are refused)."""
    _native._elem(g, "g")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(g).tangent is not None:
        raise _native.CnfError("orthogonalize is not differentiable: g carries a forward-mode tangent")
    if g.dim() < 2:
        raise _native.CnfError("g must be a matrix or a stack of matrices (got shape %s)" % (tuple(g.shape),))
    ns = _native.ns_params(steps, coefficients, eps)
    out = torch.empty(g.shape, dtype=g.dtype, device=g.device)
    if g.numel() == 0:
        return out
    rows, cols = g.shape[-2:]
    g3, o3 = g, out
    if g.dim() != 3:
        g3 = g.reshape(-1, rows, cols)
        o3 = out.view(-1, rows, cols)
    if not g3.is_contiguous() and ((cols > 1 and g3.stride(2) != 1) or (rows > 1 and g3.stride(1) < cols)):
        g3 = g3.contiguous()
    n = g3.shape[0]
    step = _at_once(n, rows, cols)
    if step == n:
        _native.orthogonalize(g3, o3, ns)
    else:
        for lo in range(0, n, step):
            _native.orthogonalize(g3[lo:lo + step], o3[lo:lo + step], ns)
    return out


def _loose(rows, cols, strides):
    """Whether the rows of a matrix are not contiguous, or overlap."""
    return cols > 1 and strides[1] != 1 or rows > 1 and strides[0] < cols


def _side_by_side(params, grads, momenta):
    """Lists of (param, gradient, momentum) for one call of the library each: matrices of one shape, type and stride.  Everything is
    checked here, before any of them is updated."""
    if not len(params) == len(grads) == len(momenta):
        raise _native.CnfError("%d params, %d grads, %d momenta" % (len(params), len(grads), len(momenta)))
    groups, seen, given, owned, read = {}, set(), 0, set(), []
    for p, g, m in zip(params, grads, momenta):
        for name, t in (("params", p), ("grads", g), ("momenta", m)):
            if not torch.is_tensor(t) or not t.is_cuda or t.dim() != 2:
                _native._elem(t, name)
                raise _native.CnfError("%s: Muon updates matrices (got shape %s)" % (name, tuple(t.shape)))
        shape, dtype, dev = p.shape, p.dtype, p.device
        if dtype not in _native.DTYPE_IDS or g.dtype != dtype or m.dtype != torch.float32:
            _native._elem(p, "params"), _native._elem(g, "grads", (dtype,)), _native._elem(m, "momenta", (torch.float32,))
        if g.shape != shape or m.shape != shape or g.device != dev or m.device != dev:
            raise _native.CnfError("grads and momenta must have the parameters' shape %s and device %s (got %s on %s, %s on %s)"
                                   % (tuple(shape), dev, tuple(g.shape), g.device, tuple(m.shape), m.device))
        rows, cols = shape
        if not rows or not cols:
            continue
        ps, gs, ms = p.stride(), g.stride(), m.stride()
        if _loose(rows, cols, ps) or _loose(rows, cols, ms):
            raise _native.CnfError("params and momenta: rows must be contiguous and must not overlap (strides %s, %s)" % (ps, ms))
        pp, gp, mp = p.data_ptr(), g.data_ptr(), m.data_ptr()
        if gp != pp:
            read.append(gp)
        if _loose(rows, cols, gs):
            g = g.contiguous()
            gs, gp = g.stride(), g.data_ptr()
        seen.update((pp, mp))
        owned.add(mp)
        given += 2
        groups.setdefault((shape, dtype, dev, ps[0], gs[0], ms[0]), []).append((p, g, m, pp, gp, mp))
    if len(seen) != given:
        raise _native.CnfError("the same parameter or momentum is given twice")
    if not seen.isdisjoint(read):
        raise _native.CnfError("a gradient is also a momentum" if not owned.isdisjoint(read) else "a gradient is another matrix's parameter")
    out = []
    for key, members in groups.items():
        step = _at_once(len(members), *key[0])
        out += [(key, members[lo:lo + step]) for lo in range(0, len(members), step)]
    return out


def _update(calls, ns, lr, momentum, nesterov, weight_decay, scale, guard=None):
    for ((rows, cols), dtype, dev, ldp, ldg, ldm), members in calls:
        n = len(members)
        ps, _, ms, pp, gp, mp = zip(*members)
        array = ctypes.c_void_p * n
        if rows == 1:
            ldp = ldg = ldm = cols
        _native.muon_launch(array(*pp), ldp, array(*gp), ldg, array(*mp), ldm, dtype, (n, rows, cols), dev, ns, lr, momentum, nesterov, weight_decay,
                            scale, guard)
        written = ps + ms                                    # (through raw pointers: autograd is told)
        try:
            torch.autograd.graph.increment_version(written)
        except RuntimeError:                                 # inference tensors have no version
            torch.autograd.graph.increment_version([t for t in written if not t.is_inference()])


def muon_step(params, grads, momenta, lr=1e-3, momentum=0.95, nesterov=True, weight_decay=0.1, scale=1.0, steps=5,
              coefficients=DEFAULT_COEFFICIENTS, eps=1e-7, guard=None):
    """One Muon update, in place, of a list of matrices:
        m <- momentum m + g;   u = g + momentum m (nesterov) or m;   p <- (1 - lr weight_decay) p - lr scale orthogonalize(u)
    grads: of the parameters' types; momenta: fp32.  Matrices of one shape, type and stride are updated side by side.  The
    matrices must not overlap.  guard: the stats words of the solve that made the gradients (a failed one changes nothing).  A call that is
    refused changes nothing either."""
    _update(_side_by_side(params, grads, momenta), _native.ns_params(steps, coefficients, eps), lr, momentum, nesterov, weight_decay, scale, guard)


def adjusted_scale(how, rows, cols):
    """The factor on the orthogonalised update: 'original' sqrt(max(1, rows / cols)), 'match_rms_adamw' 0.2 sqrt(max(rows, cols)) (the
    root mean square of an Adam update, so that Adam's learning rate carries over), or a number."""
    if how == "original":
        return math.sqrt(max(1.0, rows / cols))
    if how == "match_rms_adamw":
        return 0.2 * math.sqrt(max(rows, cols))
    if isinstance(how, str):
        raise _native.CnfError("adjust_lr must be 'original', 'match_rms_adamw' or a number (got %r)" % (how,))
    return float(how)


def _capturing(t):
    return t.is_cuda and torch.cuda.is_current_stream_capturing()


class Muon(torch.optim.Optimizer):
    """Muon for a model's matrices (2-d parameters on a HIP device); every parameter of one shape is updated in one set of
    launches.  State per parameter: `momentum_buffer`, fp32.  step() synchronises nothing and can be captured into a graph
    once the momenta exist (after the first step; refused before); a captured step keeps the learning rate it was captured with."""

    def __init__(self, params, lr=1e-3, weight_decay=0.1, momentum=0.95, nesterov=True, ns_steps=5,
                 ns_coefficients=DEFAULT_COEFFICIENTS, eps=1e-7, adjust_lr="original"):
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov, ns_steps=ns_steps,
                                      ns_coefficients=ns_coefficients, eps=eps, adjust_lr=adjust_lr))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._check(group)
            for p in group["params"]:
                if p.dim() != 2:
                    raise ValueError("Muon updates matrices; give parameters of shape %s to another optimizer" % (tuple(p.shape),))
        except Exception:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check(group):
        """CnfNewtonSchulz of a group whose hyper-parameters are valid."""
        lr, momentum, weight_decay, eps = (group[k] for k in ("lr", "momentum", "weight_decay", "eps"))
        scale = adjusted_scale(group["adjust_lr"], 1, 1)
        if not (0.0 <= lr < math.inf and 0.0 <= momentum < 1.0 and 0.0 <= weight_decay < math.inf and 0.0 < eps < math.inf and 0.0 <= scale < math.inf):
            raise ValueError("invalid hyper-parameters (lr %r, momentum %r, weight_decay %r, eps %r, adjust_lr %r)"
                             % (lr, momentum, weight_decay, eps, group["adjust_lr"]))
        return _native.checked_ns_params(group["ns_steps"], group["ns_coefficients"], eps)

    def load_state_dict(self, state_dict):
        """A state of this class only: other optimizers keep a `momentum_buffer` too (torch.optim.Muon an average of the gradients, 1 - momentum
        times this sum of them)."""
        if any("adjust_lr" not in g for g in state_dict["param_groups"]) or any("momentum_buffer" not in s for s in state_dict["state"].values()):
            raise ValueError("the state is another optimizer's")
        super().load_state_dict(state_dict)   # (casts state to the parameter's type: the momentum is fp32 whatever that is)
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        mine = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(saved, mine):
            if i in state_dict["state"]:
                self.state[p]["momentum_buffer"] = state_dict["state"][i]["momentum_buffer"].to(device=p.device, dtype=torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        updates = []                                         # (everything is checked before anything is updated)
        for group in self.param_groups:
            ns, by_shape = self._check(group), {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise _native.CnfError("Muon does not take sparse gradients")
                state = self.state[p]
                if "momentum_buffer" not in state:
                    if _capturing(p):                        # (its zeros would be written again at every replay)
                        raise _native.CnfError("Muon's momenta do not exist yet: take a step before the first one that is captured")
                    state["momentum_buffer"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                by_shape.setdefault(p.shape, []).append((p, p.grad, state["momentum_buffer"]))
            hyper = {k: group[k] for k in ("lr", "momentum", "nesterov", "weight_decay")}
            for shape, members in by_shape.items():
                scale = adjusted_scale(group["adjust_lr"], *shape)
                if not math.isfinite(hyper["lr"] * scale) or not math.isfinite(hyper["lr"] * hyper["weight_decay"]):
                    raise ValueError("invalid hyper-parameters (lr %r, weight_decay %r, scale %r)" % (hyper["lr"], hyper["weight_decay"], scale))
                updates.append((_side_by_side(*zip(*members)), ns, dict(hyper, scale=scale)))
        for calls, ns, hyper in updates:
            _update(calls, ns, **hyper)
        return loss


class MuonWithAdam:
    """Muon for the hidden matrices of the ODE nets of a flow (the weights from hidden to hidden layers), torch.optim.Adam for every other
    parameter: first and last layers, biases, time terms, end times.  `muon`, `adam`: the arguments of the two.  Behaves as an
    optimizer where gu_ffjord's training loops need one (zero_grad, step, state_dict, load_state_dict)."""

    def __init__(self, model, muon=None, adam=None):
        hidden = some_matrices(hidden_matrices(model))
        taken = {id(p) for p in hidden}
        self.muon = Muon(hidden, **dict(muon or {}))
        self.adam = torch.optim.Adam([p for p in model.parameters() if id(p) not in taken], **dict(adam or {}))

    def zero_grad(self, set_to_none=True):
        self.muon.zero_grad(set_to_none)
        self.adam.zero_grad(set_to_none)

    def step(self):
        self.muon.step()
        self.adam.step()

    def state_dict(self):
        return {"muon": self.muon.state_dict(), "adam": self.adam.state_dict()}

    def load_state_dict(self, state):
        if "muon" not in state or "adam" not in state:
            raise ValueError("the state is another optimizer's (Muon's and Adam's are wanted, got %s)" % sorted(state))
        self.muon.load_state_dict(state["muon"])
        self.adam.load_state_dict(state["adam"])


def hidden_matrices(model):
    """The weights from hidden to hidden layers of every ODE net of a flow, in the order of its blocks."""
    from .layers.cnf import CNF, _inner
    out = []
    for blk in model.chain:
        if isinstance(blk, CNF):
            out += [layer._layer.weight for layer in list(_inner(blk.odefunc).diffeq.layers)[1:-1]]
    return out


def some_matrices(hidden):
    if not hidden:
        raise ValueError("Muon updates the weights from hidden to hidden layers, and this flow has none: its nets need at least two hidden layers")
    return hidden
